"""What the kernel layer refuses before it looks for a device: sizes that no 32-bit number holds (of tensors that no memory holds either), caps that
are none in 32 bits."""
import pytest
import torch

from iian_b200.ops.cuda_backend import CudaKernels, KernelError

BIG = 2 ** 31
BF, F32, I32 = torch.bfloat16, torch.float32, torch.int32


def t(*shape, dtype=BF):
    return torch.empty(*shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("n,k,m", [(BIG, 8, 1), (1, BIG, 1), (1, 8, BIG), (BIG + 5, 8, 3), (2 ** 32 + 1, 8, 2)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_products(n, k, m, dtype):
    with pytest.raises(KernelError, match="2,147,483,647"):
        CudaKernels().linear_act(t(n, k, dtype=dtype), t(m, k, dtype=dtype), t(n, m, dtype=dtype))


@pytest.mark.parametrize("k,v", [(BIG, 4), (8, BIG), (8, 2 ** 32 + 7)])
def test_scores(k, v):
    with pytest.raises(KernelError, match="2,147,483,647"):
        CudaKernels().linear_logprobs(t(2, k), t(v, k), t(2, dtype=I32), t(2, dtype=F32), t(2, dtype=F32))


@pytest.mark.parametrize("n,e", [(BIG, 4), (2 ** 32 + 3, 4)])
def test_routing(n, e):
    with pytest.raises(KernelError, match="2,147,483,647"):
        CudaKernels().moe_route_grouped(t(n, e, dtype=F32), 1, t(n, 1, dtype=I32), t(n, 1, dtype=F32))


@pytest.mark.parametrize("cap", [1e39, 1e300, 1e-46, 1e-40, 5e-324])
def test_caps_that_32_bits_do_not_hold(cap):
    with pytest.raises(KernelError, match="softcap"):
        CudaKernels().linear_logprobs(t(2, 8), t(4, 8), t(2, dtype=I32), t(2, dtype=F32), t(2, dtype=F32), softcap=cap)


@pytest.mark.parametrize("cap", [2.0 ** -126, 30, 30.0, 3e38, None])
def test_caps_that_they_do(cap):
    with pytest.raises(KernelError, match="two tensors"):           # (the next thing that is looked at)
        CudaKernels().linear_logprobs(t(2, 8), t(4, 8), t(2, dtype=I32), t(2, dtype=F32), t(2, dtype=F32), softcap=cap)
