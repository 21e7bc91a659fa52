"""What the kernel layer refuses before it looks for a device: sizes that no 32-bit number holds (of tensors that no memory holds either)."""
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
