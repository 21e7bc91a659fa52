"""A residual that is one row for all, and operands that are rows of one tensor: calls that the rules on places allow."""
import pytest
import torch

from iian_b200.ops.cuda_backend import CudaKernels

pytestmark = pytest.mark.gpu
K = CudaKernels
BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype,wdtype,k", [(BF, BF, 512), (F32, F32, 512), (F32, F32, 77), (BF, BF, 77), (BF, F32, 64)])
@pytest.mark.parametrize("n,m", [(1, 64), (20, 700), (130, 333), (300, 256)])
@pytest.mark.parametrize("rdtype", [F32, BF])
def test_one_row_for_all(dtype, wdtype, k, n, m, rdtype):
    g = torch.Generator("cuda").manual_seed(n + m)
    store = torch.randn(n + m, k, device="cuda", generator=g) * 0.2
    x, w = store[:n].to(dtype), store[n:].to(wdtype)
    if dtype == wdtype:                                              # views of the same tensor
        both = store.to(dtype)
        x, w = both[:n], both[n:]
    r = torch.randn(1, m, device="cuda", generator=g).to(rdtype).expand(n, m)
    out = torch.empty(n, m, device="cuda")
    K().linear_act(x, w, out, residual=r)
    K().check_device_status()
    y, total = x.double() @ w.double().t(), x.double().abs() @ w.double().abs().t()
    ref = y + r.double()
    # the longer of the chains: 2^-23 of sum |x w| twice for each 16 products, or 2^-24 for each product; 32 roundings of what is joined
    tol = total * max(2 * (k / 16 + 1) * 2.0 ** -23, k * 2.0 ** -24) + 32 * 2.0 ** -24 * (total + ref.abs() + r.double().abs())
    assert ((out.double() - ref).abs() <= tol).all()
