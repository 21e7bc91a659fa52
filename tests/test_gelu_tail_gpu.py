"""gelu by erf in the products' epilogues keeps its digits where it is small: its lower tail is y times a small probability, not 1 less a number next
to it."""
import math

import pytest
import torch

from iian_b200.ops.cuda_backend import CudaKernels

pytestmark = pytest.mark.gpu
K = CudaKernels
BF, F32 = torch.bfloat16, torch.float32


def exact(y):
    return 0.5 * y.double() * torch.special.erfc(-y.double() * math.sqrt(0.5))


@pytest.mark.parametrize("dtype,n,form", [(F32, 3, 0), (F32, 40, 0), (BF, 1, 0), (BF, 100, 0 | 64 << 1 | 2 << 16), (BF, 130, 0 | 256 << 1 | 1 << 16), (BF, 300, 1 | 96 << 1 | 1 << 16)])
def test_lower_tail(dtype, n, form):
    """The product is 0, the bias the argument.  Units of 2^-24 relative to the tail |y| Q(|y|): the argument of the reciprocal and its own error 6,
    seven steps of the polynomial 4, its fit 2.2, the exponential 4, products 3; and 3 of the exponent, y^2 / 2.  A positive y has y less that tail."""
    y = torch.cat([torch.linspace(-12.5, 12.5, 20001), torch.tensor([0.0, -0.0, -1e-30, 1e-3, -4.0, -3.0, -5.0])]).cuda()
    m = y.numel()
    x, w = torch.zeros(n, 128, device="cuda", dtype=dtype), torch.zeros(m, 128, device="cuda", dtype=dtype)
    out = torch.empty(n, m, device="cuda")
    K().linear_act(x, w, out, bias=y, activation="gelu", form=form)
    K().check_device_status()
    want = exact(y)
    tail = exact(-y.abs()).abs()
    units = 20 + 1.5 * y.double().square()
    assert ((out.double() - want).abs() <= 2.0 ** -24 * (units * tail + want.abs()) + 1e-37).all()


def test_bfloat16_outputs_are_the_nearest():
    """Away from the middle between two, a bfloat16 output is the one next to the value."""
    y = torch.linspace(-6, -1, 5001).cuda()
    x, w, out = torch.zeros(2, 64, device="cuda", dtype=BF), torch.zeros(5001, 64, device="cuda", dtype=BF), torch.empty(2, 5001, device="cuda", dtype=BF)
    K().linear_act(x, w, out, bias=y, activation="gelu")
    want = exact(y)
    assert ((out.double() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -17)).all()


def test_ends():
    y = torch.tensor([float("inf"), float("-inf"), float("nan"), 3e38, -3e38, -100.0, 100.0, -14.0], device="cuda")
    for dtype in (F32, BF):
        out = torch.empty(1, 8, device="cuda")
        K().linear_act(torch.zeros(1, 64, device="cuda", dtype=dtype), torch.zeros(8, 64, device="cuda", dtype=dtype), out, bias=y, activation="gelu")
        o = out[0].tolist()
        assert o[0] == math.inf and o[1] == 0.0 and math.isnan(o[2]) and o[3] == y[3].item() and o[4] == 0.0 and o[5] == 0.0 and o[6] == 100.0 and abs(o[7]) < 1e-37
