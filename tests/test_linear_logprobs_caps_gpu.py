"""Capped scores at caps from far below the logits to far above them: a logit keeps its digits whatever the cap is, in every form."""
import pytest
import torch

from iian_b200.ops.cuda_backend import CudaKernels

pytestmark = pytest.mark.gpu
K = CudaKernels
BF, F32 = torch.bfloat16, torch.float32


def check(n, k, v, cap, dtype=BF, wdtype=None, form=0, std=0.1):
    g = torch.Generator("cuda").manual_seed(n + k + v)
    x = torch.randn(n, k, device="cuda", generator=g).to(dtype)
    w = (torch.randn(v, k, device="cuda", generator=g) * std).to(wdtype or dtype)
    t = torch.randint(0, v, (n,), device="cuda", generator=g, dtype=torch.int32)
    lp, lse = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    K().linear_logprobs(x, w, t, lp, lse, softcap=cap, form=form)
    z = x.double() @ w.double().t()
    zc = cap * torch.tanh(z / cap)
    want = torch.logsumexp(zc, 1)
    picked = zc.gather(1, t.long()[:, None])[:, 0]
    # The chain of a logit: 2^-23 of sum |x w| twice for 16 products on the tensor cores, 2^-24 for each otherwise, and 32 roundings; a cap does
    # not stretch that.  The cap itself, relative to what it gives: its argument two roundings (half a polynomial's of it, a few 2^-24), or, from 0.8 on,
    # c (1 - q) with q = 2 / (1 + e^2u) off by 2^-22 for the exponential, 2^-22 of 2 u for its argument and 2^-22 for the quotient, of which q /
    # (1 - q) <= 0.51 counts, and two roundings: 2.2 times 2^-22.  Then the sum: as without a cap.
    total = (x.double().abs() @ w.double().abs().t()).amax(1)
    tc = dtype == BF and w.dtype == BF and k % 8 == 0
    logit = total * ((2 * (k / 16 + 1)) * 2.0 ** -23 if tc else k * 2.0 ** -24) + 32 * 2.0 ** -24 * total.clamp(max=float(2 * zc.abs().max()) + 1)
    logit = logit + 2.2 * 2.0 ** -22 * zc.abs().amax(1)
    tol = logit + 2.0 ** -22 + 200 * 2.0 ** -24 + 3 * 2.0 ** -23 * zc.abs().amax(1) + 2.0 ** -23 * want.abs()
    assert ((lse.double() - want).abs() <= tol).all()
    assert ((lp.double() - (picked - want)).abs() <= tol + logit + 2.0 ** -23 * (picked - want).abs()).all()
    K().check_device_status()


CAPS = [1e-3, 0.3, 5.0, 30.0, 1e3, 1e5, 1e6, 1e30]


@pytest.mark.parametrize("cap", CAPS)
@pytest.mark.parametrize("n,k,v", [(1, 64, 4099), (60, 136, 999), (128, 64, 331), (300, 64, 2500)])
def test_bfloat16(n, k, v, cap):
    check(n, k, v, cap)
    check(n, k, v, cap, std=2.0)


@pytest.mark.parametrize("cap", CAPS)
@pytest.mark.parametrize("n", [3, 150])
def test_every_form_of_the_product(n, cap):
    check(n, 72, 3001, cap, form=0 | 80 << 1 | 1 << 16)          # x's rows as the product's
    check(n, 72, 3001, cap, form=1 | 96 << 1 | 1 << 16)          # on pairs


@pytest.mark.parametrize("cap", CAPS)
@pytest.mark.parametrize("dtype,wdtype,k", [(F32, F32, 64), (BF, BF, 67), (BF, F32, 64)])
def test_logits_in_memory(dtype, wdtype, k, cap):
    check(9, k, 5003, cap, dtype, wdtype)
    check(140, k, 503, cap, dtype, wdtype)


def test_both_ways_say_the_same():
    """The same rows with K a multiple of 8 and with a column of zeros more, at a cap a thousand times the logits."""
    g = torch.Generator("cuda").manual_seed(3)
    x, w = torch.randn(20, 64, device="cuda", generator=g).to(BF), (torch.randn(700, 64, device="cuda", generator=g) * 0.1).to(BF)
    t = torch.randint(0, 700, (20,), device="cuda", generator=g, dtype=torch.int32)
    got = []
    for pad in (0, 1):
        lp, lse = torch.empty(20, device="cuda"), torch.empty(20, device="cuda")
        K().linear_logprobs(torch.nn.functional.pad(x, (0, pad)), torch.nn.functional.pad(w, (0, pad)).contiguous(), t, lp, lse, softcap=1e6)
        got.append(lp)
    # each by the bound above: K = 64, sum |x w| below 20, logits below 6
    assert (got[0] - got[1]).abs().max().item() <= 2 * (20 * 10 * 2.0 ** -23 + 64 * 20 * 2.0 ** -24 / 2 + 64 * 2.0 ** -24 * 12 + 300 * 2.0 ** -24)


@pytest.mark.parametrize("cap", [2.0 ** -126, 3e38])
@pytest.mark.parametrize("dtype,n,k", [(BF, 3, 64), (BF, 150, 64), (F32, 9, 64), (BF, 9, 67)])
def test_the_least_and_the_largest_cap(dtype, n, k, cap):
    check(n, k, 503, cap, dtype)
