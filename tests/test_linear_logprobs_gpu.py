"""Log-probabilities of given tokens without the logits against float64: types, vocabularies no tile divides, one row to more than a
launch's, caps, targets that are none, infinities, rows behind the last, captured graphs."""
import pytest
import torch

import iian_b200.ops.cuda_backend as backend
from iian_b200.ops.cuda_backend import CudaKernels, KernelError

pytestmark = pytest.mark.gpu
K = CudaKernels
BF, F32 = torch.bfloat16, torch.float32


def exact(x, w, targets, cap):
    z = x.double() @ w.double().t()
    z = cap * torch.tanh(z / cap) if cap else z
    lse = torch.logsumexp(z, 1)
    t = targets.long()
    lp = torch.where(t < 0, 0.0, z.gather(1, t.clamp(0, z.shape[1] - 1)[:, None])[:, 0] - lse)
    return lp, lse


def tolerance(x, w, lse, lp, cap, tc):
    """A logit is off by no more than its chain's roundings (as for the products: 2^-23 of sum |x w| twice for 16 products on the tensor cores,
    2^-24 for each otherwise), which a cap does not stretch, and with a cap by c times the tanh's few 1e-7 and its argument's rounding.  The
    log-sum-exp moves by no more than the largest of these, and by the relative error of the sum: 2^-22 for an exponential, up to
    2^-24 for each addition in a row of them -- under 200 for any vocabulary -- and its argument's rounding, 2^-24 of the logit in units of
    log2 e.  lp is a difference of the two, each rounded once."""
    k = x.shape[1]
    total = (x.double().abs() @ w.double().abs().t()).amax(1)
    logit = total * (2 * (k / 16 + 1) * 2.0 ** -23 if tc else k * 2.0 ** -24) + 32 * 2.0 ** -24 * total
    if cap:
        logit = logit + cap * 1e-6
        total = total.clamp(max=cap)
    both = logit + 2.0 ** -22 + 200 * 2.0 ** -24 + 3 * 2.0 ** -23 * total + 2.0 ** -23 * lse.abs()
    return both, both + logit + 2.0 ** -23 * lp.abs()


def check(n, k, v, dtype=BF, cap=None, form=0, std=0.1, wdtype=None, x=None, w=None):
    g = torch.Generator("cuda").manual_seed(n + k + v)
    x = torch.randn(n, k, device="cuda", generator=g).to(dtype) if x is None else x
    w = (torch.randn(v, k, device="cuda", generator=g) * std).to(wdtype or dtype) if w is None else w
    t = torch.randint(0, v, (n,), device="cuda", generator=g, dtype=torch.int32)
    t[0], t[n // 2] = v - 1, 0
    if n > 3:
        t[3] = -1
    lp, lse = torch.full((n + 1,), 7.0, device="cuda"), torch.full((n + 1,), 7.0, device="cuda")
    K().linear_logprobs(x, w, t, lp[:n], lse[:n], softcap=cap, form=form)
    want_lp, want_lse = exact(x, w, t, cap)
    tc = dtype == BF and w.dtype == BF and k % 8 == 0
    tol_lse, tol_lp = tolerance(x, w, want_lse, want_lp, cap, tc)
    assert ((lse[:n].double() - want_lse).abs() <= tol_lse).all()
    assert ((lp[:n].double() - want_lp).abs() <= tol_lp).all()
    assert lp[n] == 7.0 and lse[n] == 7.0                       # what lies behind the last row
    K().check_device_status()


@pytest.mark.parametrize("n,k,v", [(1, 64, 1), (1, 8, 33), (1, 1024, 20000), (2, 512, 31), (7, 72, 503), (33, 256, 4099), (64, 2048, 1000), (100, 136, 999), (128, 512, 2048),
                                   (129, 512, 2048), (256, 64, 777), (300, 1024, 5001), (700, 320, 331), (2500, 128, 1200)])
def test_bfloat16(n, k, v):
    check(n, k, v)
    check(n, k, v, cap=15.0)


@pytest.mark.parametrize("n,k,v", [(1, 64, 1), (1, 1024, 20000), (5, 70, 503), (40, 128, 9001), (130, 256, 50000), (300, 33, 331)])
def test_float32(n, k, v):
    check(n, k, v, F32)
    check(n, k, v, F32, cap=15.0)


@pytest.mark.parametrize("dtype,wdtype,k", [(BF, BF, 71), (BF, F32, 64), (F32, BF, 64)])
def test_what_the_tensor_cores_do_not_take(dtype, wdtype, k):
    check(9, k, 5003, dtype, wdtype=wdtype)


def form(pair, bn):
    return int(pair) | bn << 1 | 1 << 16


@pytest.mark.parametrize("n", [1, 60, 128, 300])
@pytest.mark.parametrize("pair,bn", [(0, 32), (0, 80), (0, 208), (0, 256), (1, 32), (1, 160), (1, 256)])
def test_every_form(n, pair, bn):
    check(n, 264, 3001, form=form(pair, bn))


@pytest.mark.parametrize("n", [1, 17, 60, 128])
@pytest.mark.parametrize("bn", [32, 57, 115, 128])
def test_every_form_of_few_rows(n, bn):
    check(n, 264, 3001, form=form(0, bn) | 1 << 14)
    check(n, 264, 3001, cap=9.0, form=form(0, bn) | 1 << 14)


@pytest.mark.parametrize("n,bad", [(4, 0 | 16 << 1), (4, 0 | 272 << 1), (4, 0 | 40 << 1), (300, 1 | 48 << 1), (4, 1 << 14 | 144 << 1), (200, 1 << 14 | 64 << 1)])
def test_forms_there_are_none_of(n, bad):
    with pytest.raises(KernelError):
        check(n, 64, 500, form=bad | 1 << 16)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_more_rows_than_a_launch_takes(dtype, monkeypatch):
    monkeypatch.setattr(backend.CudaKernels, "SCORE_ROWS", 100)
    monkeypatch.setattr(backend.CudaKernels, "SCORE_PIECE", 1 << 14)
    check(350, 64, 9003, dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_apart(dtype):
    wide = torch.randn(40, 96, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(dtype)
    check(33, 64, 700, dtype, x=wide[3:36, 16:80])


@pytest.mark.parametrize("scale", [30.0, 1000.0])
def test_large_logits_do_not_overflow(scale):
    """Logits of some hundred and some thousand, of both signs, the largest in the first and in the last column."""
    for n, v in ((3, 5000), (200, 600)):
        g = torch.Generator("cuda").manual_seed(v)
        x = torch.randn(n, 64, device="cuda", generator=g).to(BF)
        w = (torch.randn(v, 64, device="cuda", generator=g) * scale / 8).to(BF)
        w[0], w[-1] = x[0] * scale, x[1] * scale
        check(n, 64, v, x=x, w=w)
        check(n, 64, v, F32, x=x.float(), w=w.float())


@pytest.mark.parametrize("dtype", [BF, F32])
def test_infinities_and_what_is_no_number(dtype):
    n, k, v = 6, 64, 1500
    g = torch.Generator("cuda").manual_seed(5)
    x = torch.zeros(n, k, device="cuda", dtype=dtype)
    x[:, 1:] = torch.randn(n, k - 1, device="cuda", generator=g).to(dtype)
    w = (torch.randn(v, k, device="cuda", generator=g) * 0.1).to(dtype)
    w[:, 0] = 1.0
    x[1, 0] = float("-inf")              # every logit minus infinity
    x[2, 0] = float("inf")
    x[3, 0] = float("nan")
    t = torch.tensor([5, 5, 5, 5, v, -3], device="cuda", dtype=torch.int32)
    lp, lse = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    K().linear_logprobs(x, w, t, lp, lse)
    assert torch.isfinite(lse[[0, 4, 5]]).all() and torch.isfinite(lp[0])
    assert lse[1] == float("-inf") and torch.isnan(lp[1])
    assert lse[2] == float("inf") and torch.isnan(lse[3]) and torch.isnan(lp[3])
    assert torch.isnan(lp[4]) and lp[5] == 0.0
    # some of a row's logits minus infinity, a whole tile of them among these
    w2 = w.clone()
    w2[300:900, 0] = float("-inf")
    x2 = x[[0, 5]].clone()
    x2[:, 0] = 1.0
    t2 = torch.tensor([400, 1000], device="cuda", dtype=torch.int32)
    K().linear_logprobs(x2, w2, t2, lp[:2], lse[:2])
    z = x2.double() @ w2.double().t()
    want = torch.logsumexp(z, 1)
    assert ((lse[:2].double() - want).abs() <= 1e-4).all() and lp[0] == float("-inf") and abs(lp[1].item() - (z[1, 1000] - want[1]).item()) <= 1e-4


def test_no_rows_and_refusals():
    k, z = K(), lambda *s, t=BF: torch.zeros(*s, device="cuda", dtype=t)      # noqa: E731
    i = lambda n: z(n, t=torch.int32)                                          # noqa: E731
    f = lambda n: z(n, t=F32)                                                  # noqa: E731
    k.linear_logprobs(z(0, 64), z(10, 64), i(0), f(0), f(0))
    x, w = z(4, 64), z(32, 64)
    same = f(4)
    for args in ((x, w, i(3), f(4), f(4)), (x, w, f(4), f(4), f(4)), (x, w, i(4), z(4), f(4)), (x, w, i(4), f(4), f(5)), (x, z(0, 64), i(4), f(4), f(4)),
                 (x, w, i(4), same, same), (x, w, torch.zeros(4, dtype=torch.int32), f(4), f(4)), (x, torch.zeros(32, 64, dtype=BF), i(4), f(4), f(4))):
        with pytest.raises(KernelError):
            k.linear_logprobs(*args)
    for cap in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(KernelError, match="softcap"):
            k.linear_logprobs(x, w, i(4), f(4), f(4), softcap=cap)


@pytest.mark.parametrize("dtype,n", [(BF, 1), (BF, 50), (BF, 200), (F32, 3)])
def test_captured_twice_and_replayed(dtype, n):
    """Two graphs of the same call, each with a working memory of its own, replayed on two streams at once."""
    g = torch.Generator("cuda").manual_seed(n)
    k, v = 256, 3000
    w = (torch.randn(v, k, device="cuda", generator=g) * 0.1).to(dtype)
    sets = [(torch.randn(n, k, device="cuda", generator=g).to(dtype), torch.randint(0, v, (n,), device="cuda", generator=g, dtype=torch.int32),
             torch.empty(n, device="cuda"), torch.empty(n, device="cuda")) for _ in range(2)]
    K().linear_logprobs(sets[0][0], w, *sets[0][1:])
    torch.cuda.synchronize()
    graphs = []
    for x, t, lp, lse in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            K().linear_logprobs(x, w, t, lp, lse)
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in sets]
    for x, t, lp, lse in sets:
        x.copy_(torch.randn(n, k, device="cuda", generator=g))
    torch.cuda.synchronize()
    for _ in range(10):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for x, t, lp, lse in sets:
        want_lp, want_lse = exact(x, w, t, None)
        tol_lse, tol_lp = tolerance(x, w, want_lse, want_lp, None, dtype == BF)
        assert ((lse.double() - want_lse).abs() <= tol_lse).all() and ((lp.double() - want_lp).abs() <= tol_lp).all()
