"""The choice of experts in groups against the same in float64: whole numbers are equal, ties, saturated scores, masked logits and what is
no number among them."""
import pytest
import torch

from iian_b200.ops.cuda_backend import CudaKernels, KernelError
from scored_model import choose

pytestmark = pytest.mark.gpu
K = CudaKernels


def check(z, correction, score, groups, top_groups, group_top, top, renormalise=True, scale=2.5):
    n = z.shape[0]
    ids = torch.full((n + 1, top), -7, device="cuda", dtype=torch.int32)
    w = torch.full((n + 1, top), 7.0, device="cuda")
    K().moe_route_grouped(z, top, ids[:n], w[:n], score=score, correction=correction, groups=groups, top_groups=top_groups, group_top=group_top,
                          renormalise=renormalise, scale=scale)
    want, wt = choose(z, correction, score, groups, top_groups, group_top, top, renormalise, scale)
    assert torch.equal(ids[:n].long(), want)
    # an exponential (2 units in the last place and its argument's rounding, up to 30 of 2^-24), a reciprocal or a sum of up to 1,024, the sum of
    # the chosen, two products
    assert ((w[:n].double() - wt).abs() <= 6e-6 * wt.abs() + 1e-37).all()
    assert (ids[n] == -7).all() and (w[n] == 7.0).all()


SHAPES = [(64, 8, 4, 2, 5), (256, 8, 4, 2, 8), (256, 1, 1, 1, 8), (160, 4, 2, 1, 6), (60, 12, 5, 2, 7), (512, 16, 3, 2, 10), (1024, 1, 1, 2, 32), (1020, 17, 9, 2, 20),
          (7, 7, 3, 2, 3), (8, 2, 1, 2, 4), (1, 1, 1, 2, 1), (33, 3, 3, 1, 12), (992, 31, 4, 2, 9), (640, 2, 2, 2, 31), (96, 32, 32, 1, 5), (40, 2, 1, 2, 20)]


@pytest.mark.parametrize("E,groups,top_groups,group_top,top", SHAPES)
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("corrected", [False, True])
def test_choice(E, groups, top_groups, group_top, top, score, corrected):
    g = torch.Generator("cuda").manual_seed(E + top)
    for n, std in ((1, 1.5), (61, 1.5), (700, 0.3), (300, 5.0)):
        z = torch.randn(n, E + 5, device="cuda", generator=g)[:, 2:2 + E] * std          # a slice of wider rows, not aligned
        c = torch.randn(E, device="cuda", generator=g) * 0.05 if corrected else None
        check(z, c, score, groups, top_groups, group_top, top)
        check(z.contiguous(), c, score, groups, top_groups, group_top, top, renormalise=False, scale=1.0)


@pytest.mark.parametrize("E,groups,top_groups,group_top,top", SHAPES)
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_ties_go_to_the_lower_index(E, groups, top_groups, group_top, top, score):
    g = torch.Generator("cuda").manual_seed(E)
    z = torch.randint(-3, 4, (300, E), device="cuda", generator=g).float() / 2              # seven different logits
    check(z, None, score, groups, top_groups, group_top, top)
    check(torch.zeros(3, E, device="cuda"), None, score, groups, top_groups, group_top, top)
    c = torch.randint(0, 2, (E,), device="cuda", generator=g).float() / 4
    check(z, c, score, groups, top_groups, group_top, top)
    check(z.to(torch.bfloat16).float() + 2.0 ** -20 * torch.randn(300, E, device="cuda", generator=g), c, score, groups, top_groups, group_top, top)


@pytest.mark.parametrize("E,groups,top_groups,top", [(64, 8, 4, 6), (256, 1, 1, 8), (1020, 17, 5, 10)])
def test_neighbours_that_32_bits_cannot_tell_apart(E, groups, top_groups, top):
    """Sigmoids near 1 of logits between 9 and 18, whose float32 values are the same for many of them."""
    g = torch.Generator("cuda").manual_seed(E)
    z = torch.rand(200, E, device="cuda", generator=g) * 9 + 9
    check(z, None, "sigmoid", groups, top_groups, 2, top)
    check(z, torch.full((E,), -0.5, device="cuda"), "sigmoid", groups, top_groups, 2, top)
    check(-z, torch.full((E,), 0.5, device="cuda"), "sigmoid", groups, top_groups, 2, top)
    check(z * 3, None, "softmax", groups, top_groups, 2, top)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_masked_logits(score):
    E, groups = 64, 8
    g = torch.Generator("cuda").manual_seed(2)
    z = torch.randn(8, E, device="cuda", generator=g)
    z[1, :40] = float("-inf")                                          # whole groups
    z[2] = float("-inf")                                               # nothing is left: the first experts, which weigh nothing
    z[3] = torch.finfo(torch.float32).min
    z[4, 1:] = float("-inf")
    z[5, ::2] = torch.finfo(torch.float32).min
    z[6] = 80.0
    c = torch.randn(E, device="cuda", generator=g) * 0.1
    for corr in (None, c):
        check(z, corr, score, groups, 4, 2, 6)
        check(z, corr, score, 1, 1, 1, 6)
    ids, w = torch.empty(8, 6, device="cuda", dtype=torch.int32), torch.empty(8, 6, device="cuda")
    K().moe_route_grouped(z, 6, ids, w, score=score, groups=groups, top_groups=4)
    assert ids[2].tolist() == [0, 1, 2, 3, 4, 5] and (w[2] == 0).all()
    minus = torch.zeros(E, device="cuda")
    minus[:56] = float("-inf")                                         # experts that may not be chosen
    K().moe_route_grouped(z[:1], 6, ids[:1], w[:1], score=score, correction=minus, groups=1, top_groups=1)
    assert (ids[0] >= 56).all() and len(set(ids[0].tolist())) == 6


def test_what_is_no_number_is_chosen_last():
    z = torch.randn(4, 32, device="cuda", generator=torch.Generator("cuda").manual_seed(4))
    z[0, 3] = float("nan")
    z[1, :30] = float("nan")
    z[2, 9] = float("inf")
    ids, w = torch.empty(4, 4, device="cuda", dtype=torch.int32), torch.empty(4, 4, device="cuda")
    K().moe_route_grouped(z, 4, ids, w, score="sigmoid", renormalise=False)
    assert 3 not in ids[0].tolist() and torch.isfinite(w[0]).all()
    assert set(ids[1].tolist()) == {30, 31, 0, 1} and torch.isnan(w[1, 2:]).all() and torch.isfinite(w[1, :2]).all()
    assert ids[2, 0] == 9 and w[2, 0] == 1.0
    for score in ("sigmoid", "softmax"):                               # whatever stands there, four different experts come back
        K().moe_route_grouped(torch.full((1, 32), float("nan"), device="cuda"), 4, ids[:1], w[:1], score=score, groups=4, top_groups=2)
        assert len(set(ids[0].tolist())) == 4


def test_many_tokens_and_no_tokens():
    g = torch.Generator("cuda").manual_seed(9)
    check(torch.randn(20001, 128, device="cuda", generator=g), torch.randn(128, device="cuda", generator=g) * 0.02, "sigmoid", 4, 2, 2, 8)
    K().moe_route_grouped(torch.empty(0, 64, device="cuda"), 4, torch.empty(0, 4, device="cuda", dtype=torch.int32), torch.empty(0, 4, device="cuda"))


def test_refusals():
    f = lambda *s: torch.zeros(*s, device="cuda")                                                  # noqa: E731
    i = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.int32)                               # noqa: E731
    k = K()
    for E, top, kw in ((1025, 4, {}), (66, 4, {"groups": 33}), (64, 33, {})):
        with pytest.raises(KernelError):
            k.moe_route_grouped(f(3, E), top, i(3, top), f(3, top), **kw)
    for a, kw in (((f(3, 8), 2, f(3, 2), f(3, 2)), {}), ((f(3, 8), 2, i(3, 2), i(3, 2)), {}), ((f(8, 3).t(), 2, i(3, 2), f(3, 2)), {}),
                  ((f(3, 8), 2, i(3, 2), f(3, 2)), {"correction": torch.zeros(8)}), ((f(3, 8), 2, torch.zeros(3, 2, dtype=torch.int32), f(3, 2)), {}),
                  ((f(3, 8), 2, i(2, 3).t(), f(3, 2)), {})):
        with pytest.raises(KernelError):
            k.moe_route_grouped(*a, **kw)


def test_captured_and_replayed():
    g = torch.Generator("cuda").manual_seed(1)
    z, c = torch.randn(40, 128, device="cuda", generator=g), torch.randn(128, device="cuda", generator=g) * 0.05
    ids, w = torch.empty(40, 6, device="cuda", dtype=torch.int32), torch.empty(40, 6, device="cuda")
    run = lambda: K().moe_route_grouped(z, 6, ids, w, correction=c, groups=4, top_groups=2)         # noqa: E731
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    z.normal_(generator=g)
    graph.replay()
    want, wt = choose(z, c, "sigmoid", 4, 2, 2, 6)
    assert torch.equal(ids.long(), want) and ((w.double() - wt).abs() <= 6e-6 * wt).all()
