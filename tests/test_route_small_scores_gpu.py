"""Weights of experts whose scores are small: they are what the definition says however far below 1 the chosen scores lie, whichever way a
token takes through the kernel."""
import pytest
import torch

from iian_b200.ops.cuda_backend import CudaKernels
from scored_model import choose

pytestmark = pytest.mark.gpu
K = CudaKernels
SHAPES = [(64, 8, 4, 2, 5), (256, 8, 4, 2, 8), (256, 1, 1, 1, 8), (160, 4, 2, 1, 6), (1024, 1, 1, 2, 32), (12, 4, 2, 2, 6), (40, 2, 1, 2, 20)]


def check(z, correction, score, groups, top_groups, group_top, top, renormalise=True, scale=2.5, far=0.0):
    """A chosen score: an exponential (2 units in the last place, 4 of 2^-24), a sum and a quotient; their sum 5 roundings for up to 32 of them;
    a quotient and a product: 2 (4 + 2) + 5 + 2 of 2^-24.  A softmax's exponent is a difference of float32, off by 2^-24 of its own size
    (``far``) in the score and in the sum; where it is not divided by the chosen ones its own sum counts too: 1,024 terms added in 37 steps,
    with exponentials of 3 units."""
    n = z.shape[0]
    ids, w = torch.empty(n, top, device="cuda", dtype=torch.int32), torch.empty(n, top, device="cuda")
    K().moe_route_grouped(z, top, ids, w, score=score, correction=correction, groups=groups, top_groups=top_groups, group_top=group_top,
                          renormalise=renormalise, scale=scale)
    want, wt = choose(z, correction, score, groups, top_groups, group_top, top, renormalise, scale)
    assert torch.equal(ids.long(), want)
    off = 19 + 2 * far + (0 if renormalise else 43)
    assert ((w.double() - wt).abs() <= off * 2.0 ** -24 * wt + 1e-37).all()
    if renormalise:
        assert ((w.double().sum(1) - scale).abs() <= scale * 1e-5).all()


@pytest.mark.parametrize("E,groups,top_groups,group_top,top", SHAPES)
@pytest.mark.parametrize("low,high", [(-40, -1), (-87, -60), (-89, -86), (-104, -88), (-130, -60), (-100, -100), (-300, -300), (-300, -290), (-700, -90)])
def test_sigmoids(E, groups, top_groups, group_top, top, low, high):
    g = torch.Generator("cuda").manual_seed(E + top)
    for n in (1, 33, 400):
        z = torch.rand(n, E, device="cuda", generator=g) * (high - low) + low
        c = torch.randperm(E, device="cuda", generator=g).float() / 64 - 1          # far apart: no two are near
        for correction in (c, c * 0.0, None, -c * 1e-3):
            check(z, correction, "sigmoid", groups, top_groups, group_top, top)
            check(z, correction, "sigmoid", groups, top_groups, group_top, top, renormalise=False, scale=1.0)


@pytest.mark.parametrize("E,groups,top_groups,group_top,top", SHAPES)
@pytest.mark.parametrize("below", [20, 80, 90, 110, 600])
def test_softmax_scores_far_below_the_largest(E, groups, top_groups, group_top, top, below):
    """The largest logits are shut by their corrections; those that are chosen lie ``below`` them."""
    g = torch.Generator("cuda").manual_seed(E + below)
    per = E // groups
    for n in (1, 33, 400):
        z = torch.randn(n, E, device="cuda", generator=g)
        c = 1 + torch.randperm(E, device="cuda", generator=g).float() / 64
        z[:, ::per] += below                                         # one of each group
        c[::per] = -50.0
        if top <= top_groups * (per - 1):
            check(z, c, "softmax", groups, top_groups, group_top, top, far=below + 10)
            c[::per] = float("-inf")
            check(z, c, "softmax", groups, top_groups, group_top, top, far=below + 10)


def test_some_chosen_scores_are_small_and_some_are_not():
    E, top = 32, 6
    z = torch.full((1, E), -3.0, device="cuda")
    z[0, :top] = torch.tensor([-69.0, -92.0, -99.0, -80.0, -101.0, -88.5], device="cuda")
    c = torch.zeros(E, device="cuda")
    c[:top] = torch.arange(top, 0, -1, device="cuda").float() * 2
    check(z, c, "sigmoid", 1, 1, 2, top)
    z[0, 0] = float("-inf")                                          # a score of 0 among them stays 0
    check(z, c, "sigmoid", 1, 1, 2, top)
    z[0, 1:top] = float("-inf")
    ids, w = torch.empty(1, top, device="cuda", dtype=torch.int32), torch.empty(1, top, device="cuda")
    K().moe_route_grouped(z, top, ids, w, correction=c)
    assert (w == 0).all() and ids[0].tolist() == list(range(top))
