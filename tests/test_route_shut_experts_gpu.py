"""Experts shut by a correction of minus infinity: a group that has fewer left than its score is made of has the score minus infinity, wherever
in the group they lie."""
import pytest
import torch

from iian_b200.ops.cuda_backend import CudaKernels
from scored_model import choose

pytestmark = pytest.mark.gpu
K = CudaKernels
SHAPES = [(160, 32, 5, 19), (256, 8, 4, 8), (64, 8, 4, 5), (64, 16, 7, 12), (1024, 4, 2, 20), (512, 8, 3, 8), (12, 4, 2, 3), (1020, 17, 9, 20), (40, 5, 2, 9)]


def check(z, c, score, groups, top_groups, top, renormalise):
    n = z.shape[0]
    ids, w = torch.empty(n, top, device="cuda", dtype=torch.int32), torch.empty(n, top, device="cuda")
    K().moe_route_grouped(z, top, ids, w, score=score, correction=c, groups=groups, top_groups=top_groups, group_top=2, renormalise=renormalise, scale=2.5)
    want, wt = choose(z, c, score, groups, top_groups, 2, top, renormalise, 2.5)
    assert torch.equal(ids.long(), want)
    assert ((w.double() - wt).abs() <= 6e-6 * wt + 1e-37).all()         # logits of ordinary size: an exponential with its argument's rounding, sums, quotients


@pytest.mark.parametrize("E,groups,top_groups,top", SHAPES)
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("left", [0, 1, 2])
def test_groups_with_few_experts_left(E, groups, top_groups, top, score, left):
    g = torch.Generator("cuda").manual_seed(E + left)
    per = E // groups
    for place in range(per if per <= 16 else 5):
        z = torch.randn(200, E, device="cuda", generator=g) * 2
        c = torch.randn(E, device="cuda", generator=g) * 0.1
        for shut in (groups // 2, groups - 1, 0):
            keep = [(shut * per + (place + 3 * j) % per) for j in range(min(left, per))]
            saved = c[keep].clone()
            c[shut * per: (shut + 1) * per] = float("-inf")
            c[keep] = saved + 5                                     # the best of all, were the group open
        check(z, c, score, groups, top_groups, top, True)
        check(z, c, score, groups, top_groups, top, False)
        z[::3, :per] = float("-inf")
        check(z, c, score, groups, top_groups, top, True)


@pytest.mark.parametrize("E,groups,top_groups,top", SHAPES)
def test_experts_shut_at_random(E, groups, top_groups, top):
    g = torch.Generator("cuda").manual_seed(E)
    for share in (0.1, 0.5, 0.9):
        c = torch.randn(E, device="cuda", generator=g) * 0.1
        c[torch.rand(E, device="cuda", generator=g) < share] = float("-inf")
        z = torch.randn(200, E, device="cuda", generator=g)
        for score in ("sigmoid", "softmax"):
            check(z, c, score, groups, top_groups, top, True)
