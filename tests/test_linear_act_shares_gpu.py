"""Products whose K a cluster of CTAs shares: parts sent into shared memory behind the ring and over it, calls that crowd one another so that a
cluster's CTAs begin apart, results that are the same bits each time."""
import pytest
import torch

from iian_b200.ops.cuda_backend import CudaKernels

pytestmark = pytest.mark.gpu
K = CudaKernels
BF = torch.bfloat16


def form(pair, bn, ks, rows=0):
    return int(pair) | bn << 1 | rows << 14 | ks << 16


# (rows, K, columns, form): parts of up to 80 KB lie behind the ring, larger ones over it; tiles enough for many clusters an SM, one behind the other
CASES = [(61, 256, 40000, form(0, 48, 3, 1)), (1, 512, 9000, form(0, 32, 6, 1)), (128, 1024, 8192, form(0, 128, 4, 1)), (128, 512, 16000, form(0, 256, 2)),
         (100, 2048, 6000, form(0, 64, 8)), (500, 1024, 5000, form(0, 256, 6)), (500, 1024, 5000, form(1, 96, 3)), (61, 4096, 4096, 0), (1, 1024, 4096, 0)]


@pytest.mark.parametrize("n,k,m,f", CASES)
def test_crowded_calls_give_the_same_bits(n, k, m, f):
    g = torch.Generator("cuda").manual_seed(n + m)
    x, w = torch.randn(n, k, device="cuda", generator=g).to(BF), (torch.randn(m, k, device="cuda", generator=g) * 0.05).to(BF)
    r = torch.randn(n, m, device="cuda", generator=g)
    alone = torch.empty(n, m, device="cuda")
    K().linear_act(x, w, alone, residual=r, form=f)
    torch.cuda.synchronize()
    # the same in 64 bits: 2^-23 of sum |x w| for each of K / 16 + 1 steps twice over, and 32 roundings of what is joined
    ref, total = x.double() @ w.double().t(), x.double().abs() @ w.double().abs().t()
    tol = total * (2 * (k / 16 + 1) * 2.0 ** -23) + 32 * 2.0 ** -24 * (total + ref.abs() + r.double().abs())
    assert ((alone.double() - ref - r.double()).abs() <= tol).all()
    streams, outs = [torch.cuda.Stream() for _ in range(3)], [[torch.full((n, m), float("nan"), device="cuda") for _ in range(4)] for _ in range(3)]
    torch.cuda.synchronize()
    for i in range(4):
        for s, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                K().linear_act(x, w, outs[s][i], residual=r, form=f)
    torch.cuda.synchronize()
    K().check_device_status()
    assert all(torch.equal(o, alone) for row in outs for o in row)
