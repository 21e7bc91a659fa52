"""Scores in 32 bits are the same bits however the rows are cut: alone, beside others, in another order, as rows of a wider matrix, in portions
of the engine's.  (The logits of the 32-bit path are.)"""
import pytest
import torch

import iian_b200.ops.cuda_backend as backend
from helpers import TINY, random_tokens, write_tiny
from iian_b200 import EngineConfig, SchedulerConfig
from iian_b200.engine.engine import Engine
from iian_b200.engine.model import Model
from iian_b200.ops.cuda_backend import CudaKernels

pytestmark = pytest.mark.gpu
K = CudaKernels
F32, BF = torch.float32, torch.bfloat16


def scores(x, w, t, cap):
    lp, lse = torch.empty(x.shape[0], device="cuda"), torch.empty(x.shape[0], device="cuda")
    K().linear_logprobs(x, w, t, lp, lse, softcap=cap)
    return lp, lse


@pytest.mark.parametrize("k,v", [(64, 331), (1024, 9003), (515, 5003), (2776, 4097), (700, 2048), (4096, 2500), (1, 5000)])
@pytest.mark.parametrize("cap", [None, 20.0])
def test_rows_have_the_same_bits_in_any_batch(k, v, cap, monkeypatch):
    g = torch.Generator("cuda").manual_seed(k + v)
    n = 700
    x, w = torch.randn(n, k, device="cuda", generator=g), torch.randn(v, k, device="cuda", generator=g) * 0.05
    t = torch.randint(0, v, (n,), device="cuda", generator=g, dtype=torch.int32)
    whole = scores(x, w, t, cap)
    want = torch.logsumexp(x.double() @ w.double().t() if cap is None else cap * torch.tanh(x.double() @ w.double().t() / cap), 1)
    assert ((whole[1].double() - want).abs() <= 1e-4).all()          # (its accuracy is held to elsewhere)
    for first, m in ((0, 1), (3, 2), (5, 7), (12, 17), (40, 61), (100, 127), (100, 128), (150, 500)):
        wide, off = torch.empty(m, k + 3, device="cuda"), torch.empty(m * k + 1, device="cuda")
        wide[:, 1:1 + k] = x[first: first + m]
        off[1:] = x[first: first + m].reshape(-1)
        for rows in (x[first: first + m], wide[:, 1:1 + k], off[1:].view(m, k)):
            got = scores(rows, w, t[first: first + m].contiguous(), cap)
            assert torch.equal(got[0], whole[0][first: first + m]) and torch.equal(got[1], whole[1][first: first + m])
    monkeypatch.setattr(backend.CudaKernels, "SCORE_ROWS", 90)
    monkeypatch.setattr(backend.CudaKernels, "SCORE_PIECE", 1 << 12)
    got = scores(x, w, t, cap)
    assert torch.equal(got[0], whole[0]) and torch.equal(got[1], whole[1])


@pytest.mark.parametrize("dtype,wdtype,k", [(BF, BF, 67), (BF, F32, 64), (F32, BF, 64)])
def test_mixed_types_too(dtype, wdtype, k):
    g = torch.Generator("cuda").manual_seed(k)
    x, w = torch.randn(200, k, device="cuda", generator=g).to(dtype), (torch.randn(5003, k, device="cuda", generator=g) * 0.1).to(wdtype)
    t = torch.randint(0, 5003, (200,), device="cuda", generator=g, dtype=torch.int32)
    whole = scores(x, w, t, None)
    for first, m in ((0, 1), (7, 20), (20, 150)):
        got = scores(x[first: first + m], w, t[first: first + m].contiguous(), None)
        assert torch.equal(got[0], whole[0][first: first + m]) and torch.equal(got[1], whole[1][first: first + m])


def test_a_logit_of_a_score_is_the_head_s():
    """With one token in the vocabulary's place of interest far above the rest, the log-sum-exp is its logit, the one that ``linear`` gives."""
    g = torch.Generator("cuda").manual_seed(9)
    x, w = torch.randn(40, 256, device="cuda", generator=g), torch.randn(3000, 256, device="cuda", generator=g) * 1e-3
    w[1234] = torch.randn(256, device="cuda", generator=g) * 30
    z = torch.empty(40, 3000, device="cuda")
    K().linear(x, w, z)
    rows = (z[:, 1234] > 200).nonzero()[:, 0]
    assert rows.numel() >= 5
    for m in (1, 5, rows.numel()):
        some = rows[:m]
        _, lse = scores(x[some], w, torch.zeros(m, device="cuda", dtype=torch.int32), None)
        assert torch.equal(lse, z[some, 1234])


@pytest.mark.parametrize("name", ["B", "D"])
def test_the_engine_s_portions(tmp_path, name):
    d = write_tiny(tmp_path, name)
    lists = [random_tokens(TINY[name]["vocab_size"], n, n) for n in (200, 2, 133, 61, 7)]
    got = []
    for budget, seqs in ((1024, 4), (29, 4), (150, 1)):
        sched = SchedulerConfig(max_num_batched_tokens=budget, max_num_seqs=seqs)
        eng = Engine(Model.from_folder(d, "float32"), EngineConfig(dtype="float32", block_size=16, warmup=False, sched=sched, kv_cache_tokens=1024, max_model_len=256))
        got.append(eng.score(lists))
    assert got[0] == got[1] == got[2]
