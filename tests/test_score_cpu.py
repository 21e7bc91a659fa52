"""Scoring given tokens, products with an epilogue and experts in groups, without a GPU: the engine's host side over the kernels' stand-in,
the parts' parameters, and what the kernel layer refuses before it looks for a device."""
import json
import math

import pytest
import torch

import plain_qwen3 as plain
import scored_model as sm
from helpers import random_tokens, write_tiny
from iian_b200 import EngineConfig, SchedulerConfig, ops
from iian_b200.cli.main import main
from iian_b200.config.spec import PartSpec
from iian_b200.engine.engine import Engine
from iian_b200.engine.model import Model
from iian_b200.engine.runner import StepEntry
from iian_b200.ops.cuda_backend import CudaKernels, KernelError
from iian_b200.parts.experts import RoutedExperts
from iian_b200.parts.mlp import PlainMLP

CPU = torch.device("cpu")


@pytest.fixture(scope="module")
def qwen(tmp_path_factory):
    d = write_tiny(tmp_path_factory.mktemp("m"), "B")
    cfg, w = plain.load_folder(d)
    with ops.use_kernels(sm.ScoredFakes()):
        model = Model.from_folder(d, "float32", "cpu")

    def want(tokens, start=1):
        lp = torch.log_softmax(plain.forward(cfg, w, tokens), 1)
        return [lp[i - 1, tokens[i]].item() for i in range(start, len(tokens))]
    return d, model, want


@pytest.fixture(scope="module")
def scored(tmp_path_factory):
    sm.register()
    d = sm.write(str(tmp_path_factory.mktemp("s")))
    with ops.use_kernels(sm.ScoredFakes()):
        model = Model.from_folder(d, "float32", "cpu")
    yield d, model
    sm.unregister()


def engine(model, **kw):
    sched = SchedulerConfig(max_num_batched_tokens=kw.pop("budget", 13), max_num_seqs=kw.pop("seqs", 4))
    return Engine(model, EngineConfig(dtype="float32", block_size=8, warmup=False, sched=sched, **kw))


def close(got, want, tol=2e-4):        # float32 through three or four layers of widths up to 96, on the CPU
    assert [len(g) for g in got] == [len(w) for w in want]
    for g, w in zip(got, want):
        assert all(abs(a - b) <= tol for a, b in zip(g, w))


@pytest.mark.parametrize("budget,seqs,tokens", [(1024, 4, 512), (13, 4, 512), (5, 1, 128), (16, 8, 128), (1, 2, 128)])
def test_scores_are_the_log_softmax(qwen, budget, seqs, tokens):
    _, model, want = qwen
    lists = [random_tokens(503, n, 40 + n) for n in (24, 1, 61, 2, 97, 8, 9)]
    with ops.use_kernels(sm.ScoredFakes()):
        eng = engine(model, kv_cache_tokens=tokens, max_model_len=112, budget=budget, seqs=seqs)
        close(eng.score(lists), [want(t) for t in lists])
        starts = [5, 1, 40, 1, 96, 8, 20]
        close(eng.score(lists, starts), [want(t, s) for t, s in zip(lists, starts)])
        assert eng.score([]) == [] and eng.score([[7]]) == [[]]
        assert eng.generate([lists[0]], max_tokens=3, temperature=0.0)           # the engine goes on as before
    eng.cache.check_invariants()
    assert all(p.num_free == p.num_blocks for p in eng.cache.pools)


def test_sequences_that_do_not_fit_together_wait_for_one_another(qwen):
    _, model, want = qwen
    lists = [random_tokens(503, 90, i) for i in range(3)]
    with ops.use_kernels(sm.ScoredFakes()):
        eng = engine(model, kv_cache_tokens=96, max_model_len=96, budget=50, seqs=3)
        close(eng.score(lists), [want(t) for t in lists])
    eng.cache.check_invariants()


def test_sequences_none_of_which_fits_beside_a_request(qwen):
    _, model, _ = qwen
    from iian_b200 import SamplingParams
    with ops.use_kernels(sm.ScoredFakes()):
        eng = engine(model, kv_cache_tokens=96, max_model_len=96, budget=16, seqs=4)
        req = eng.submit(random_tokens(503, 60, 1), SamplingParams(temperature=0.0, max_tokens=4))
        while not req.output_tokens:
            eng.step()
        for lists in ([random_tokens(503, 90, i) for i in range(3)], [random_tokens(503, 20, 5), random_tokens(503, 90, 6), random_tokens(503, 91, 7)]):
            with pytest.raises(RuntimeError, match="does not fit"):
                eng.score(lists)
        while not req.is_finished:
            eng.step()
    eng.cache.check_invariants()


def test_beside_requests_under_way(qwen):
    _, model, want = qwen
    prompt, tokens = random_tokens(503, 30, 1), random_tokens(503, 40, 2)
    with ops.use_kernels(sm.ScoredFakes()):
        eng = engine(model, kv_cache_tokens=160, max_model_len=96, budget=64)
        alone = eng.generate([prompt], max_tokens=6, temperature=0.0)
        from iian_b200 import SamplingParams
        req = eng.submit(prompt, SamplingParams(temperature=0.0, max_tokens=6))
        eng.step()
        close(eng.score([tokens]), [want(tokens)])
        while not req.is_finished:
            eng.step()
        assert [req.output_tokens] == alone
        # a request that holds all pages leaves none to score with
        held = eng.cache.new_request()
        assert eng.cache.allot_state(held) and eng.cache.allocate(held, 0, 150)
        with pytest.raises(RuntimeError, match="does not fit"):
            eng.score([tokens])
        eng.cache.free(held)
        close(eng.score([tokens]), [want(tokens)])


def test_what_score_refuses(qwen):
    _, model, _ = qwen
    with ops.use_kernels(sm.ScoredFakes()):
        eng = engine(model, kv_cache_tokens=128, max_model_len=64)
        for bad, why in (([[1, 503]], "out of range"), ([[1, -1]], "out of range"), ([[]], "empty"), ([[1] * 65], "max_model_len")):
            with pytest.raises(ValueError, match=why):
                eng.score(bad)
        with pytest.raises(ValueError, match="starts"):
            eng.score([[1, 2]], [1, 1])
        with pytest.raises(ValueError, match="nothing before"):
            eng.score([[1, 2]], [0])
        eng.start()
        with pytest.raises(RuntimeError, match="background"):
            eng.score([[1, 2]])
        eng.stop()
        rc = eng.cache.new_request()
        assert eng.cache.allot_state(rc) and eng.cache.allocate(rc, 0, 2)
        entry = StepEntry(rc, [1, 2], 0, [0])
        with pytest.raises(ValueError, match="wanted place"):
            eng.runner.score([entry], [[1, 2]])
        with pytest.raises(ValueError, match="vocabulary"):
            eng.runner.score([entry], [[503]])
        lp, lse = eng.runner.score([entry], [[-1]])
        assert lp.tolist() == [0.0] and math.isfinite(lse.item())
        eng.cache.free(rc)


def test_a_model_of_the_new_parts(scored):
    d, model = scored
    lists = [random_tokens(331, n, n) for n in (33, 7, 18)]
    with ops.use_kernels(sm.ScoredFakes()):
        eng = engine(model, kv_cache_tokens=256, max_model_len=128, budget=17)
        close(eng.score(lists), [sm.plain_scores(d, t) for t in lists], 5e-4)


def test_score_command(qwen, capsys, monkeypatch):
    d, model, want = qwen
    monkeypatch.setattr("iian_b200.engine.engine.Model.from_folder", lambda *a, **k: model)
    args = ["score", d, "--dtype", "float32", "--kv-cache-tokens", "512", "-c", "64", "--no-warmup", "-q"]
    with ops.use_kernels(sm.ScoredFakes()):
        assert main(args + ["-p", "5,17,3,99; 8 9 10", "--json"]) == 0
        rows = [json.loads(line) for line in capsys.readouterr().out.splitlines()]
        assert [r["tokens"] for r in rows] == [[5, 17, 3, 99], [8, 9, 10]]
        for r in rows:
            w = want(r["tokens"])
            close([r["logprobs"]], [w])
            assert abs(r["sum"] - sum(w)) < 1e-3 and abs(r["perplexity"] - math.exp(-sum(w) / len(w))) < 1e-2 * r["perplexity"]
        assert main(args + ["-p", "5,17,3", "--start", "2"]) == 0
        assert capsys.readouterr().out.startswith("1 tokens  log-probability")
        assert main(args) == 1 and main(args + ["-p", "5,600"]) == 1
    assert "iian score" in capsys.readouterr().err


@pytest.mark.parametrize("params,why", [({"activation": "tanh"}, "no kernel"), ({"activation": "xielu", "bias": True}, "no form with biases")])
def test_plain_mlp_parameters(params, why):
    with pytest.raises(ValueError, match=why):
        PlainMLP(PartSpec("plain_mlp", dict(hidden_size=8, intermediate_size=16, **params)), torch.float32, CPU)


def test_plain_mlp_tensors():
    p = PlainMLP(PartSpec("plain_mlp", {"hidden_size": 8, "intermediate_size": 16, "activation": "relu2", "bias": True}), torch.float32, CPU)
    assert set(p.tensors()) == {"up", "down", "up.b", "down.b"} and p.adds_residual
    p = PlainMLP(PartSpec("plain_mlp", {"hidden_size": 8, "intermediate_size": 16, "activation": "gelu", "names": ("a", "b", "c")}), torch.float32, CPU)
    assert set(p.tensors()) == {"a", "b"} and p.adds_residual
    p = PlainMLP(PartSpec("plain_mlp", {"hidden_size": 8, "intermediate_size": 16, "activation": "relu2"}), torch.float32, CPU)
    assert set(p.tensors()) == {"up", "down"} and not p.adds_residual           # as it was: product, activation kernel, product


BASE = dict(hidden_size=8, num_experts=12, top=3, intermediate_size=8, score="grouped", weight_on="output", groups=4, top_groups=2)


@pytest.mark.parametrize("change,why", [({"weight_on": "input"}, "on the output"), ({"groups": 5}, "groups"), ({"top_groups": 5}, "groups"),
                                        ({"top_groups": 0}, "groups"), ({"group_top": 3}, "best"), ({"top": 7}, "experts"),
                                        ({"score_function": "tanh"}, "score_function"), ({"identity_experts": 1}, "identity"),
                                        ({"num_experts": 1028, "groups": 4}, "1,024"), ({"num_experts": 66, "groups": 33}, "32 groups")])
def test_grouped_experts_parameters(change, why):
    with pytest.raises(ValueError, match=why):
        RoutedExperts(PartSpec("routed_experts", dict(BASE, **change)), torch.float32, CPU)


def test_grouped_experts_tensors():
    p = RoutedExperts(PartSpec("routed_experts", dict(BASE)), torch.float32, CPU)
    assert p.tensors()["correction"].shape == (12,) and "moe_groups" in p.kernel_libraries()
    p = RoutedExperts(PartSpec("routed_experts", dict(BASE, correction=False, weight_scale=2.0)), torch.float32, CPU)
    assert "correction" not in p.tensors()


# ---- refusals that need no device --------------------------------------------------------------------------------------------
def test_kernel_layer_refuses():
    k, f = CudaKernels(), torch.zeros
    i32 = torch.int32
    z, ids, w = f(3, 8), f(3, 2, dtype=i32), f(3, 2)
    for change in ({"score": "tanh"}, {"groups": 3}, {"groups": 0}, {"top_groups": 3, "groups": 2}, {"top_groups": 0}, {"group_top": 0},
                   {"groups": 8, "top_groups": 1}, {"correction": f(7)}):
        with pytest.raises(KernelError):
            k.moe_route_grouped(z, 2, ids, w, **change)
    for a in ((z.double(), 2, ids, w), (z, 3, ids, w), (z, 2, ids[:2], w)):
        with pytest.raises(KernelError):
            k.moe_route_grouped(*a)
    with pytest.raises(KernelError, match="CUDA only"):
        k.moe_route_grouped(z, 2, ids, w)
    x, m, out = f(3, 8), f(5, 8), f(3, 5)
    for a in ((f(3, 7), m, out), (x, f(5), out), (x.half(), m, out), (x, m.half(), out)):
        with pytest.raises(KernelError):
            k.linear_act(*a)
        with pytest.raises(KernelError):
            k.linear_logprobs(a[0], a[1], f(3, dtype=i32), f(3), f(3))
    with pytest.raises(KernelError, match="CUDA only"):
        k.linear_act(x, m, out)
    with pytest.raises(KernelError, match="CUDA only"):
        k.linear_logprobs(x, m, f(3, dtype=i32), f(3), f(3))
