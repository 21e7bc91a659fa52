"""Scoring through the engine on the device: against the plain implementation in 32 bits, against the log-softmax of the same step's logits
in bfloat16; a model made of products with epilogues, experts in groups and a capped head; decoded, captured and generated beside it."""
import json
import subprocess
import sys

import pytest
import torch

import plain_qwen3 as plain
import scored_model as sm
from helpers import TINY, random_tokens, write_tiny
from iian_b200 import EngineConfig, SchedulerConfig, ops
from iian_b200.engine.engine import Engine
from iian_b200.engine.model import Model
from iian_b200.engine.replay import TraceReplayer

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def scored(tmp_path_factory):
    sm.register()
    yield sm.write(str(tmp_path_factory.mktemp("s")))
    sm.unregister()


def engine(model, **kw):
    sched = SchedulerConfig(max_num_batched_tokens=kw.pop("budget", 1024), max_num_seqs=kw.pop("seqs", 4))
    return Engine(model, EngineConfig(dtype=kw.pop("dtype"), block_size=16, warmup=False, sched=sched, **kw))


def close(got, want, tol):
    assert [len(g) for g in got] == [len(w) for w in want]
    worst = max(abs(a - b) for g, w in zip(got, want) for a, b in zip(g, w))
    assert worst <= tol, worst


def by_logits(d, dtype, tokens):
    """The same from a step's logits: the whole sequence but its last token at once, as one portion."""
    r = TraceReplayer.from_folder(d, dtype, 256, native=False)
    logits = r.run_step({"step": 0, "entries": [{"id": "a", "tokens": tokens[:-1], "want": list(range(len(tokens) - 1))}], "end": ["a"]})
    lp = torch.log_softmax(logits.double(), 1)
    return [lp[i, t].item() for i, t in enumerate(tokens[1:])]


@pytest.mark.parametrize("name", ["B", "D"])
@pytest.mark.parametrize("budget", [1024, 29])
def test_float32_against_the_plain_implementation(tmp_path, name, budget):
    d = write_tiny(tmp_path, name)
    cfg, w = plain.load_folder(d)
    lists = [random_tokens(TINY[name]["vocab_size"], n, n) for n in (90, 2, 33, 61, 7)]
    want = []
    for t in lists:
        lp = torch.log_softmax(plain.forward(cfg, w, t), 1)
        want.append([lp[i - 1, t[i]].item() for i in range(1, len(t))])
    eng = engine(Model.from_folder(d, "float32"), dtype="float32", kv_cache_tokens=512, max_model_len=128, budget=budget)
    before = eng.generate([lists[0]], max_tokens=5, temperature=0.0)
    close(eng.score(lists), want, 2e-4)             # the logits are held to 1e-4 by the replays in 32 bits; a difference of two
    close(eng.score(lists, [80, 1, 10, 61, 7]), [w[s - 1:] for w, s in zip(want, [80, 1, 10, 61, 7])], 2e-4)
    assert eng.generate([lists[0]], max_tokens=5, temperature=0.0) == before
    assert all(p.num_free == p.num_blocks for p in eng.cache.pools)


@pytest.mark.parametrize("name", ["D", "E"])
def test_bfloat16_against_the_logits_of_the_same_step(tmp_path, name):
    d = write_tiny(tmp_path, name, torch.bfloat16)
    eng = engine(Model.from_folder(d, "bfloat16"), dtype="bfloat16", kv_cache_tokens=512, max_model_len=256)
    for n in (2, 40, 200):
        t = random_tokens(TINY[name]["vocab_size"], n, n)
        # the rows that the head reads are the same; its logits are float32 sums of up to 256 products in another order, of size 1 or so
        close(eng.score([t]), [by_logits(d, "bfloat16", t)], 1e-4)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_model_of_the_new_parts(scored, dtype):
    eng = engine(Model.from_folder(scored, dtype), dtype=dtype, kv_cache_tokens=512, max_model_len=256)
    lists = [random_tokens(331, n, n) for n in (150, 33, 7)]
    if dtype == "float32":
        close(eng.score(lists), [sm.plain_scores(scored, t) for t in lists], 1e-3)
    for t in lists:
        close(eng.score([t]), [by_logits(scored, dtype, t)], 1e-4)
    # decoding through the same parts, from captured graphs and eagerly: the same tokens
    graphs = eng.generate(lists, max_tokens=12, temperature=0.0)
    eager = engine(Model.from_folder(scored, dtype), dtype=dtype, kv_cache_tokens=512, max_model_len=256, cuda_graphs=False)
    assert graphs == eager.generate(lists, max_tokens=12, temperature=0.0)
    # what greedy decoding picked is the likeliest token: no other continuation of one token scores above it (float32: bits may differ by a hair)
    if dtype == "float32":
        head = lists[2]
        best = eng.score([head + graphs[2][:1]], [len(head)])[0][0]
        others = eng.score([head + [t] for t in range(0, 331, 7)], [len(head)] * len(range(0, 331, 7)))
        assert all(o[0] <= best + 1e-4 for o in others)


def test_score_goes_through_the_kernels(scored):
    from iian_b200.ops import cuda_backend
    eng = engine(Model.from_folder(scored, "bfloat16"), dtype="bfloat16", kv_cache_tokens=256, max_model_len=128)
    before = dict(cuda_backend.LAUNCHES_BY_ENTRY)
    eng.score([random_tokens(331, 40, 1)])
    ran = {k for k, v in cuda_backend.LAUNCHES_BY_ENTRY.items() if v > before.get(k, 0)}
    assert {"linear_logprobs", "linear_act", "moe_route_grouped"} <= ran


def test_command(tmp_path):
    d = write_tiny(tmp_path, "B")
    out = subprocess.run([sys.executable, "-m", "iian_b200", "score", d, "-p", "5,17,3,99,4", "--dtype", "float32", "-c", "64", "--json", "-q"],
                         capture_output=True, text=True, timeout=240)
    assert out.returncode == 0, out.stderr
    row = json.loads(out.stdout.splitlines()[-1])
    cfg, w = plain.load_folder(d)
    lp = torch.log_softmax(plain.forward(cfg, w, row["tokens"]), 1)
    close([row["logprobs"]], [[lp[i, t].item() for i, t in enumerate(row["tokens"][1:])]], 2e-4)
