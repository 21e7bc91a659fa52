"""Three operators that a pass over a prompt or a decoded step is made of, as measurable cases: each in its plain form (elementary torch
operations) and, with ``own`` set, as a call of this framework.

* ``route``: router logits -> the experts of each token and their weights (sigmoid or softmax scores, a correction for balance that
  decides the choice alone, groups of experts, renormalised weights).
* ``product``: ``residual + act(x W^T + bias)``, one rounding at the end.
* ``score``: log-probability of a given token per row under ``softmax(x W^T)`` over the vocabulary, and the row's log-sum-exp, without
  the logits.

Weights are N(0, 0.02) as a freshly initialised model's, rows N(0, 1) as norms leave them, the residual stream N(0, 2).  Everything
follows from the seed."""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
ACTIVATIONS = ("none", "silu", "gelu_tanh", "gelu", "relu", "relu2")
VOCAB = 151936


def listed():
    return [
        # one user's token: the smallest call there is, bound by its launch
        dict(name="route_one", kind="route", n=1, experts=64, groups=8, top_groups=4, top=5, score="sigmoid", correction=True),
        # a loaded server's decode step through many small experts
        dict(name="route_batch", kind="route", n=61, experts=256, groups=8, top_groups=4, top=8, score="sigmoid", correction=True),
        # a step of long prompts
        dict(name="route_prompt", kind="route", n=8192, experts=256, groups=8, top_groups=4, top=8, score="sigmoid", correction=True),
        # softmax scores, a group known by its best expert, no correction; an odd number of tokens
        dict(name="route_softmax", kind="route", n=2047, experts=160, groups=4, top_groups=2, top=6, score="softmax", correction=False),
        # a decoded token through a small model's first matrix
        dict(name="product_one", kind="product", n=1, k=1024, m=4096, act="gelu_tanh", bias=True, residual=False, dtype="bf16", out="bf16"),
        # a loaded decode step: the second matrix of a feed-forward, into the stream
        dict(name="product_batch", kind="product", n=61, k=12288, m=4096, act="none", bias=True, residual=True, dtype="bf16", out="f32"),
        # a portion of a prompt of odd length, a width that no tile divides
        dict(name="product_chunk", kind="product", n=517, k=2048, m=1416, act="silu", bias=True, residual=True, dtype="bf16", out="f32"),
        # a long prompt through a large model's first matrix
        dict(name="product_prompt", kind="product", n=2048, k=4096, m=12288, act="gelu", bias=True, residual=False, dtype="bf16", out="bf16"),
        # the true 32-bit path
        dict(name="product_f32", kind="product", n=301, k=1024, m=2048, act="relu2", bias=True, residual=True, dtype="f32", out="f32"),
        # one answer's last token
        dict(name="score_one", kind="score", n=1, k=1024, vocab=VOCAB, dtype="bf16", cap=0.0),
        # a few short answers
        dict(name="score_batch", kind="score", n=61, k=4096, vocab=VOCAB, dtype="bf16", cap=0.0),
        # a whole prompt
        dict(name="score_prompt", kind="score", n=2048, k=4096, vocab=VOCAB, dtype="bf16", cap=0.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["route", "product", "product", "score"])
    if kind == "route":
        groups = rng.choice([1, 2, 4, 8, 16])
        per = _log(rng, 4, 512 // groups)
        top_groups = rng.randint(1, groups)
        return dict(kind=kind, n=_log(rng, 1, 8192), experts=groups * per, groups=groups, top_groups=top_groups,
                    top=rng.randint(1, min(10, top_groups * per)), score=rng.choice(["sigmoid", "softmax"]), correction=rng.random() < 0.7)
    dtype = "bf16" if rng.random() < 0.8 else "f32"
    if kind == "product":
        n, k, m = _log(rng, 1, 4096), _log(rng, 128, 12288), _log(rng, 100, 12288)
        most = 2048 * 4096 * 12288 // (1 if dtype == "bf16" else 32)
        while n * k * m > most:
            n, k, m = max(1, n // 2), k * 4 // 5, m * 4 // 5
        residual = rng.random() < 0.5
        return dict(kind=kind, n=n, k=max(8, k // 8 * 8) if dtype == "bf16" else k, m=m, act=rng.choice(ACTIVATIONS), bias=rng.random() < 0.7,
                    residual=residual, dtype=dtype, out="f32" if residual or dtype == "f32" else "bf16")
    n, k, vocab = _log(rng, 1, 2048), max(8, _log(rng, 256, 4096) // 8 * 8), _log(rng, 1000, VOCAB)
    while dtype == "f32" and n * k * vocab > 64 * 4096 * VOCAB:
        n, vocab = max(1, n // 2), max(1000, vocab // 2)
    return dict(kind=kind, n=n, k=k, vocab=vocab, dtype=dtype, cap=30.0 if rng.random() < 0.3 else 0.0)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.float32):
        return torch.empty(*shape, device=DEV, dtype=torch.float32).normal_(0.0, std, generator=g).to(dtype)

    s = dict(case)
    n = case["n"]
    if case["kind"] == "route":
        e, top = case["experts"], case["top"]
        s.update(logits=normal(n, e, std=1.5), bias=normal(e, std=0.05) if case["correction"] else None,
                 ids=torch.empty(n, top, dtype=torch.int32, device=DEV), weights=torch.empty(n, top, device=DEV))
        return s
    k, dtype = case["k"], TYPES[case["dtype"]]
    s["x"] = normal(n, k, dtype=dtype)
    if case["kind"] == "product":
        m = case["m"]
        s.update(w=normal(m, k, std=0.02, dtype=dtype), b=normal(m, std=0.1) if case["bias"] else None,
                 r=normal(n, m, std=2.0) if case["residual"] else None, y=torch.empty(n, m, dtype=TYPES[case["out"]], device=DEV))
    else:
        s.update(w=normal(case["vocab"], k, std=0.02, dtype=dtype),
                 targets=torch.randint(0, case["vocab"], (n,), generator=g, device=DEV, dtype=torch.int32),
                 lp=torch.empty(n, device=DEV), lse=torch.empty(n, device=DEV))
    return s


GROUP_TOP = {"sigmoid": 2, "softmax": 1}        # how many of a group's largest scores make the group's
SCALE = 2.5


def run(s):
    if own:
        from iian_b200 import ops
        kernels = ops.kernels()
        if s["kind"] == "route":
            kernels.moe_route_grouped(s["logits"], s["top"], s["ids"], s["weights"], score=s["score"], correction=s["bias"], groups=s["groups"],
                                      top_groups=s["top_groups"], group_top=GROUP_TOP[s["score"]], renormalise=True, scale=SCALE)
            return s["ids"], s["weights"]
        if s["kind"] == "product":
            kernels.linear_act(s["x"], s["w"], s["y"], bias=s["b"], activation=s["act"], residual=s["r"])
            return s["y"]
        kernels.linear_logprobs(s["x"], s["w"], s["targets"], s["lp"], s["lse"], softcap=s["cap"] or None)
        return s["lp"], s["lse"]
    return {"route": plain_route, "product": plain_product, "score": plain_score}[s["kind"]](s)


def plain_route(s):
    # in 64 bits: two scores next to one another decide which expert is taken
    z = s["logits"].double()
    n, e = z.shape
    if s["score"] == "sigmoid":
        score = 1.0 / (1.0 + torch.exp(-z))
    else:
        p = torch.exp(z - z.amax(1, keepdim=True))
        score = p / p.sum(1, keepdim=True)
    choice = score if s["bias"] is None else score + s["bias"].double()
    by_group = choice.view(n, s["groups"], e // s["groups"])
    group_score = torch.sort(by_group, dim=2, descending=True).values[:, :, : GROUP_TOP[s["score"]]].sum(2)
    kept = torch.sort(group_score, dim=1, descending=True, stable=True).indices[:, : s["top_groups"]]
    open_ = torch.zeros(n, s["groups"], dtype=torch.bool, device=z.device).scatter_(1, kept, True)
    masked = by_group.masked_fill(~open_[:, :, None], -math.inf).view(n, e)
    ids = torch.sort(masked, dim=1, descending=True, stable=True).indices[:, : s["top"]]
    w = score.gather(1, ids)
    return ids.int(), (w / w.sum(1, keepdim=True) * SCALE).float()


def activate(y, act):
    if act == "silu":
        return y / (1.0 + torch.exp(-y))
    if act == "gelu_tanh":
        return 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))
    if act == "gelu":
        return 0.5 * y * (1.0 + torch.erf(y * math.sqrt(0.5)))
    if act == "relu":
        return torch.clamp(y, min=0.0)
    if act == "relu2":
        return torch.clamp(y, min=0.0) ** 2
    return y


def plain_product(s):
    y = s["x"].float() @ s["w"].float().t()
    if s["b"] is not None:
        y = y + s["b"]
    y = activate(y, s["act"])
    if s["r"] is not None:
        y = y + s["r"]
    return y.to(TYPES[s["out"]])


def plain_score(s):
    z = s["x"].float() @ s["w"].float().t()
    if s["cap"]:
        z = s["cap"] * torch.tanh(z / s["cap"])
    top = z.amax(1, keepdim=True)
    lse = top[:, 0] + torch.log(torch.exp(z - top).sum(1))
    return z.gather(1, s["targets"].long()[:, None])[:, 0] - lse, lse


def work(case):
    n = case["n"]
    if case["kind"] == "route":
        e = case["experts"]
        return {"bytes": 4 * n * e + (4 * e if case["correction"] else 0) + 8 * n * case["top"], "flops": 10 * n * e}
    k, size = case["k"], 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "product":
        m = case["m"]
        moved = size * (n * k + m * k) + (4 * m if case["bias"] else 0) + (4 * n * m if case["residual"] else 0)
        return {"bytes": moved + n * m * (2 if case["out"] == "bf16" else 4), "flops": 2 * n * m * k}
    v = case["vocab"]
    return {"bytes": size * (n * k + v * k) + 12 * n, "flops": 2 * n * v * k}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "route":
        z = s["logits"].double().cpu()
        n, e = z.shape
        score = torch.sigmoid(z) if case["score"] == "sigmoid" else torch.softmax(z, 1)
        choice = score + (s["bias"].double().cpu() if s["bias"] is not None else 0.0)
        per = e // case["groups"]
        best = choice.unfold(1, per, per).topk(GROUP_TOP[case["score"]], dim=2).values.sum(2)
        order = torch.argsort(-best, dim=1, stable=True)
        rank = torch.empty_like(order).scatter_(1, order, torch.arange(case["groups"]).expand(n, -1))
        shut = torch.repeat_interleave(rank >= case["top_groups"], per, dim=1)
        ids = torch.argsort(torch.where(shut, math.inf, -choice), dim=1, stable=True)[:, : case["top"]]
        w = torch.take_along_dim(score, ids, 1)
        return ids.int(), SCALE * w / w.sum(1, keepdim=True)
    x, w = s["x"].double(), s["w"]
    if case["kind"] == "product":
        y = torch.cat([torch.einsum("nk,mk->nm", x, part.double()) for part in w.split(4096)], 1)
        if case["bias"]:
            y += s["b"].double()
        f = torch.nn.functional
        y = {"none": lambda t: t, "silu": f.silu, "gelu": f.gelu, "gelu_tanh": lambda t: f.gelu(t, approximate="tanh"), "relu": f.relu,
             "relu2": lambda t: f.relu(t).square()}[case["act"]](y)
        return y + s["r"].double() if case["residual"] else y
    lse = torch.full((case["n"],), -math.inf, dtype=torch.float64, device=DEV)
    cap = case["cap"] or None
    for part in w.split(16384):
        z = torch.einsum("nk,vk->nv", x, part.double())
        z = cap * torch.tanh(z / cap) if cap else z
        lse = torch.logaddexp(lse, torch.logsumexp(z, 1))
    z = (x * w[s["targets"].long()].double()).sum(1)
    z = cap * torch.tanh(z / cap) if cap else z
    return z - lse, lse
