"""A small architecture of the tests' own made of the framework's parts: feed-forwards of two products with bias and activation in their
epilogues (one that adds into the stream itself, one beside its mixer), experts in groups with a shared one, a capped head; the same model
written out in float64; and the kernels' stand-in on the CPU for what it needs."""
import math

import torch

import plain_qwen3 as plain
from fake_kernels import FakeKernels
from iian_b200.config.registry import Architecture, get_architecture, register_architecture, unregister_architecture
from iian_b200.config.spec import LayerCall, LayerSpec, ModelSpec, PartSpec

CFG = {"architectures": ["ScoredForCausalLM"], "vocab_size": 331, "hidden_size": 64, "heads": 4, "kv_heads": 2, "head_dim": 16, "ffn": 96,
       "eps": 1e-5, "theta": 10000.0, "max_position": 256, "experts": 12, "groups": 4, "top_groups": 2, "top": 3, "expert_ffn": 32,
       "shared_ffn": 48, "score_function": "sigmoid", "softcap": 20.0}

ACTIVATIONS = {"none": lambda t: t, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu,
               "gelu_tanh": lambda t: torch.nn.functional.gelu(t, approximate="tanh"), "relu2": lambda t: torch.relu(t).square()}


def choose(z, correction, score, groups, top_groups, group_top, top, renormalise=True, scale=1.0):
    """The choice of experts in 64 bits: (ids [N, top], weights [N, top])."""
    n, e = z.shape
    z = z.double()
    s = torch.sigmoid(z) if score == "sigmoid" else torch.softmax(z, 1)
    s = torch.where(torch.isinf(z).all(1, keepdim=True) & (z < 0), 0.0, s) if score == "softmax" else s
    c = s if correction is None else s + correction.double()
    by_group = torch.sort(c.view(n, groups, e // groups), dim=2, descending=True).values[:, :, :group_top].sum(2)
    kept = torch.sort(by_group, dim=1, descending=True, stable=True).indices[:, :top_groups]
    open_ = torch.zeros(n, groups, dtype=torch.bool, device=z.device).scatter_(1, kept, True).repeat_interleave(e // groups, 1)
    # two keys: outputs of the groups taken first, then by c
    order = torch.sort(c, dim=1, descending=True, stable=True).indices
    order = order.gather(1, torch.sort(open_.gather(1, order).int(), dim=1, descending=True, stable=True).indices)
    ids = order[:, :top]
    w = s.gather(1, ids)
    if renormalise:
        total = w.sum(1, keepdim=True)
        w = torch.where(total == 0, 0.0, w / total)
    return ids, w * scale


class ScoredFakes(FakeKernels):
    def linear_act(self, x, w, out, bias=None, activation="none", residual=None, form=0):
        y = x.float() @ w.float().t()
        y = ACTIVATIONS[activation](y + bias if bias is not None else y)
        out.copy_((y + residual.float() if residual is not None else y).to(out.dtype))

    def linear_logprobs(self, x, w, targets, logprobs, lse, softcap=None, form=0):
        z = x.float() @ w.float().t()
        z = softcap * torch.tanh(z / softcap) if softcap else z
        lse.copy_(torch.logsumexp(z, 1))
        t = targets.long()
        logprobs.copy_(torch.where(t < 0, 0.0, z.gather(1, t.clamp(min=0)[:, None])[:, 0] - lse))

    def moe_route_grouped(self, logits, top, ids, weights, *, score="sigmoid", correction=None, groups=1, top_groups=1, group_top=2,
                          renormalise=True, scale=1.0):
        i, w = choose(logits, correction, score, groups, top_groups, group_top, top, renormalise, scale)
        ids.copy_(i)
        weights.copy_(w)


class ScoredArch(Architecture):
    name = "ScoredForCausalLM"

    def load_config(self, raw):
        return dict(raw)

    def config_to_dict(self, c):
        return dict(c)

    def build_spec(self, c):
        h = c["hidden_size"]
        norm = PartSpec("rms_norm", {"size": h, "eps": c["eps"]})
        attn = PartSpec("attention", {"hidden_size": h, "num_heads": c["heads"], "num_kv_heads": c["kv_heads"], "head_dim": c["head_dim"],
                                      "scale": 1 / math.sqrt(c["head_dim"]), "qk_norm": False, "window": None,
                                      "position": PartSpec("rotary", {"dim": c["head_dim"], "base": c["theta"], "style": "neox"})})
        dense = PartSpec("plain_mlp", {"hidden_size": h, "intermediate_size": c["ffn"], "activation": "gelu", "bias": True})
        beside = PartSpec("plain_mlp", {"hidden_size": h, "intermediate_size": c["ffn"], "activation": "silu"})
        experts = PartSpec("routed_experts", {"hidden_size": h, "num_experts": c["experts"], "top": c["top"], "activation": "silu",
                                              "intermediate_size": c["expert_ffn"], "score": "grouped", "weight_on": "output",
                                              "score_function": c["score_function"], "groups": c["groups"], "top_groups": c["top_groups"],
                                              "group_top": 2, "weight_scale": 1.5, "shared_intermediate_size": c["shared_ffn"]})
        layers = (LayerSpec(attn, dense, norm, norm), LayerSpec(attn, experts, norm, norm),
                  LayerSpec(mixer=attn, feed_forward=beside, mixer_norm=norm, arrangement="parallel_residual"), LayerSpec(attn, dense, norm, norm))
        return ModelSpec(h, c["vocab_size"], c["max_position"], PartSpec("token_embedding", {"vocab_size": c["vocab_size"], "hidden_size": h}),
                         layers, tuple(LayerCall(i, i) for i in range(4)), norm,
                         PartSpec("lm_head", {"hidden_size": h, "vocab_size": c["vocab_size"], "tied": False, "softcap": c["softcap"]}))

    def tensor_name(self, scope, local):
        return ".".join(str(s) for s in scope) + "." + local


def register():
    register_architecture(ScoredArch)
    return get_architecture("ScoredForCausalLM")


def unregister():
    unregister_architecture("ScoredForCausalLM")


def write(d, cfg=CFG, seed=11):
    from iian_b200.weights.random_init import write_model_folder
    write_model_folder(d, get_architecture("ScoredForCausalLM"), dict(cfg), seed=seed, store_dtype=torch.bfloat16, std=0.08)
    return d


def plain_logits(d, tokens, c=CFG):
    """Logits of every place of one whole sequence, in float64, without the framework; and how near each token's choice of experts was (the
    least distance between two corrected scores or group scores that decide it)."""
    import os
    w = plain.read_safetensors(os.path.join(d, "model.safetensors"))
    T, nh, nkv, hd = len(tokens), c["heads"], c["kv_heads"], c["head_dim"]
    pos = torch.arange(T)
    x = w["embedding.weight"][torch.tensor(tokens)]

    def attention(h, li):
        p = f"layer.{li}.mixer."
        q = plain.rope_neox((h @ w[p + "q_proj.weight"].T).view(T, nh, hd), pos, c["theta"], hd)
        k = plain.rope_neox((h @ w[p + "k_proj.weight"].T).view(T, nkv, hd), pos, c["theta"], hd)
        v = (h @ w[p + "v_proj.weight"].T).view(T, nkv, hd)
        return plain.attention(q, k, v, 1 / math.sqrt(hd), None).reshape(T, nh * hd) @ w[p + "o_proj.weight"].T

    def mlp(h, li, act, bias):
        p = f"layer.{li}.feed_forward."
        up = h @ w[p + "up"].T + (w[p + "up.b"] if bias else 0.0)
        return ACTIVATIONS[act](up) @ w[p + "down"].T + (w[p + "down.b"] if bias else 0.0)

    def experts(h, li):
        p = f"layer.{li}.feed_forward."
        z = h @ w[p + "router"].T
        ids, wt = choose(z, w[p + "correction"], c["score_function"], c["groups"], c["top_groups"], 2, c["top"], True, 1.5)
        out = plain.gated_mlp(h, w[p + "shared.gate"], w[p + "shared.up"], w[p + "shared.down"])
        for t in range(T):
            for e, g in zip(ids[t].tolist(), wt[t]):
                out[t] += g * plain.gated_mlp(h[t:t + 1], w[f"{p}e{e}.gate"], w[f"{p}e{e}.up"], w[f"{p}e{e}.down"])[0]
        return out

    norm = lambda x, name: plain.rms_norm(x, w[name], c["eps"])      # noqa: E731
    for li in range(4):
        h = norm(x, f"layer.{li}.mixer_norm.weight")
        if li == 2:
            x = x + attention(h, li) + mlp(h, li, "silu", False)
            continue
        x = x + attention(h, li)
        h = norm(x, f"layer.{li}.feed_forward_norm.weight")
        x = x + (experts(h, li) if li == 1 else mlp(h, li, "gelu", True))
    z = norm(x, "final_norm.weight") @ w["head.weight"].T
    return c["softcap"] * torch.tanh(z / c["softcap"]) if c["softcap"] else z


def plain_scores(d, tokens, c=CFG, start=1):
    """Log-probabilities of tokens[start:] given those before them."""
    lp = torch.log_softmax(plain_logits(d, tokens, c), 1)
    return [lp[i - 1, tokens[i]].item() for i in range(start, len(tokens))]
