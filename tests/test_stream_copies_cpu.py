"""The 16-bit copy of the stream that its last writer may leave: an identity norm takes it only while it still says what the stream is."""
import math

import pytest
import torch

import scored_model as sm
from helpers import random_tokens
from iian_b200 import ops
from iian_b200.config.registry import get_architecture, register_architecture, unregister_architecture
from iian_b200.config.spec import LayerCall, LayerSpec, ModelSpec, PartSpec
from iian_b200.engine.model import Model
from iian_b200.engine.runner import ModelRunner, StepEntry
from iian_b200.parts.norm import Identity

CFG = {"architectures": ["CopiesForCausalLM"], "vocab_size": 97, "hidden_size": 32, "heads": 2, "kv_heads": 1, "head_dim": 16, "ffn": 48, "max_position": 64,
       "first": "mlp", "placed": "positions"}


class CopiesArch(sm.ScoredArch):
    name = "CopiesForCausalLM"

    def build_spec(self, c):
        h = c["hidden_size"]
        norm, none = PartSpec("rms_norm", {"size": h, "eps": 1e-5}), PartSpec("identity", {})
        attn = PartSpec("attention", {"hidden_size": h, "num_heads": c["heads"], "num_kv_heads": c["kv_heads"], "head_dim": c["head_dim"],
                                      "scale": 1 / math.sqrt(c["head_dim"]), "qk_norm": False, "window": None,
                                      "position": PartSpec("rotary", {"dim": c["head_dim"], "base": 1e4, "style": "neox"})})
        adds = PartSpec("plain_mlp", {"hidden_size": h, "intermediate_size": c["ffn"], "activation": "gelu", "bias": True})
        gated = PartSpec("gated_mlp", {"hidden_size": h, "intermediate_size": c["ffn"], "activation": "silu"})
        first = {"mlp": LayerSpec(attn, adds, norm, norm),
                 "scaled": LayerSpec(mixer=attn, feed_forward=gated, mixer_norm=norm, feed_forward_norm=norm, arrangement="scaled_residual",
                                     extra=(("residual_mult", PartSpec("value", {"value": 0.5})),))}[c["first"]]
        place = {"positions": {"positions": c["max_position"]}, "norm": {"norm": {"eps": 1e-5}}, "none": {}}[c["placed"]]
        return ModelSpec(h, c["vocab_size"], c["max_position"], PartSpec("token_embedding", {"vocab_size": c["vocab_size"], "hidden_size": h, **place}),
                         (first, LayerSpec(attn, adds, none, none), LayerSpec(attn, adds, none, none)), tuple(LayerCall(i, i) for i in range(3)), norm,
                         PartSpec("lm_head", {"hidden_size": h, "vocab_size": c["vocab_size"], "tied": False}))


@pytest.mark.parametrize("placed", ["positions", "norm", "none"])
@pytest.mark.parametrize("first", ["mlp", "scaled"])
def test_an_identity_norm_reads_the_stream_as_it_is(tmp_path, monkeypatch, first, placed):
    register_architecture(CopiesArch)
    try:
        from iian_b200.weights.random_init import write_model_folder
        cfg = dict(CFG, first=first, placed=placed)
        write_model_folder(str(tmp_path), get_architecture("CopiesForCausalLM"), cfg, seed=3, store_dtype=torch.bfloat16, std=0.2)
        with ops.use_kernels(sm.ScoredFakes()):
            model = Model.from_folder(str(tmp_path), "bfloat16", "cpu")
            runner = ModelRunner(model, block_size=8, capacity_tokens=64, max_num_seqs=2)
            read, plain = [], Identity.forward

            def look(self, residual, delta, ctx, delta_scale=1.0):
                out = plain(self, residual, delta, ctx, delta_scale)
                read.append((out - residual.to(out.dtype)).abs().max().item())
                return out
            monkeypatch.setattr(Identity, "forward", look)
            rc = runner.manager.new_request()
            assert runner.manager.allot_state(rc) and runner.manager.allocate(rc, 0, 11)
            runner.step([StepEntry(rc, random_tokens(97, 11, 5), 0, range(11))])
        assert len(read) == 4 and max(read) == 0.0
    finally:
        unregister_architecture("CopiesForCausalLM")
