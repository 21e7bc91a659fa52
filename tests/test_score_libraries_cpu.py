"""What a model names as its kernels' libraries is what its scoring calls, too: they are compiled and loaded when it is, not at the first prompt."""
import re

import pytest
import torch

import iian_b200.ops.cuda_backend as backend
from iian_b200.config.spec import PartSpec
from iian_b200.parts.embedding import LMHead


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("softcap", [None, 30.0])
def test_the_head_names_what_its_scores_call(dtype, softcap):
    head = LMHead(PartSpec("lm_head", {"hidden_size": 64, "vocab_size": 100, "tied": True, "softcap": softcap}), dtype, torch.device("cpu"))
    source = open(backend.__file__).read()
    calls = source[source.index("def linear_logprobs("):source.index("# ---- sampling")]
    called = set(re.findall(r'_entry\("(\w+)"', calls))
    assert {"linear_fused", "linear_f32", "gemm_simt"} == called <= set(head.kernel_libraries())
