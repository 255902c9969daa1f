"""A Qwen3.5 model's 4-bit weights: sizes that are not the model's are refused as the
adapter is made (the one-call passes and the feed-forward block's kernels are given the
model's)."""

import pytest
import torch

from kadllm_amd.adapters import Qwen35GRBeamAdapter, native_model
from kadllm_amd.config import tiny_hybrid_config
from kadllm_amd.weights import random_state_dict

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name, dim", [
    ("mlp.gate_proj", 0), ("mlp.gate_proj", 1), ("mlp.up_proj", 0), ("mlp.up_proj", 1),
    ("mlp.down_proj", 0), ("mlp.down_proj", 1), ("linear_attn.in_proj_z", 0),
    ("linear_attn.out_proj", 0), ("linear_attn.out_proj", 1), ("self_attn.k_proj", 0),
    ("self_attn.o_proj", 0), ("self_attn.o_proj", 1), ("lm_head", 1)])
def test_weights_of_other_sizes_are_refused(device, name, dim):
    cfg = tiny_hybrid_config()
    sd = random_state_dict(cfg, seed=0, dtype=torch.bfloat16, device=device)
    if name == "lm_head":
        full = "lm_head.weight"
        sd.setdefault(full, sd["embed_tokens.weight"])
    else:
        full = next(n for n in sd if n.endswith(name + ".weight"))
    sd[full] = sd[full].narrow(dim, 0, sd[full].shape[dim] - 16).contiguous()
    model, head = native_model(cfg, sd)
    with pytest.raises(ValueError):
        Qwen35GRBeamAdapter(model, head, weights="e2m1")
