"""The Qwen3.5 adapter with its projections, FFN and head in 4 bits.

A 4-bit weight's values are bf16 numbers, so an adapter of the same values in bf16 is
the same model, rounded elsewhere.  Both are held to the oracle in fp32 on those
values, as the other model tests are: the 4-bit path's error at most 1.5 times that of
the bf16 path, +0.2%."""

import pytest
import torch

from kadllm_amd import _lib, dequantize_weight, grbeam_search, quantize_weight
from kadllm_amd.adapters import Qwen35GRBeamAdapter, native_model
from kadllm_amd.config import qwen35_08b_config, tiny_hybrid_config
from kadllm_amd.weights import random_state_dict
from oracle.qwen35_ref import Qwen35Oracle

pytestmark = pytest.mark.gpu


def _dequantized(sd):
    """The state dict with the values that the adapter's 4-bit weights stand for, and
    those of the head (the embedding itself stays)."""
    out, names = {}, ("qkv", "z", "q_proj", "k_proj", "v_proj", "o_proj", "out_proj", "gate_proj",
                      "up_proj", "down_proj")
    for name, w in sd.items():
        if any(name.endswith(f"{n}.weight") for n in names):
            w = dequantize_weight(quantize_weight(w.cuda())).to(w.device)
        out[name] = w
    head = sd.get("lm_head.weight", sd["embed_tokens.weight"])
    return out, dequantize_weight(quantize_weight(head.cuda())).to(head.device)


def _pair(cfg, sd, device, **kwargs):
    """(4-bit adapter, bf16 adapter of the same values, oracle in fp32)."""
    model, head = native_model(cfg, {k: v.to(device) for k, v in sd.items()})
    q = Qwen35GRBeamAdapter(model, head, weights="e2m1", **kwargs)
    values, lm_head = _dequantized(sd)
    dense, dense_head = native_model(cfg, {**{k: v.to(device) for k, v in values.items()},
                                           "lm_head.weight": lm_head.to(device)})
    b = Qwen35GRBeamAdapter(dense, dense_head, **kwargs)
    truth = Qwen35Oracle(cfg, {**{k: v.float() for k, v in values.items()},
                               "lm_head.weight": lm_head.float()})
    return q, b, truth


@pytest.fixture(scope="module")
def tiny(device):
    cfg = tiny_hybrid_config()
    sd = random_state_dict(cfg, seed=0, dtype=torch.bfloat16)
    return (cfg, *_pair(cfg, sd, device))


def _rel(a, e):
    a, e = a.float().cpu(), e.float().cpu()
    return ((a - e).norm() / e.norm()).item()


def _no_worse(got, plain, exact):
    assert _rel(got, exact) <= 1.5 * _rel(plain, exact) + 2e-3


@pytest.mark.parametrize("B, L, W, T", [(2, 64, 8, 1), (2, 65, 5, 3), (1, 7, 10, 2),
                                        (3, 200, 40, 2), (1, 1, 1, 9)])
def test_prefill_and_decode(device, tiny, B, L, W, T):
    cfg, q, b, truth = tiny
    g = torch.Generator().manual_seed(B * L)
    ids = torch.randint(0, cfg.vocab_size, (B, L), generator=g)
    history = torch.randint(0, cfg.vocab_size, (B, W, T), generator=g)
    exact, state = truth.prefill(ids)
    mine, plain = q.prefill(ids.to(device)), b.prefill(ids.to(device))
    _no_worse(mine.logits, plain.logits, exact)
    exact = truth.decode(history, state)
    _no_worse(q.decode(history.to(device), mine.state), b.decode(history.to(device), plain.state),
              exact)


def test_incremental_decode_is_decode(device, tiny):
    cfg, q, b, truth = tiny
    ids = torch.randint(0, cfg.vocab_size, (2, 50), generator=torch.Generator().manual_seed(1))
    state = q.prefill(ids.to(device)).state
    exact_state = truth.prefill(ids)[1]
    plain_state = b.prefill(ids.to(device)).state
    history, cache = None, None
    g = torch.Generator().manual_seed(2)
    for step in range(3):
        tokens = torch.randint(0, cfg.vocab_size, (2, 6, 1), generator=g).to(device)
        parents = torch.randint(0, 6, (2, 6), generator=g).to(device)
        if history is None:
            history = tokens
        else:
            history = torch.cat((history.gather(1, parents[..., None].expand(-1, -1, step)),
                                 tokens), 2)
        logits, cache = q.decode_incremental(history, parents, state, cache)
        exact = truth.decode(history.cpu(), exact_state)
        plain = b.decode(history, plain_state)
        _no_worse(logits, plain, exact)


def test_one_call_layers_give_the_single_steps_bits(device):
    # the passes that C enqueues are the passes that Python enqueues, call by call
    cfg = _small_08b()
    sd = random_state_dict(cfg, seed=3, dtype=torch.bfloat16)
    model, head = native_model(cfg, {k: v.to(device) for k, v in sd.items()})
    q = Qwen35GRBeamAdapter(model, head, weights="e2m1")
    ids = torch.randint(0, cfg.vocab_size, (2, 40), generator=torch.Generator().manual_seed(4))
    ids = ids.to(device)
    names = []

    def run():
        pre = q.prefill(ids)
        first = torch.arange(12, device=device).view(2, 6, 1)
        parents = torch.tensor([[0, 2, 1, 5, 3, 3]] * 2, device=device)
        a, cache = q.decode_incremental(first, parents, pre.state)
        second = torch.cat((first.gather(1, parents[..., None]), first + 7), 2)
        b, _ = q.decode_incremental(second, parents, pre.state, cache, keep_cache=False)
        return pre.logits, a, b

    assert q._runner._native_layers() is not None
    want = run()
    try:
        _lib.set_call_hook(lambda name, args, launch: (names.append(name), launch()))
        got = run()
    finally:
        _lib.set_call_hook(None)
    assert "kad_quantized_gated_ffn" in names and "kad_quantized_linear" in names
    for x, y in zip(want, got):
        assert torch.equal(x, y)


def _small_08b():
    """The 0.8B shape with 4 layers and a small vocabulary."""
    import dataclasses
    cfg = qwen35_08b_config()
    return dataclasses.replace(cfg, num_hidden_layers=4, layer_types=cfg.layer_types[:4],
                               vocab_size=1000)


def test_search(device, tiny):
    cfg, q, b, truth = tiny
    ids = torch.randint(0, cfg.vocab_size, (2, 33), generator=torch.Generator().manual_seed(5))
    result = grbeam_search(q, ids.to(device), [8, 8, 8])
    assert result.tokens.shape == (2, 8, 3) and bool(result.valid.all())
    again = grbeam_search(q, ids.to(device), [8, 8, 8])
    assert torch.equal(result.tokens, again.tokens) and torch.equal(result.scores, again.scores)
    # the scores are those of the found sequences
    logp = torch.log_softmax(truth.prefill(ids)[0].double(), -1)
    first = logp.gather(1, result.tokens[:, :, 0].cpu())
    state = truth.prefill(ids)[1]
    total = first
    for t in (1, 2):
        step = torch.log_softmax(truth.decode(result.tokens[:, :, :t].cpu(), state).double(), -1)
        total = total + step.gather(2, result.tokens[:, :, t:t + 1].cpu())[..., 0]
    assert (result.scores.cpu().double() - total).abs().max() <= 0.1


def test_with_the_8_bit_prefix_cache(device, tiny):
    cfg, q, b, truth = tiny
    sd = random_state_dict(cfg, seed=0, dtype=torch.bfloat16)
    model, head = native_model(cfg, {k: v.to(device) for k, v in sd.items()})
    both = Qwen35GRBeamAdapter(model, head, weights="e2m1", prefix_cache="e4m3")
    ids = torch.randint(0, cfg.vocab_size, (2, 100), generator=torch.Generator().manual_seed(6))
    history = torch.randint(0, cfg.vocab_size, (2, 5, 2),
                            generator=torch.Generator().manual_seed(7)).to(device)
    ids = ids.to(device)
    a = q.decode(history, q.prefill(ids).state)
    c = both.decode(history, both.prefill(ids).state)
    assert _rel(c, a) <= 0.1  # prefixes to e4m3: 2^-4 a value at most


def test_head_tokens_and_odd_widths(device):
    # an FFN wider than the others and of odd width, and a head of some tokens
    cfg = tiny_hybrid_config()
    sd = random_state_dict(cfg, seed=1, dtype=torch.bfloat16)
    g = torch.Generator().manual_seed(8)
    H = cfg.hidden_size
    for name, shape in (("gate", (301, H)), ("up", (301, H)), ("down", (H, 301))):
        sd[f"layers.1.mlp.{name}_proj.weight"] = (torch.randn(shape, generator=g) * 0.05).bfloat16()
    tokens = torch.randperm(cfg.vocab_size, generator=g)[:37].tolist()
    q, b, truth = _pair(cfg, sd, device, head_tokens=tokens)
    ids = torch.randint(0, cfg.vocab_size, (2, 30), generator=g)
    exact = truth.prefill(ids)[0][:, tokens]
    _no_worse(q.prefill(ids.to(device)).logits, b.prefill(ids.to(device)).logits, exact)


def test_refusals(device, tiny):
    cfg = tiny[0]
    sd = random_state_dict(cfg, seed=0, dtype=torch.bfloat16)
    model, head = native_model(cfg, {k: v.to(device) for k, v in sd.items()})
    with pytest.raises(ValueError):
        Qwen35GRBeamAdapter(model, head, weights="int4")
    model, head = native_model(cfg, {k: v.float().to(device) for k, v in sd.items()})
    with pytest.raises(ValueError):
        Qwen35GRBeamAdapter(model, head, weights="e2m1")
