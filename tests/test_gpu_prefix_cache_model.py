"""The Qwen3.5 adapter with its attention prefixes in the 8-bit cache.

A page's codes times its scale are bf16 numbers (4 significant bits), so an
adapter that keeps bf16 prefixes can hold exactly what the 8-bit one holds: its
logits on those prefixes are the same sums, rounded elsewhere.  Both are held
to the oracle in fp32 on the same prefixes, as the other model tests are: the
8-bit path's error at most 1.5 times that of the bf16 path, +0.2%.
"""

import pytest
import torch

from kadllm_amd import grbeam_search
from kadllm_amd.adapters import Qwen35GRBeamAdapter, Qwen35Prefix, native_model
from kadllm_amd.config import qwen35_08b_config, tiny_hybrid_config
from kadllm_amd.prefix_cache import PagedPrefix
from kadllm_amd.weights import random_state_dict
from oracle import prefix_cache_ref as ref
from oracle.qwen35_ref import OraclePrefix, Qwen35Oracle

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tiny(device):
    cfg = tiny_hybrid_config()
    sd = random_state_dict(cfg, seed=0, dtype=torch.bfloat16)
    model, head = native_model(cfg, {k: v.to(device) for k, v in sd.items()})
    truth = Qwen35Oracle(cfg, {k: v.float() for k, v in sd.items()})
    return cfg, truth, Qwen35GRBeamAdapter(model, head), \
        Qwen35GRBeamAdapter(model, head, prefix_cache="e4m3")


def _dense(prefix, owner):
    """The prefix with its pages' values as bf16 (K, V) pairs."""
    layers = []
    for layer in prefix.layers:
        if not isinstance(layer, PagedPrefix):
            layers.append(layer)
            continue
        pair = []
        for codes, scales in ((layer.blocks.k, layer.blocks.k_scale),
                              (layer.blocks.v, layer.blocks.v_scale)):
            values = codes.float() * scales.float()[..., None, None]
            values = values[layer.tables.long()]           # [B, pages, HK, block, D]
            values = values.transpose(2, 3).flatten(1, 2)[:, :prefix.length]
            assert torch.equal(values.bfloat16().float(), values)
            pair.append(values.bfloat16())
        layers.append(tuple(pair))
    return Qwen35Prefix(prefix.length, prefix.batch, owner, tuple(layers))


def _rel(a, e):
    a, e = a.float().cpu(), e.float().cpu()
    return ((a - e).norm() / e.norm()).item()


@pytest.mark.parametrize("B, L, W, T", [(2, 128, 8, 1), (2, 65, 5, 3), (1, 7, 10, 2),
                                        (3, 200, 40, 2), (1, 64, 1, 9)])
def test_decode_over_8_bit_prefixes(device, tiny, B, L, W, T):
    cfg, truth, plain, paged = tiny
    g = torch.Generator().manual_seed(L)
    ids = torch.randint(0, cfg.vocab_size, (B, L), generator=g).to(device)
    history = torch.randint(0, cfg.vocab_size, (B, W, T), generator=g).to(device)
    want, got = plain.prefill(ids), paged.prefill(ids)
    assert torch.equal(want.logits, got.logits)
    kinds = [isinstance(x, PagedPrefix) for x in got.state.layers]
    assert kinds == [k == "full_attention" for k in cfg.layer_types]
    # what the pages hold is the prompt's keys and values, rounded to e4m3
    for layer, (k, v) in zip(got.state.layers, want.state.layers):
        if isinstance(layer, PagedPrefix):
            for x, codes, scales in ((k, layer.blocks.k, layer.blocks.k_scale),
                                     (v, layer.blocks.v, layer.blocks.v_scale)):
                c = torch.zeros(codes.shape, dtype=torch.float64)
                s = torch.zeros(scales.shape, dtype=torch.float64)
                ref.write(c, s, x.double().cpu(), layer.tables.tolist(), [L] * B, [0] * B,
                          codes.shape[2])
                now = ref.decode(codes, scales)
                assert torch.equal(now[0], c) and torch.equal(now[1], s)
    dense = _dense(got.state, plain._owner)
    a = paged.decode(history, got.state)
    b = plain.decode(history, dense)
    exact = truth.decode(history.cpu(), _oracle_state(dense))
    e_paged, e_plain = _rel(a, exact), _rel(b, exact)
    assert e_paged <= 1.5 * e_plain + 2e-3, (e_paged, e_plain)


def _oracle_state(dense):
    """The oracle's prefix with these layers' tensors, in fp32."""
    return OraclePrefix(dense.length, dense.batch,
                        tuple(tuple(x.float().cpu() for x in layer) for layer in dense.layers))


def test_search_over_8_bit_prefixes(device, tiny):
    cfg, truth, plain, paged = tiny
    ids = torch.randint(0, cfg.vocab_size, (2, 100), generator=torch.Generator().manual_seed(1))
    result = grbeam_search(paged, ids.to(device), [8, 8, 8])
    assert result.tokens.shape == (2, 8, 3) and bool(result.valid.all())
    # the incremental levels of the search and the stateless decode agree
    state = paged.prefill(ids.to(device)).state
    history = result.tokens[:, :, :2].contiguous()
    whole = paged.decode(history, state)
    first, cache = paged.decode_incremental(history[:, :, :1].contiguous(), None, state)
    parents = torch.arange(8, device=device).expand(2, 8).contiguous()
    step, _ = paged.decode_incremental(history, parents, state, cache)
    dense = _dense(state, plain._owner)
    exact = truth.decode(history.cpu(), _oracle_state(dense))
    assert _rel(step, exact) <= 1.5 * _rel(whole, exact) + 2e-3
    assert first.shape == (2, 8, cfg.vocab_size)


def test_08b_shape_over_8_bit_prefixes(device):
    cfg = qwen35_08b_config()
    sd = random_state_dict(cfg, seed=0, dtype=torch.bfloat16, device=device)
    model, head = native_model(cfg, sd)
    paged = Qwen35GRBeamAdapter(model, head, prefix_cache="e4m3")
    plain = Qwen35GRBeamAdapter(model, head)
    ids = torch.randint(0, cfg.vocab_size, (2, 150),
                        generator=torch.Generator().manual_seed(2)).to(device)
    state = paged.prefill(ids).state
    history = torch.randint(0, cfg.vocab_size, (2, 16, 2),
                            generator=torch.Generator().manual_seed(3)).to(device)
    a = paged.decode(history, state).float()
    b = plain.decode(history, _dense(state, plain._owner)).float()
    # two bf16 evaluations of one model: each is up to ~12% off the exact logits on
    # this shape (24 layers), at random
    assert a.isfinite().all() and (a - b).norm() <= 0.17 * b.norm()
    held = sum(t.numel() for x in state.layers if isinstance(x, PagedPrefix) for t in x.blocks)
    dense = sum(t.numel() * 2 for x in plain.prefill(ids).state.layers
                for t in x if t.dtype == torch.bfloat16 and t.ndim == 4)
    assert held < 0.7 * dense       # 150 tokens in pages of 64: 192 of them


def test_refusals(device, tiny):
    cfg, _, plain, paged = tiny
    with pytest.raises(ValueError, match="prefix_cache"):
        Qwen35GRBeamAdapter(plain.model, plain.lm_head, prefix_cache="int4")
    sd = random_state_dict(cfg, seed=0, dtype=torch.float32)
    model, head = native_model(cfg, {k: v.to(device) for k, v in sd.items()})
    with pytest.raises(ValueError, match="bf16"):
        Qwen35GRBeamAdapter(model, head, prefix_cache="e4m3")
    ids = torch.zeros(1, 5, dtype=torch.int64, device=device)
    state = paged.prefill(ids).state
    with pytest.raises(ValueError, match="different adapter"):
        plain.decode(ids[:, None], state)
    with pytest.raises(ValueError, match="transformers"):
        paged.prefix_to_cache(state)


def test_prefixes_from_a_transformers_cache(device, tiny):
    """The pages that prefix_from_cache fills are those that the prefill fills."""
    cfg, _, plain, paged = tiny
    ids = torch.randint(0, cfg.vocab_size, (2, 77),
                        generator=torch.Generator().manual_seed(4)).to(device)
    want = paged.prefill(ids).state
    got = paged.prefix_from_cache(plain.prefix_to_cache(plain.prefill(ids).state), 77)
    assert (got.length, got.batch) == (77, 2)
    for kind, a, b in zip(cfg.layer_types, got.layers, want.layers):
        assert isinstance(a, PagedPrefix) == (kind == "full_attention")
        if isinstance(a, PagedPrefix):
            for x, y in zip((*a.blocks, a.tables, a.lengths), (*b.blocks, b.tables, b.lengths)):
                assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
        else:
            assert all(torch.equal(x, y) for x, y in zip(a, b))
    history = torch.randint(0, cfg.vocab_size, (2, 5, 2),
                            generator=torch.Generator().manual_seed(5)).to(device)
    assert torch.equal(paged.decode(history, got), paged.decode(history, want))
