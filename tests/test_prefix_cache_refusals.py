"""Refusals of the 8-bit prefix cache's operators, and its oracle (CPU only:
every argument is checked on the host before any launch)."""

import ctypes

import pytest
import torch

import kadllm
from kadllm_amd import _lib
from kadllm_amd.ops import (PrefixBlocks, block_prefix_attention, prefix_block_tables,
                            write_prefix_blocks)
from oracle import prefix_cache_ref as ref

I32 = torch.int32


def _blocks(pages=3, HK=2, D=64, block=32):
    return PrefixBlocks.empty(pages, HK, D, block_size=block, device="cpu")


def test_names_are_public():
    for name in ("PrefixBlocks", "prefix_block_tables", "write_prefix_blocks",
                 "block_prefix_attention"):
        assert getattr(kadllm, name) is getattr(kadllm.ops, name)
        assert name in kadllm.__all__


def test_empty_pool():
    k, v, ks, vs = _blocks()
    assert k.shape == v.shape == (3, 2, 32, 64) and k.dtype == torch.float8_e4m3fn
    assert ks.shape == vs.shape == (3, 2) and vs.dtype == torch.float8_e8m0fnu
    for bad in (dict(block=48), dict(D=96), dict(pages=0), dict(HK=0)):
        with pytest.raises(ValueError):
            _blocks(**bad)


@pytest.mark.parametrize("change, error", [
    (dict(lengths=torch.ones(2)), TypeError),
    (dict(lengths=torch.ones(2, 1, dtype=I32)), ValueError),
    (dict(lengths=torch.ones(0, dtype=I32)), ValueError),
    (dict(free_blocks=torch.ones(2, dtype=torch.int64)), TypeError),
    (dict(block_size=48), ValueError),
    (dict(block_size=64.0), ValueError),
    (dict(max_length=0), ValueError),
    (dict(max_length=True), ValueError),
    (dict(max_length=2**31), ValueError),
    (dict(starts=torch.ones(3, dtype=I32)), ValueError),
    (dict(tables=torch.ones(2, 1, dtype=I32)), ValueError),
    (dict(starts=torch.ones(2, dtype=I32), tables=torch.ones(3, 1, dtype=I32)), ValueError),
    (dict(), RuntimeError),  # well-formed, but not on a ROCm device
])
def test_tables_refusals(change, error):
    args = dict(lengths=torch.ones(2, dtype=I32), free_blocks=torch.arange(4, dtype=I32),
                block_size=64, max_length=100)
    args.update(change)
    with pytest.raises(error):
        prefix_block_tables(args.pop("lengths"), args.pop("free_blocks"), **args)


@pytest.mark.parametrize("change, error", [
    (dict(blocks=tuple(_blocks())), TypeError),
    (dict(blocks=_blocks()._replace(k=torch.zeros(3, 2, 32, 64))), TypeError),
    (dict(blocks=_blocks()._replace(k_scale=torch.zeros(3, 2))), TypeError),
    (dict(blocks=_blocks()._replace(v=_blocks(pages=2).v)), ValueError),
    (dict(blocks=_blocks()._replace(v_scale=_blocks(HK=1).v_scale)), ValueError),
    (dict(k=torch.zeros(2, 5, 2, 64, dtype=torch.float64),
          v=torch.zeros(2, 5, 2, 64, dtype=torch.float64)), TypeError),
    (dict(v=torch.zeros(2, 5, 2, 64, dtype=torch.float16)), ValueError),
    (dict(v=torch.zeros(2, 4, 2, 64, dtype=torch.bfloat16)), ValueError),
    (dict(k=torch.zeros(2, 0, 2, 64, dtype=torch.bfloat16),
          v=torch.zeros(2, 0, 2, 64, dtype=torch.bfloat16)), ValueError),
    (dict(k=torch.zeros(2, 5, 1, 64, dtype=torch.bfloat16),
          v=torch.zeros(2, 5, 1, 64, dtype=torch.bfloat16)), ValueError),
    (dict(tables=torch.zeros(3, 1, dtype=I32)), ValueError),
    (dict(tables=torch.zeros(2, 0, dtype=I32)), ValueError),
    (dict(tables=torch.zeros(2, 1, dtype=torch.int64)), TypeError),
    (dict(lengths=torch.zeros(1, dtype=I32)), ValueError),
    (dict(starts=torch.zeros(2, dtype=torch.int64)), TypeError),
    (dict(k=torch.zeros(2, 5, 2, 64, dtype=torch.bfloat16).requires_grad_()), RuntimeError),
    (dict(v=torch.zeros(2, 5, 2, 64, dtype=torch.bfloat16).requires_grad_()), RuntimeError),
    (dict(), RuntimeError),
])
def test_write_refusals(change, error):
    args = dict(blocks=_blocks(), k=torch.zeros(2, 5, 2, 64, dtype=torch.bfloat16),
                v=torch.zeros(2, 5, 2, 64, dtype=torch.bfloat16),
                tables=torch.zeros(2, 1, dtype=I32), lengths=torch.zeros(2, dtype=I32))
    args.update(change)
    starts = args.pop("starts", None)
    with pytest.raises(error):
        write_prefix_blocks(*args.values(), starts=starts)


def _bf(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


@pytest.mark.parametrize("change, error", [
    (dict(q=_bf(4, 1, 4, 128)), ValueError),
    (dict(q=_bf(4, 4, 64)), ValueError),
    (dict(q=_bf(3, 1, 4, 64)), ValueError),
    (dict(q=_bf(4, 1, 3, 64)), ValueError),
    (dict(q=torch.zeros(4, 1, 4, 64)), TypeError),
    (dict(beam_width=0), ValueError),
    (dict(beam_width=True), ValueError),
    (dict(tables=torch.zeros(1, 1, dtype=I32)), ValueError),
    (dict(tables=torch.zeros(2, 0, dtype=I32)), ValueError),
    (dict(lengths=torch.zeros(2, dtype=torch.int64)), TypeError),
    (dict(suffix_k=_bf(4, 1, 2, 64)), ValueError),
    (dict(suffix_k=_bf(4, 0, 2, 64), suffix_v=_bf(4, 0, 2, 64)), ValueError),
    (dict(suffix_k=_bf(4, 1, 4, 64), suffix_v=_bf(4, 1, 4, 64)), ValueError),
    (dict(suffix_k=_bf(4, 2, 2, 64), suffix_v=_bf(4, 1, 2, 64)), ValueError),
    (dict(suffix_k=_bf(1, 1, 2, 64).expand(4, 2**22 + 1, 2, 64),
          suffix_v=_bf(1, 1, 2, 64).expand(4, 2**22 + 1, 2, 64)), ValueError),
    (dict(suffix_k=_bf(4, 1, 2, 64).half(), suffix_v=_bf(4, 1, 2, 64)), ValueError),
    (dict(gate=_bf(4, 1, 64)), ValueError),
    (dict(gate=torch.zeros(4, 1, 256)), ValueError),
    (dict(q=_bf(4, 1, 4, 64).requires_grad_()), RuntimeError),
    (dict(), RuntimeError),
])
def test_attention_refusals(change, error):
    args = dict(q=_bf(4, 1, 4, 64), blocks=_blocks(), tables=torch.zeros(2, 1, dtype=I32),
                lengths=torch.zeros(2, dtype=I32), beam_width=2)
    args.update(change)
    with pytest.raises(error):
        block_prefix_attention(**args)


def test_entry_points_refuse_before_any_launch():
    """The C entry points check sizes and pointers on the host."""
    lib = _lib.load()
    p = ctypes.c_void_p(256)  # never read: every call below is refused
    tables = lambda **k: lib.kad_prefix_block_tables(  # noqa: E731
        k.get("lengths", p), None, k.get("old", None), 0, p, 1, p, k.get("width", 2), p, 1, 64,
        k.get("most", 100), None)
    assert tables(lengths=None) == tables(width=1) == tables(old=p) == tables(most=0) == -1
    write = lambda **k: lib.kad_write_prefix_blocks(  # noqa: E731
        k.get("k", p), 0, 0, 0, p, 0, 0, 0, k.get("dtype", 0), p, k.get("width", 1), p, None, p, p, p,
        p, 1, k.get("B", 1), 1, 1, k.get("D", 64), k.get("block", 64), None)
    assert write(k=None) == write(B=0) == write(D=96) == write(block=48) == -1
    assert write(width=2**30) == -1
    assert write(dtype=7) == -2
    attend = lambda **k: lib.kad_block_prefix_attention(  # noqa: E731
        k.get("q", p), 0, 0, k.get("sq", 0), p, p, p, p, 1, p, k.get("width", 1), p,
        k.get("sk", None), 0, 0, 0, k.get("sk", None), 0, 0, 0, None, 0, 0, 0, p, 0, 0, 0,
        k.get("ws", None), 2**40, k.get("B", 1), 1, 1, k.get("Tk", 0), k.get("H", 2), 2,
        k.get("D", 64), k.get("block", 64), k.get("dtype", 0), 1.0, None)
    assert attend(q=None) == attend(Tk=1) == attend(H=3) == attend(D=32) == attend(block=16) == -1
    assert attend(sq=4) == attend(q=ctypes.c_void_p(264)) == attend(width=2**30) == -1
    assert attend(width=64) == -1 and b"workspace" in lib.kad_last_error()
    assert attend(Tk=2**22 + 1, sk=p) == -1 and b"suffix" in lib.kad_last_error()
    assert attend(width=64, ws=ctypes.c_void_p(264)) == -1
    assert attend(B=2**30, H=2**20) == -1 and b"rows" in lib.kad_last_error()
    assert attend(dtype=2) == -2
    need = ctypes.c_int64(-1)
    size = lib.kad_block_prefix_attention_workspace_bytes
    assert size(1, 1, 1, 2, 2, 64, 1, 64, ctypes.byref(need)) == 0 and need.value == 0
    assert size(1, 1, 1, 2, 2, 64, 64, 64, ctypes.byref(need)) == 0 and need.value > 0
    assert size(1, 1, 1, 3, 2, 64, 1, 64, ctypes.byref(need)) == -1
    assert size(1, 1, 1, 2, 2, 64, 1, 64, None) == -1


def test_oracle_codes_agree_with_torch():
    x = torch.cat((torch.linspace(-448, 448, 3001), torch.linspace(-0.03, 0.03, 1001)))
    assert torch.equal(ref.round_e4m3(x.double()), x.to(torch.float8_e4m3fn).double())
    bytes_ = torch.arange(256, dtype=torch.uint8)
    values, _ = ref.decode(bytes_.view(torch.float8_e4m3fn), bytes_.view(torch.float8_e8m0fnu))
    assert torch.equal(values.nan_to_num(1e9),
                       bytes_.view(torch.float8_e4m3fn).double().nan_to_num(1e9))


def test_oracle_scale_is_the_smallest_that_holds_the_values():
    for amax, want in ((448.0, 1.0), (448.5, 2.0), (0.0, 2.0 ** -100), (3.5, 2.0 ** -7)):
        codes, scales = torch.zeros(1, 1, 32, 64).double(), torch.ones(1, 1).double()
        x = torch.zeros(1, 2, 1, 64).double()
        x[0, 1, 0, 5] = -amax
        ref.write(codes, scales, x, [[0]], [2], [0], 32)
        assert scales.item() == want and codes.abs().max() <= 448
        assert codes[0, 0, 1, 5].item() * want == pytest.approx(-amax, rel=2 ** -4)


def test_tables_refuse_a_count_of_another_kind():
    lengths, free = torch.ones(2, dtype=I32), torch.arange(4, dtype=I32)
    for taken, error in ((torch.zeros(1, dtype=torch.int64), TypeError),
                         (torch.zeros(2, dtype=I32), ValueError),
                         (torch.zeros((), dtype=I32), ValueError),
                         (torch.zeros(1, dtype=I32), RuntimeError)):   # not on a ROCm device
        with pytest.raises(error):
            prefix_block_tables(lengths, free, block_size=64, max_length=100, taken=taken)


def test_launches_past_a_grid_are_refused():
    """A grid holds fewer than 2^32 work-items a dimension.  Addresses are never
    read: every call is refused on the host, and one below the limit is not made."""
    lib, p = _lib.load(), ctypes.c_void_p(256)
    assert lib.kad_prefix_block_tables(p, None, None, 0, p, 1, p, 2, p, 2**20 + 1, 64, 100,
                                       None) == -1
    assert b"requests" in lib.kad_last_error()
    with pytest.raises(ValueError, match="requests"):
        prefix_block_tables(torch.ones(1, dtype=I32).expand(2**20 + 1), torch.arange(4, dtype=I32),
                            block_size=64, max_length=100)
    # 1024, 64 and 128 threads a page
    for B, N, D, block, starts in ((2**22, 1, 256, 256, None), (2**26, 1, 64, 32, None),
                                   (2**16, 2**16, 64, 128, None), (2**25, 2, 64, 64, p)):
        assert lib.kad_write_prefix_blocks(p, 0, 0, 0, p, 0, 0, 0, 0, p, 2**16, p, starts, p, p, p, p,
                                           1, B, N, 1, D, block, None) == -1
        assert b"pages" in lib.kad_last_error()
    need = ctypes.c_int64()
    for B, W, H, HK, D, width in ((2**24, 1, 1, 1, 64, 1), (2**23, 1, 2, 2, 256, 1),
                                  (2, 2**30, 1, 1, 128, 1), (2, 2**30, 1, 1, 64, 64)):
        assert lib.kad_block_prefix_attention_workspace_bytes(
            B, W, 1, H, HK, D, width, 64, ctypes.byref(need)) == -1
        assert b"rows" in lib.kad_last_error()
        assert lib.kad_block_prefix_attention(
            p, 0, 0, 0, p, p, p, p, 1, p, width, p, None, 0, 0, 0, None, 0, 0, 0, None, 0, 0, 0, p, 0,
            0, 0, p, 2**62, B, W, 1, 0, H, HK, D, 64, 0, 1.0, None) == -1
        assert b"rows" in lib.kad_last_error()
    size = lib.kad_block_prefix_attention_workspace_bytes
    assert size(1, 1, 1, 2, 2, 96, 1, 64, ctypes.byref(need)) == -1
    assert size(1, 1, 1, 2, 2, 64, 1, -64, ctypes.byref(need)) == -1
    # one form's workgroups fit where the other's do not
    assert size(1, 2**30, 1, 1, 1, 64, 1, 64, ctypes.byref(need)) == 0 and need.value == 0
    assert size(2**24 - 1, 1, 1, 1, 1, 64, 1, 64, ctypes.byref(need)) == 0 and need.value == 0
