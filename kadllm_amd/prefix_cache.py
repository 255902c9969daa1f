"""The 8-bit prefix cache: pages for a batch's requests, keys and values into
them, and attention of the beams over them.

A ``PrefixBlocks`` holds the pages of one attention layer.  A page holds
``block_size`` tokens as e4m3 codes [HK, block_size, D] with one e8m0 scale (a
power of two) per KV head; a token's value is code * scale.  A table [B,
columns] int32 names each request's pages in order (-1: none), so requests of
unequal length share one pool, and requests that begin alike may share pages.

    tables, used = prefix_block_tables(lengths, free, block_size=64, max_length=L)
    write_prefix_blocks(blocks, k, v, tables, lengths)
    out = block_prefix_attention(q, blocks, tables, lengths, suffix_k, suffix_v,
                                 beam_width=W)

Everything runs on the GPU without a host synchronisation; no counterpart in
the reference, whose prefix stays in the model's type
(src/kadllm/adapters/qwen3_5.py:106-133).
"""

import contextlib
import ctypes
import math
from typing import NamedTuple

import torch

from . import _lib

BLOCK_SIZES = (32, 64, 128, 256)
HEAD_DIMS = (64, 128, 256)
_CODES, _SCALES = torch.float8_e4m3fn, torch.float8_e8m0fnu


class PrefixBlocks(NamedTuple):
    """The pages of one layer: codes k, v [pages, HK, block_size, D]
    (torch.float8_e4m3fn) and scales [pages, HK] (torch.float8_e8m0fnu)."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor

    @classmethod
    def empty(cls, pages, kv_heads, head_dim, *, block_size=64, device="cuda"):
        """A pool of ``pages`` unwritten pages (zeros)."""
        if block_size not in BLOCK_SIZES:
            raise ValueError(f"block_size must be one of {BLOCK_SIZES}")
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}")
        if pages < 1 or kv_heads < 1:
            raise ValueError("a pool needs pages and KV heads")
        codes = [torch.zeros(pages, kv_heads, block_size, head_dim, dtype=torch.uint8,
                             device=device).view(_CODES) for _ in range(2)]
        scales = [torch.zeros(pages, kv_heads, dtype=torch.uint8, device=device).view(_SCALES)
                  for _ in range(2)]
        return cls(*codes, *scales)


def _on_device(t):
    """A context in which ``t``'s device is the current one."""
    if t.get_device() == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(t.device)


def _check_devices(first, *others):
    for t in others:
        if t is not None and t.device != first.device:
            raise ValueError("all tensors must be on the same device")
    if not first.is_cuda:
        raise RuntimeError(
            "kadllm_amd operators run on ROCm devices only; move tensors to the GPU")


def _check_int32(name, t, shape):
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be int32")
    if t.ndim != len(shape) or any(w is not None and w != s for w, s in zip(shape, t.shape)):
        want = ", ".join("*" if w is None else str(w) for w in shape)
        raise ValueError(f"{name} must have shape [{want}]")


def _check_blocks(blocks):
    """(pages, HK, block_size, D) of a well-formed PrefixBlocks."""
    if not isinstance(blocks, PrefixBlocks):
        raise TypeError("blocks must be a PrefixBlocks")
    k, v, k_scale, v_scale = blocks
    if k.dtype != _CODES or v.dtype != _CODES:
        raise TypeError("the codes of a prefix cache are torch.float8_e4m3fn")
    if k_scale.dtype != _SCALES or v_scale.dtype != _SCALES:
        raise TypeError("the scales of a prefix cache are torch.float8_e8m0fnu")
    if k.ndim != 4 or v.shape != k.shape or min(k.shape) < 1:
        raise ValueError("codes must be [pages, HK, block_size, D]")
    if k_scale.shape != k.shape[:2] or v_scale.shape != k.shape[:2]:
        raise ValueError("scales must be [pages, HK]")
    if k.shape[2] not in BLOCK_SIZES:
        raise ValueError(f"block_size must be one of {BLOCK_SIZES}")
    if k.shape[3] not in HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {HEAD_DIMS}")
    if not all(t.is_contiguous() for t in blocks):
        raise ValueError("the tensors of a prefix cache must be contiguous")
    return k.shape


def prefix_block_tables(lengths, free_blocks, *, block_size, max_length, starts=None, tables=None):
    """Pages for requests of ``lengths`` tokens.

    lengths [B] int32 are the requests' tokens after this step, at most
    ``max_length`` (longer ones are cut there); starts [B] int32 the tokens
    they hold already (default none), in the pages of the earlier ``tables``
    [B, columns].  A request gets ceil(lengths / block_size) -
    ceil(starts / block_size) pages more, in request order from the front of
    ``free_blocks`` [F] int32.  Returns (tables [B, ceil(max_length /
    block_size)] int32 with -1 past a request's last page, used [1] int32: the
    pages taken).  Where ``used`` exceeds F the list was too short: the entries
    it could not fill are -1, and the other operators leave such tokens out.
    """
    if not isinstance(block_size, int) or block_size not in BLOCK_SIZES:
        raise ValueError(f"block_size must be one of {BLOCK_SIZES}")
    if not isinstance(max_length, int) or isinstance(max_length, bool) or \
            not 0 < max_length < 2**31 - 256:
        raise ValueError("max_length must be a positive integer below 2**31 - 256")
    _check_int32("lengths", lengths, (None,))
    _check_int32("free_blocks", free_blocks, (None,))
    B = lengths.shape[0]
    if B < 1:
        raise ValueError("lengths must not be empty")
    if starts is not None:
        _check_int32("starts", starts, (B,))
    if tables is not None:
        if starts is None:
            raise ValueError("earlier tables need the tokens held (starts)")
        _check_int32("tables", tables, (B, None))
    _check_devices(lengths, free_blocks, starts, tables)
    lengths, free_blocks = lengths.contiguous(), free_blocks.contiguous()
    starts = None if starts is None else starts.contiguous()
    tables = None if tables is None else tables.contiguous()
    width = -(-max_length // block_size)
    out = torch.empty(B, width, dtype=torch.int32, device=lengths.device)
    used = torch.empty(1, dtype=torch.int32, device=lengths.device)
    with _on_device(lengths):
        _lib.call("kad_prefix_block_tables", _lib.ptr(lengths), _lib.ptr(starts),
                  _lib.ptr(tables), 0 if tables is None else tables.shape[1],
                  _lib.ptr(free_blocks), free_blocks.shape[0], _lib.ptr(out), width,
                  _lib.ptr(used), B, block_size, max_length, _lib.stream_of(lengths))
    return out, used


def write_prefix_blocks(blocks, k, v, tables, lengths, *, starts=None):
    """Keys and values into their requests' pages, in place.

    k, v [B, N, HK, D] (bf16, fp16 or fp32, any strides with a contiguous last
    dimension): token i of request b goes to position starts[b] + i (starts:
    [B] int32, default 0) while that is below lengths[b]; tables [B, columns]
    int32 and lengths [B] int32 as prefix_block_tables takes and gives them.

    A page's scale is the smallest power of two s >= 2**-100 with amax <= 448 s
    over the finite values written to it.  A page that holds earlier tokens
    keeps the larger of its scale and the new tokens'; when that grows, the
    earlier codes are rounded to the new scale.  Codes are x / s to the nearest
    e4m3 value (ties to even); infinities and NaN become NaN.  Rows behind
    lengths[b] and pages the call does not reach are left as they were; tokens
    whose table entry names no page are left out.  Two requests of one call
    must not write to the same page.  Returns ``blocks``.
    """
    pages, HK, block, D = _check_blocks(blocks)
    if k.ndim != 4 or v.shape != k.shape:
        raise ValueError("k and v must be [B, N, HK, D]")
    if k.dtype != v.dtype:
        raise ValueError("k and v must have the same dtype")
    if k.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise TypeError("k and v must be bf16, fp16 or fp32")
    B, N = k.shape[:2]
    if min(B, N) < 1 or k.shape[2:] != (HK, D):
        raise ValueError("k and v do not fit the cache's heads")
    _check_int32("tables", tables, (B, None))
    _check_int32("lengths", lengths, (B,))
    if starts is not None:
        _check_int32("starts", starts, (B,))
    if tables.shape[1] < 1:
        raise ValueError("tables must have columns")
    _check_devices(k, v, tables, lengths, starts, *blocks)
    k = k if k.stride(3) == 1 else k.contiguous()
    v = v if v.stride(3) == 1 else v.contiguous()
    tables, lengths = tables.contiguous(), lengths.contiguous()
    starts = None if starts is None else starts.contiguous()
    with _on_device(k):
        _lib.call("kad_write_prefix_blocks", _lib.ptr(k), *k.stride()[:3], _lib.ptr(v),
                  *v.stride()[:3], _lib.dtype_code(k.dtype), _lib.ptr(tables), tables.shape[1],
                  _lib.ptr(lengths), _lib.ptr(starts), *map(_lib.ptr, blocks), pages, B, N, HK, D,
                  block, _lib.stream_of(k))
    return blocks


def block_prefix_attention(q, blocks, tables, lengths, suffix_k=None, suffix_v=None, *,
                           beam_width=1, scale=None, gate=None):
    """prefix_attention over a prefix in the 8-bit cache.

    q [B*W, T, H, D] bf16 or fp16; tables [B, columns] and lengths [B] int32:
    a query sees the first lengths[b] cached tokens of its request, except any
    whose table entry names no page.  suffix_k, suffix_v [B*W, Tk, HK, D] in
    q's type, Tk >= T: the beam's own tokens, of which the queries are the last
    T (query t sees suffix keys up to Tk - T + t); None for none, as when the
    newest tokens are already in the cache.  ``scale`` defaults to D**-0.5;
    ``gate`` [B*W, T, H*D] multiplies the output by sigmoid(gate).  Returns
    [B*W, T, H, D] in q's type; a query that sees no key gets zeros.
    """
    from .ops import _width

    _width(beam_width)
    pages, HK, block, D = _check_blocks(blocks)
    if q.ndim != 4 or q.shape[3] != D:
        raise ValueError("q must be [B*W, T, H, D] with the cache's head dim")
    BW, T, H, _ = q.shape
    if min(BW, T, H) < 1 or BW % beam_width or H % HK:
        raise ValueError("empty dimensions or incompatible beam/head counts")
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError("queries over the 8-bit cache must be bf16 or fp16")
    B = BW // beam_width
    _check_int32("tables", tables, (B, None))
    _check_int32("lengths", lengths, (B,))
    if tables.shape[1] < 1:
        raise ValueError("tables must have columns")
    if (suffix_k is None) != (suffix_v is None):
        raise ValueError("give both suffix_k and suffix_v or neither")
    Tk = 0
    if suffix_k is not None:
        Tk = suffix_k.shape[1] if suffix_k.ndim == 4 else -1
        if Tk < T or suffix_k.shape != (BW, Tk, HK, D) or suffix_v.shape != suffix_k.shape:
            raise ValueError("suffix_k and suffix_v must be [B*W, Tk, HK, D] with Tk >= T")
        if suffix_k.dtype != q.dtype or suffix_v.dtype != q.dtype:
            raise ValueError("attention inputs must have the same dtype")
    if gate is not None and (gate.shape != (BW, T, H * D) or gate.dtype != q.dtype):
        raise ValueError("gate must be [B*W, T, H*D] in the query dtype")
    given = [t for t in (q, suffix_k, suffix_v, gate) if t is not None]
    if torch.is_grad_enabled() and any(t.requires_grad for t in given):
        raise RuntimeError("kadllm_amd operators are inference-only; disable gradients")
    _check_devices(q, tables, lengths, suffix_k, suffix_v, gate, *blocks)
    scale = 1 / math.sqrt(D) if scale is None else scale
    gate_strides = None
    if gate is not None:
        gate = _rows(gate, 4)
        gate_strides = (gate.stride(0), gate.stride(1), D)
    return _block_attention(q, blocks, tables, lengths, suffix_k, suffix_v, beam_width, scale,
                            gate, gate_strides)


def _rows(t, elements):
    """t, or a copy whose rows start at multiples of ``elements`` elements."""
    strides = t.stride()
    if strides[-1] == 1 and not any(s % elements for s in strides[:-1]) and \
            t.data_ptr() % (2 * elements) == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _block_attention(q, blocks, tables, lengths, suffix_k, suffix_v, beam_width, scale, gate=None,
                     gate_strides=None):
    """block_prefix_attention on checked arguments; ``gate`` any tensor whose
    data pointer is head 0's gate with element strides ``gate_strides`` =
    (beam, token, head)."""
    BW, T, H, D = q.shape
    pages, HK, block, _ = blocks.k.shape
    q = _rows(q, 8)
    tables, lengths = tables.contiguous(), lengths.contiguous()
    none = (None, 0, 0, 0)
    sk = sv = g = none
    Tk = 0
    if suffix_k is not None:
        suffix_k, suffix_v = _rows(suffix_k, 8), _rows(suffix_v, 8)
        Tk = suffix_k.shape[1]
        sk = (_lib.ptr(suffix_k), *suffix_k.stride()[:3])
        sv = (_lib.ptr(suffix_v), *suffix_v.stride()[:3])
    if gate is not None:
        g = (_lib.ptr(gate), *gate_strides)
    out = torch.empty(BW, T, H, D, dtype=q.dtype, device=q.device)
    need = ctypes.c_int64(0)
    _lib.call("kad_block_prefix_attention_workspace_bytes", BW // beam_width, beam_width, T, H, HK,
              D, tables.shape[1], block, ctypes.byref(need))
    ws = torch.empty(need.value, dtype=torch.uint8, device=q.device) if need.value else None
    with _on_device(q):
        _lib.call("kad_block_prefix_attention", _lib.ptr(q), *q.stride()[:3],
                  *map(_lib.ptr, blocks), pages, _lib.ptr(tables), tables.shape[1],
                  _lib.ptr(lengths), *sk, *sv, *g, _lib.ptr(out), *out.stride()[:3],
                  _lib.ptr(ws), need.value, BW // beam_width, beam_width, T, Tk, H, HK, D, block,
                  _lib.dtype_code(q.dtype), float(scale), _lib.stream_of(q))
    return out
