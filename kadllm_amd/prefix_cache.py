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

import ctypes
import functools
from typing import NamedTuple

import torch

from . import _lib

BLOCK_SIZES = (32, 64, 128, 256)
HEAD_DIMS = (64, 128, 256)
MAX_LENGTH = 2**30          # tokens of a request
MAX_REQUESTS = 2**20        # rows of a block table
MAX_SUFFIX = 2**22          # suffix keys of a beam
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


def _launch(device, name, *args):
    """An entry point on the current stream of ``device`` (an index), which
    need not be the current device."""
    if device == torch.cuda.current_device():
        _lib.call(name, *args, _lib.stream_of_index(device))
    else:
        with torch.cuda.device(device):
            _lib.call(name, *args, _lib.stream_of_index(device))


def _device_of(first, *others):
    """The index of the ROCm device that all the tensors are on."""
    index = first.get_device()
    for t in others:
        if t is not None and t.get_device() != index:
            raise ValueError("all tensors must be on the same device")
    if index < 0 or not first.is_cuda:
        raise RuntimeError(
            "kadllm_amd operators run on ROCm devices only; move tensors to the GPU")
    return index


def _check_int32(name, t, ndim, rows=None):
    """t is int32 with ``ndim`` dimensions, the first of ``rows``; contiguous."""
    if t.dtype is not torch.int32:
        raise TypeError(f"{name} must be int32")
    if t.ndim != ndim or (rows is not None and t.shape[0] != rows):
        raise ValueError(f"{name} must have {ndim} dimension(s)"
                         + ("" if rows is None else f", the first of {rows}"))
    return t if t.is_contiguous() else t.contiguous()


def _check_blocks(blocks):
    """(pages, HK, block_size, D) of a well-formed PrefixBlocks."""
    if not isinstance(blocks, PrefixBlocks):
        raise TypeError("blocks must be a PrefixBlocks")
    k, v, k_scale, v_scale = blocks
    if k.dtype is not _CODES or v.dtype is not _CODES:
        raise TypeError("the codes of a prefix cache are torch.float8_e4m3fn")
    if k_scale.dtype is not _SCALES or v_scale.dtype is not _SCALES:
        raise TypeError("the scales of a prefix cache are torch.float8_e8m0fnu")
    shape = k.shape
    if len(shape) != 4 or v.shape != shape or 0 in shape:
        raise ValueError("codes must be [pages, HK, block_size, D]")
    if k_scale.shape != shape[:2] or v_scale.shape != shape[:2]:
        raise ValueError("scales must be [pages, HK]")
    if shape[2] not in BLOCK_SIZES:
        raise ValueError(f"block_size must be one of {BLOCK_SIZES}")
    if shape[3] not in HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {HEAD_DIMS}")
    if not (k.is_contiguous() and v.is_contiguous() and k_scale.is_contiguous()
            and v_scale.is_contiguous()):
        raise ValueError("the tensors of a prefix cache must be contiguous")
    return shape


def prefix_block_tables(lengths, free_blocks, *, block_size, max_length, starts=None, tables=None,
                        taken=None):
    """Pages for requests of ``lengths`` tokens.

    lengths [B] int32, B <= 2**20, are the requests' tokens after this step, at
    most ``max_length`` (longer ones are cut there); starts [B] int32 the tokens
    they hold already (default none), in the pages of the earlier ``tables``
    [B, columns].  A request gets ceil(lengths / block_size) -
    ceil(starts / block_size) pages more, in request order from the front of
    ``free_blocks`` [F] int32, behind the first ``taken`` [1] int32 (default
    none).  Returns (tables [B, ceil(max_length / block_size)] int32 with -1 past
    a request's last page, used [1] int32: the pages of the list that are taken
    now, those before this call included, at most 2**31 - 1).  Where ``used``
    exceeds F the list was too short: the entries it could not fill are -1, and
    the other operators leave such tokens out.  A loop that hands ``used`` on as
    the next call's ``taken`` gives out no page twice.
    """
    if not isinstance(block_size, int) or block_size not in BLOCK_SIZES:
        raise ValueError(f"block_size must be one of {BLOCK_SIZES}")
    if not isinstance(max_length, int) or isinstance(max_length, bool) or \
            not 0 < max_length <= MAX_LENGTH:
        raise ValueError(f"max_length must be a positive integer of at most {MAX_LENGTH}")
    lengths = _check_int32("lengths", lengths, 1)
    free_blocks = _check_int32("free_blocks", free_blocks, 1)
    B = lengths.shape[0]
    if not 0 < B <= MAX_REQUESTS:
        raise ValueError(f"lengths must be those of 1 to {MAX_REQUESTS} requests")
    if starts is not None:
        starts = _check_int32("starts", starts, 1, B)
    if tables is not None:
        if starts is None:
            raise ValueError("earlier tables need the tokens held (starts)")
        tables = _check_int32("tables", tables, 2, B)
    if taken is not None:
        taken = _check_int32("taken", taken, 1, 1)
    device = _device_of(lengths, free_blocks, starts, tables, taken)
    width = -(-max_length // block_size)
    out = torch.empty((B, width), dtype=torch.int32, device=lengths.device)
    used = torch.empty(1, dtype=torch.int32, device=lengths.device)
    _launch(device, "kad_prefix_block_tables_ex", lengths.data_ptr(), _lib.ptr(starts),
            _lib.ptr(tables), 0 if tables is None else tables.shape[1], free_blocks.data_ptr(),
            free_blocks.shape[0], _lib.ptr(taken), out.data_ptr(), width, used.data_ptr(), B,
            block_size, max_length)
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
    earlier codes are rounded to the new scale (a scale that is not a number
    stays, and the new codes are NaN).  Codes are x / s to the nearest e4m3 value
    (ties to even): off by up to 2**-4 of x, or by 2**-10 s where that is more;
    infinities and NaN become NaN.  Rows behind lengths[b] and pages the call
    does not reach are left as they were; tokens whose table entry names no page
    are left out.  Tokens are written in order: codes behind the last one written
    to a page stay, but not the scale they were made for.  One call must not
    write to a page twice.  Returns ``blocks``.
    """
    pages, HK, block, D = _check_blocks(blocks)
    shape = k.shape
    if len(shape) != 4 or v.shape != shape:
        raise ValueError("k and v must be [B, N, HK, D]")
    if k.dtype is not v.dtype:
        raise ValueError("k and v must have the same dtype")
    if k.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise TypeError("k and v must be bf16, fp16 or fp32")
    B, N, heads, dim = shape
    if 0 in shape or heads != HK or dim != D:
        raise ValueError("k and v do not fit the cache's heads")
    tables = _check_int32("tables", tables, 2, B)
    lengths = _check_int32("lengths", lengths, 1, B)
    if starts is not None:
        starts = _check_int32("starts", starts, 1, B)
    if not 0 < tables.shape[1] * block <= MAX_LENGTH:
        raise ValueError(f"tables must have columns, for at most {MAX_LENGTH} tokens")
    if torch.is_grad_enabled() and (k.requires_grad or v.requires_grad):
        raise RuntimeError("kadllm_amd operators are inference-only; disable gradients")
    device = _device_of(k, v, tables, lengths, starts, *blocks)
    k = k if k.stride(3) == 1 else k.contiguous()
    v = v if v.stride(3) == 1 else v.contiguous()
    _launch(device, "kad_write_prefix_blocks", k.data_ptr(), *k.stride()[:3], v.data_ptr(),
            *v.stride()[:3], _lib.dtype_code(k.dtype), tables.data_ptr(), tables.shape[1],
            lengths.data_ptr(), _lib.ptr(starts), *[x.data_ptr() for x in blocks], pages, B, N,
            HK, D, block)
    return blocks


def block_prefix_attention(q, blocks, tables, lengths, suffix_k=None, suffix_v=None, *,
                           beam_width=1, scale=None, gate=None):
    """prefix_attention over a prefix in the 8-bit cache.

    q [B*W, T, H, D] bf16 or fp16; tables [B, columns] and lengths [B] int32:
    a query sees the first lengths[b] cached tokens of its request, except any
    whose table entry names no page.  suffix_k, suffix_v [B*W, Tk, HK, D] in
    q's type, T <= Tk <= 2**22: the beam's own tokens, of which the queries are the
    last T (query t sees suffix keys up to Tk - T + t); None for none, as when the
    newest tokens are already in the cache.  ``scale`` defaults to D**-0.5;
    ``gate`` [B*W, T, H*D] multiplies the output by sigmoid(gate).  Returns
    [B*W, T, H, D] in q's type; a query that sees no key gets zeros.

    Scores, sums and the output are held in fp32.  The softmax weights of cached
    keys are off by up to 2**-8 of themselves for bf16 and 2**-12 for fp16, or 2**-17
    of the largest where that is more; those of suffix keys are rounded to q's
    type; elements of q below 2**-10 of their row's largest are off by up to 2**-21
    of it.  A suffix is walked 16 keys at a time by a part of the workgroups, which
    suits the few tokens of a search; the bulk of a long one is better written to
    the cache first.
    """
    if type(beam_width) is not int or beam_width <= 0:
        raise ValueError("beam_width must be a positive integer")
    pages, HK, block, D = _check_blocks(blocks)
    shape = q.shape
    if len(shape) != 4 or shape[3] != D:
        raise ValueError("q must be [B*W, T, H, D] with the cache's head dim")
    BW, T, H, _ = shape
    if 0 in shape or BW % beam_width or H % HK:
        raise ValueError("empty dimensions or incompatible beam/head counts")
    dtype = q.dtype
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise TypeError("queries over the 8-bit cache must be bf16 or fp16")
    B = BW // beam_width
    tables = _check_int32("tables", tables, 2, B)
    lengths = _check_int32("lengths", lengths, 1, B)
    if not 0 < tables.shape[1] * block <= MAX_LENGTH:
        raise ValueError(f"tables must have columns, for at most {MAX_LENGTH} tokens")
    if (suffix_k is None) != (suffix_v is None):
        raise ValueError("give both suffix_k and suffix_v or neither")
    if suffix_k is not None:
        s = suffix_k.shape
        if len(s) != 4 or s[0] != BW or s[1] < T or s[2] != HK or s[3] != D or \
                suffix_v.shape != s:
            raise ValueError("suffix_k and suffix_v must be [B*W, Tk, HK, D] with Tk >= T")
        if s[1] > MAX_SUFFIX:
            raise ValueError(f"a suffix has at most {MAX_SUFFIX} keys")
        if suffix_k.dtype is not dtype or suffix_v.dtype is not dtype:
            raise ValueError("attention inputs must have the same dtype")
    if gate is not None and (gate.shape != (BW, T, H * D) or gate.dtype is not dtype):
        raise ValueError("gate must be [B*W, T, H*D] in the query dtype")
    if torch.is_grad_enabled() and any(x is not None and x.requires_grad
                                       for x in (q, suffix_k, suffix_v, gate)):
        raise RuntimeError("kadllm_amd operators are inference-only; disable gradients")
    _device_of(q, tables, lengths, suffix_k, suffix_v, gate, *blocks)
    return _block_attention(q, blocks, tables, lengths, suffix_k, suffix_v, beam_width,
                            D ** -0.5 if scale is None else scale,
                            gate if gate is None else gate.view(BW, T, H, D))


def _rows(t):
    """(t, its address, its first three strides); a copy where t's rows do not
    start at 16-byte boundaries (of 16-bit elements)."""
    a, b, c, d = t.stride()
    p = t.data_ptr()
    if d != 1 or (a | b | c) & 7 or p & 15:
        t = t.clone(memory_format=torch.contiguous_format)
        a, b, c, _ = t.stride()
        p = t.data_ptr()
    return t, p, a, b, c


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(*sizes):
    need = ctypes.c_int64(0)
    _lib.call("kad_block_prefix_attention_workspace_bytes", *sizes, ctypes.byref(need))
    return need.value


_NONE = (None, None, 0, 0, 0)


def _block_attention(q, blocks, tables, lengths, suffix_k, suffix_v, beam_width, scale,
                     gate=None):
    """block_prefix_attention on checked arguments, with ``gate`` [B*W, T, H, D]
    of any strides."""
    BW, T, H, D = q.shape
    k, v, k_scale, v_scale = blocks
    pages, HK, block, _ = k.shape
    B, width = BW // beam_width, tables.shape[1]
    q, *q_at = _rows(q)
    Tk = 0 if suffix_k is None else suffix_k.shape[1]
    sk, *sk_at = _NONE if suffix_k is None else _rows(suffix_k)
    sv, *sv_at = _NONE if suffix_v is None else _rows(suffix_v)
    g, *g_at = _NONE if gate is None else _rows(gate)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    need = _workspace_bytes(B, beam_width, T, H, HK, D, width, block)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    _launch(q.get_device(), "kad_block_prefix_attention", *q_at, k.data_ptr(), v.data_ptr(),
            k_scale.data_ptr(), v_scale.data_ptr(), pages, tables.data_ptr(), width,
            lengths.data_ptr(), *sk_at, *sv_at, *g_at, out.data_ptr(), T * H * D, H * D, D,
            _lib.ptr(ws), need, B, beam_width, T, Tk, H, HK, D, block, _lib.DTYPE_CODES[q.dtype],
            float(scale))
    return out


class PagedPrefix(NamedTuple):
    """An attention layer's prefix in the 8-bit cache, in the place of the
    layer's (K, V) pair."""

    blocks: PrefixBlocks
    tables: torch.Tensor
    lengths: torch.Tensor


def paged_prefixes(pairs, *, block_size=64):
    """PagedPrefix for each (K, V) of ``pairs``, all [B, L, HK, D] of one shape: one
    table for all layers, a pool each."""
    K = pairs[0][0]
    B, L, HK, D = K.shape
    device = K.device
    width = -(-L // block_size)
    lengths = torch.full((B,), L, dtype=torch.int32, device=device)
    tables, _ = prefix_block_tables(lengths, torch.arange(B * width, dtype=torch.int32,
                                                          device=device),
                                    block_size=block_size, max_length=L)
    return [PagedPrefix(write_prefix_blocks(
        PrefixBlocks.empty(B * width, HK, D, block_size=block_size, device=device), k, v, tables,
        lengths), tables, lengths) for k, v in pairs]


def paged_attention_decode(q, prefix, suffix_k, suffix_v, beam_width, scale, gate, gate_strides):
    """attention.prefix_attention_decode over a PagedPrefix: ``gate`` any tensor
    whose data pointer is head 0's gate with strides ``gate_strides`` = (beam,
    token, head)."""
    gate = gate.as_strided(q.shape, (*gate_strides, 1))
    return _block_attention(q, *prefix, suffix_k, suffix_v, beam_width, scale, gate)
