"""Weights in 4 bits, and products with them.

A ``QuantizedWeight`` holds a weight [N, K] in groups of 32 neighbours of a row:
e2m1 codes (0, 1/2, 1, 3/2, 2, 3, 4, 6 and their negatives) and one e8m0 scale (a
power of two) for each group, 4.25 bits an element.  A value is code * scale, which is
exact in bf16.

    q = quantize_weight(w)                       # or QuantizedWeight.pack(codes, scales)
    y = quantized_linear(x, q, residual=r)       # x W^T + r
    y = quantized_gated_ffn(x, gate, up, down)   # (silu(x G^T) * (x U^T)) D^T

Everything runs on the GPU without a host synchronisation (but for ``pack``, which
looks at the scales once); no counterpart in the reference, whose weights stay in the
model's type (src/kadllm/adapters/qwen3_5.py:144-235).
"""

import ctypes
import functools

import torch

from . import _lib
from .prefix_cache import _device_of, _launch

GROUP = 32                  # columns of a row that share a scale
MAX_COLS = 2**20            # columns of a weight
MAX_WEIGHT_ROWS = 2**26     # rows of a weight
MAX_ROWS = 16 * 65535       # rows of x
_TYPES = (torch.bfloat16, torch.float16, torch.float32)
_SCALES = torch.float8_e8m0fnu


def _padded(rows, cols):
    """The shapes of a weight's codes and scales."""
    nb, kb = -(-rows // 16), -(-cols // 128)
    return (nb, kb, 64, 16), (nb, kb, 16, 4)


class QuantizedWeight:
    """A weight [rows, cols] in 4 bits, as quantized_linear reads it: codes uint8
    [rows/16, cols/128, 64, 16] (sizes rounded up), of which bytes 4 j to 4 j + 3 of
    entry l of a block are row l % 16, columns 32 j + 8 (l // 16) to + 7, and scales
    torch.float8_e8m0fnu [rows/16, cols/128, 16 rows, 4 groups].  Types and sizes are
    checked when it is made, and it is not changed afterwards; scales outside 2**-100 to
    2**125 (which ``pack`` refuses) give undefined values."""

    __slots__ = ("codes", "scales", "rows", "cols")

    def __init__(self, codes, scales, rows, cols):
        if codes.dtype is not torch.uint8 or scales.dtype is not _SCALES:
            raise TypeError("the codes of a weight are uint8 and its scales float8_e8m0fnu")
        _check_size(rows, cols)
        if (codes.shape, scales.shape) != _padded(rows, cols):
            raise ValueError("codes and scales do not fit the weight's size")
        if not (codes.is_contiguous() and scales.is_contiguous()):
            raise ValueError("the tensors of a 4-bit weight must be contiguous")
        if codes.device != scales.device:
            raise ValueError("all tensors must be on the same device")
        self._set(codes, scales, rows, cols)

    def _set(self, *values):
        for name, value in zip(self.__slots__, values):
            object.__setattr__(self, name, value)
        return self

    def __setattr__(self, name, value):
        raise AttributeError("a QuantizedWeight is not changed; make another")

    def __reduce__(self):
        return type(self), (self.codes, self.scales, self.rows, self.cols)

    def __repr__(self):
        return f"QuantizedWeight({self.rows} x {self.cols}, {self.codes.device})"

    def row_range(self, first, last):
        """The rows first to last - 1 (multiples of 16, or the end), sharing memory."""
        if first % 16 or last % 16 and last != self.rows or not 0 <= first < last <= self.rows:
            raise ValueError("a range of rows begins and ends at multiples of 16")
        blocks = slice(first // 16, -(-last // 16))
        return QuantizedWeight(self.codes[blocks], self.scales[blocks], last - first, self.cols)

    def to(self, device):
        """This weight on another device."""
        return QuantizedWeight(self.codes.to(device), self.scales.to(device), self.rows, self.cols)

    @classmethod
    def pack(cls, codes, scales, *, cols=None):
        """From row-major parts: codes [N, ceil(K / 2)] (uint8, or
        torch.float4_e2m1fn_x2, the even column in a byte's low half) and scales
        [N, ceil(K / 32)] (torch.float8_e8m0fnu or its bytes as uint8), from 2**-100
        to 2**125 or NaN; a group of zeros may have 2**-127 (byte 0) too, as it is
        commonly stored, and gets 1.  ``cols`` is K (default: two for each byte)."""
        if codes.dtype is torch.float4_e2m1fn_x2:
            codes = codes.view(torch.uint8)
        if scales.dtype is _SCALES:
            scales = scales.view(torch.uint8)
        if codes.dtype is not torch.uint8 or scales.dtype is not torch.uint8:
            raise TypeError("codes are uint8 or float4_e2m1fn_x2, scales float8_e8m0fnu or uint8")
        if codes.ndim != 2 or scales.ndim != 2 or 0 in codes.shape:
            raise ValueError("codes must be [N, K / 2] and scales [N, K / 32]")
        N, half = codes.shape
        K = 2 * half if cols is None else cols
        _check_size(N, K)
        if half != -(-K // 2) or scales.shape != (N, -(-K // GROUP)):
            raise ValueError("codes must be [N, K / 2] and scales [N, K / 32]")
        if codes.device != scales.device:
            raise ValueError("all tensors must be on the same device")
        if K % 2:
            codes = torch.cat((codes[:, :-1], codes[:, -1:] & 15), 1)
        pad = torch.nn.functional.pad
        bad = (scales < 27) | ((scales > 252) & (scales < 255))
        if bool(bad.any()):
            nonzero = (pad(codes, (0, -half % 16)).reshape(N, -1, 16) & 0x77).ne(0).any(2)
            unused = (scales == 0) & ~nonzero
            if bool((bad & ~unused).any()):
                raise ValueError("scales must be from 2**-100 to 2**125, or NaN")
            scales = scales.masked_fill(unused, 127)
        nb, kb = _padded(N, K)[0][:2]
        codes = pad(codes, (0, kb * 64 - half, 0, nb * 16 - N))
        codes = codes.view(nb, 16, kb, 4, 4, 4).permute(0, 2, 4, 1, 3, 5)
        scales = pad(scales, (0, kb * 4 - scales.shape[1], 0, nb * 16 - N), value=127)
        scales = scales.view(nb, 16, kb, 4).transpose(1, 2)
        return cls(codes.reshape(nb, kb, 64, 16), scales.contiguous().view(_SCALES), N, K)

    def unpack(self):
        """(codes [N, ceil(K / 2)] uint8, scales [N, ceil(K / 32)] float8_e8m0fnu):
        the row-major parts that ``pack`` takes."""
        nb, kb = self.codes.shape[:2]
        codes = self.codes.view(nb, kb, 4, 16, 4, 4).permute(0, 3, 1, 4, 2, 5).reshape(nb * 16, -1)
        scales = self.scales.view(torch.uint8).transpose(1, 2).reshape(nb * 16, -1)
        scales = scales[:self.rows, :-(-self.cols // GROUP)]
        return (codes[:self.rows, :-(-self.cols // 2)].contiguous(),
                scales.contiguous().view(_SCALES))


def _check_size(rows, cols):
    if type(rows) is not int or type(cols) is not int or not 0 < rows <= MAX_WEIGHT_ROWS or \
            not 0 < cols <= MAX_COLS:
        raise ValueError(f"a weight has 1 to {MAX_WEIGHT_ROWS} rows of 1 to {MAX_COLS} columns")


def _check_weight(w, name="weight"):
    if type(w) is not QuantizedWeight:
        raise TypeError(f"{name} must be a QuantizedWeight")


def _rows(t):
    """t [M, C] with a contiguous last dimension and rows that do not overlap, and
    the stride of its rows."""
    M, C = t.shape
    ld, one = t.stride()
    if one == 1 and ld >= C:
        return t, ld
    if one != 1 and C > 1 or M > 1:
        t = t.contiguous()
    return t, C


def quantize_weight(weight):
    """``weight`` [N, K] (bf16, fp16 or fp32, any strides) in 4 bits.

    A group's scale is the smallest power of two s, from 2**-100 to 2**125, with amax <=
    7 s (1 for a group of zeros); its codes are w / s to the nearest e2m1 value, ties to
    the even code, at most 6.  An element is off by up to s / 4 below 2 s, s / 2 below 4 s
    and s above.
    A group that holds an infinity or NaN reads as NaN.  Columns past K and rows past N
    of the padded arrays are zeros.  Returns a QuantizedWeight."""
    if weight.ndim != 2 or 0 in weight.shape:
        raise ValueError("a weight must be [N, K]")
    if weight.dtype not in _TYPES:
        raise TypeError("weights must be bf16, fp16 or fp32")
    N, K = weight.shape
    _check_size(N, K)
    if torch.is_grad_enabled() and weight.requires_grad:
        raise RuntimeError("kadllm_amd operators are inference-only; disable gradients")
    device = _device_of(weight)
    weight, ld = _rows(weight)
    shapes = _padded(N, K)
    codes = weight.new_empty(*shapes[0], dtype=torch.uint8)
    scales = weight.new_empty(*shapes[1], dtype=_SCALES)
    _launch(device, "kad_quantize_weight", weight.data_ptr(), ld, _lib.dtype_code(weight.dtype),
            codes.data_ptr(), scales.data_ptr(), N, K)
    return QuantizedWeight.__new__(QuantizedWeight)._set(codes, scales, N, K)


def dequantize_weight(weight, dtype=torch.bfloat16):
    """The values [N, K] of a QuantizedWeight in ``dtype`` (bf16 and fp32: exactly)."""
    _check_weight(weight)
    if dtype not in _TYPES:
        raise TypeError("weights must be bf16, fp16 or fp32")
    device = _device_of(weight.codes, weight.scales)
    out = weight.codes.new_empty(weight.rows, weight.cols, dtype=dtype)
    _launch(device, "kad_dequantize_weight", weight.codes.data_ptr(), weight.scales.data_ptr(),
            out.data_ptr(), weight.cols, _lib.dtype_code(dtype), weight.rows, weight.cols)
    return out


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(name, offset, *sizes):
    """Of a call whose x is ``offset`` bytes past a 16-byte boundary."""
    need = ctypes.c_int64(0)
    _lib.call(name, offset, *sizes, ctypes.byref(need))
    return need.value


def _check_rows(x, cols, out_cols, residual):
    """x [..., cols] and residual [..., out_cols] (or None) as 2-D rows."""
    shape = x.shape
    if not shape or shape[-1] != cols or 0 in shape:
        raise ValueError(f"x must be [..., {cols}], the weight's columns, and not empty")
    if x.numel() > MAX_ROWS * cols:
        raise ValueError(f"x has at most {MAX_ROWS} rows")
    dtype = x.dtype
    if dtype not in _TYPES:
        raise TypeError("x must be bf16, fp16 or fp32")
    if residual is not None:
        if residual.shape != (*shape[:-1], out_cols):
            raise ValueError(f"residual must be x's rows of {out_cols}")
        if residual.dtype is not dtype:
            raise ValueError("x and residual must have the same dtype")
    if torch.is_grad_enabled() and (x.requires_grad or
                                    residual is not None and residual.requires_grad):
        raise RuntimeError("kadllm_amd operators are inference-only; disable gradients")
    if len(shape) != 2:
        x = x.reshape(-1, cols)
        residual = residual if residual is None else residual.reshape(-1, out_cols)
    return x, residual


def quantized_linear(x, weight, *, residual=None):
    """x W^T (+ residual) for a QuantizedWeight W [N, K].

    x [..., K] bf16, fp16 or fp32 (any strides); residual [..., N] of x's type.
    Returns [..., N] in x's type.  Products are exact, sums are fp32 and are rounded
    once, with the residual added; of fp32 rows, values below 2**-110 count to within
    2**-134 (they are taken in bf16 pieces, which end there).  fp16 rows take half as long
    where all scales are from 2**-15 to 1."""
    _check_weight(weight)
    rows, r = _check_rows(x, weight.cols, weight.rows, residual)
    _device_of(x, weight.codes, residual)
    out = _linear(rows, weight, rows.new_empty(rows.shape[0], weight.rows), r)
    return out if rows is x else out.view(*x.shape[:-1], weight.rows)


def _linear(x, weight, out, residual=None):
    """quantized_linear on checked 2-D rows, into ``out`` (rows of any stride; it
    may be ``residual``)."""
    x, ldx = _rows(x)
    M, N, K = x.shape[0], weight.rows, weight.cols
    r, ldr = (None, 0) if residual is None else _rows(residual)
    code, at = _lib.DTYPE_CODES[x.dtype], x.data_ptr()
    need = _workspace_bytes("kad_quantized_linear_workspace_bytes", at & 15, ldx, code, M, N, K)
    ws = x.new_empty(need, dtype=torch.uint8) if need else None
    _launch(x.get_device(), "kad_quantized_linear", at, ldx, code, weight.codes.data_ptr(),
            weight.scales.data_ptr(), _lib.ptr(r), ldr, out.data_ptr(), max(out.stride(0), N),
            _lib.ptr(ws), need, M, N, K)
    return out


def quantized_gated_ffn(x, gate, up, down, *, residual=None):
    """(silu(x G^T) * (x U^T)) D^T (+ residual) for QuantizedWeights gate and up
    [F, H] and down [H, F].

    x [..., H] bf16, fp16 or fp32 (any strides); residual [..., H] of x's type.
    Returns [..., H] in x's type.  Sums are fp32.  The product of the two
    projections, whose SiLU is computed in fp32, is held in bf16 for bf16 rows (off
    by up to 2**-8 of itself), to 2**-15 for fp16 and 2**-22 for fp32, or 2**-134."""
    for name, w in (("gate", gate), ("up", up), ("down", down)):
        _check_weight(w, name)
    F, H = gate.rows, gate.cols
    if up.rows != F or up.cols != H or down.rows != H or down.cols != F:
        raise ValueError("gate and up must be [F, H] and down [H, F]")
    rows, r = _check_rows(x, H, H, residual)
    _device_of(x, gate.codes, up.codes, down.codes, residual)
    out = _gated_ffn(rows, gate, up, down, rows.new_empty(*rows.shape), r)
    return out if rows is x else out.view(x.shape)


def _gated_ffn(x, gate, up, down, out, residual=None):
    """quantized_gated_ffn on checked 2-D rows, into ``out`` (rows of any stride; it
    may be ``residual``)."""
    x, ldx = _rows(x)
    M, F, H = x.shape[0], gate.rows, gate.cols
    r, ldr = (None, 0) if residual is None else _rows(residual)
    code, at = _lib.DTYPE_CODES[x.dtype], x.data_ptr()
    need = _workspace_bytes("kad_quantized_gated_ffn_workspace_bytes", at & 15, ldx, code, M, H, F)
    ws = x.new_empty(need, dtype=torch.uint8)
    _launch(x.get_device(), "kad_quantized_gated_ffn", at, ldx, code, gate.codes.data_ptr(),
            gate.scales.data_ptr(), up.codes.data_ptr(), up.scales.data_ptr(),
            down.codes.data_ptr(), down.scales.data_ptr(), _lib.ptr(r), ldr, out.data_ptr(),
            max(out.stride(0), H), ws.data_ptr(), need, M, H, F)
    return out
