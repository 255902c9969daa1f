"""4-bit weights on the GPU: every kernel that is compiled for their products, by calls
that reach it, against the definition in 64 bits.

The tolerances are those of test_gpu_quantized.py: a product of a bf16 piece and a weight
is exact, a sum of n terms is off by at most n 2^-23 of their magnitudes, and a result is
rounded once; where a single product makes the sum, bit for bit."""

import re

import pytest
import torch

from kadllm_amd import _lib
from kadllm_amd.ops import (dequantize_weight, quantize_weight, quantized_gated_ffn,
                            quantized_linear)

pytestmark = pytest.mark.gpu

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
TYPES = [BF, F16, F32]
PIECES = {BF: 1, F16: 2, F32: 3}

# rows x outputs x columns.  A few rows: tiles of 16, 32 and 64 columns and of 32 rows, K over
# 4 and 8 waves; many: tiles of 32 x 128 to 128 x 256, rows of whole blocks of 128 columns, of
# whole 16 bytes, and of neither
FEW = [(M, N, K) for M in (3, 13) for N in (200, 4200, 8300) for K in (200, 1700, 3100)]
FEW += [(300, 1800, 200)]
MANY = [(M, 512, K) for M in (3000, 6000, 9000, 20000) for K in (256, 200, 131)]
# rows, hidden size, width
FFN_FEW = [(M, H, F) for M in (3, 13) for H in (200, 1700, 4200, 8300) for F in (200, 1700, 4200)]
FFN_FEW += [(300, 1800, 900)]
FFN_MANY = [(M, H, 200) for M in (3000, 6000, 9000, 20000) for H in (512, 504, 500)]


def _values(shape, seed, dtype=F32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(shape, generator=g, device="cuda")
    return (x * torch.randn(shape[-1], generator=g, device="cuda").exp()).to(dtype)


def _weight(w):
    """(QuantizedWeight, its values in float64)."""
    q = quantize_weight(w)
    return q, dequantize_weight(q, F32).double()


def _inside(x, first):
    """x inside a wider buffer of NaN, from column ``first``."""
    M, K = x.shape
    wide = torch.full((M, -(-(K + 16) // 8) * 8), float("nan"), dtype=x.dtype, device="cuda")
    wide[:, first:first + K] = x
    return wide[:, first:first + K]


def _silu(x):
    return x * torch.sigmoid(x)


def _assert_linear(out, x, w, residual=None, columns=slice(None)):
    """out = x w^T + residual (in some columns) within the sums' rounding and the type's."""
    dtype, xd, w = x.dtype, x.double(), w[columns]
    y, size = xd @ w.T, xd.abs() @ w.abs().T
    if residual is not None:
        r = residual[:, columns].double()
        y, size = y + r, size + r.abs()
    bound = (PIECES[dtype] * x.shape[1] + 2) * 2.0 ** -23 * size + \
        torch.finfo(dtype).eps / 2 * y.abs() * 1.01 + (2.0 ** -25 if dtype is F16 else 0)
    err = (out[:, columns].double() - y).abs()
    assert (err <= bound).all(), (err - bound).max().item()


def _assert_ffn(out, x, gate, up, down, residual=None, columns=slice(None)):
    dtype, P, xd, down = x.dtype, PIECES[x.dtype], x.double(), down[columns]
    g, gs, u, us = xd @ gate.T, xd.abs() @ gate.abs().T, xd @ up.T, xd.abs() @ up.abs().T
    h = _silu(g) * u
    terms = (P * x.shape[1] + 2) * 2.0 ** -23
    # both sums (|silu'| <= 1.1), the exponential, and h's own rounding to its pieces
    own = {BF: 2.0 ** -8, F16: 2.0 ** -15, F32: 2.0 ** -22}[dtype]
    err_h = 1.1 * terms * gs * u.abs() + terms * us * _silu(g).abs() + \
        (own + 2.0 ** -20) * h.abs() + 1.1 * terms ** 2 * gs * us
    y, size = h @ down.T, (h.abs() + err_h) @ down.abs().T
    if residual is not None:
        r = residual[:, columns].double()
        y, size = y + r, size + r.abs()
    n = (P * h.shape[1] + 2) * 2.0 ** -23
    bound = err_h @ down.abs().T + n * size + torch.finfo(dtype).eps / 2 * y.abs() * 1.01
    bound = bound * 1.01 + (2.0 ** -25 if dtype is F16 else 0)
    err = (out[:, columns].double() - y).abs()
    assert (err <= bound).all(), (err - bound).max().item()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M, N, K", FEW + MANY)
def test_linear_in_every_tile(device, M, N, K, dtype):
    q, w = _weight(_values((N, K), 1) * K ** -0.5)
    x, r = _values((M, K), 2, dtype), _values((M, N), 3, dtype)
    _assert_linear(quantized_linear(x, q, residual=r), x, w, r)
    _assert_linear(quantized_linear(_inside(x, 3), q), x, w)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M, H, F", FFN_FEW + FFN_MANY)
def test_ffn_in_every_tile(device, M, H, F, dtype):
    gate, up, down = (_values(s, i) * s[1] ** -0.5 for i, s in enumerate(((F, H), (F, H), (H, F))))
    x, r = _values((M, H), 4, dtype), _values((M, H), 5, dtype)
    (qg, g), (qu, u), (qd, d) = map(_weight, (gate, up, down))
    _assert_ffn(quantized_gated_ffn(x, qg, qu, qd, residual=r), x, g, u, d, r)
    _assert_ffn(quantized_gated_ffn(_inside(x, 8), qg, qu, qd), x, g, u, d)
    # scales that fp16 does not hold, in some groups: far below the others, and above one
    gate[F // 3:F // 2, 130:190] *= 2.0 ** -25
    gate[5:9, 32:64] *= 64
    up[-7:, :32] *= 2.0 ** -60
    down[H // 2:, 64:96] *= 2.0 ** -30
    (qg, g), (qu, u), (qd, d) = map(_weight, (gate, up, down))
    _assert_ffn(quantized_gated_ffn(x, qg, qu, qd), x, g, u, d)


def _variants(names):
    """The products' kernels among the names, mangled or not, as (kernel, type, numbers)."""
    found = set()
    for name in names:
        m = re.search(r"(q4_(?:stream|tile)_kernel)(?:I(\w+?E)Ev|<([^<>]*)>)", name)
        if m and m.group(2):
            kind = re.match(r"DF16_|f|t", m.group(2)).group()
            found.add((m.group(1), kind, *map(int, re.findall(r"L[bi](\d+)E", m.group(2)))))
        elif m:
            kind, *rest = m.group(3).split(", ")
            kind = {"_Float16": "DF16_", "float": "f", "unsigned short": "t"}[kind]
            found.add((m.group(1), kind, *(int({"true": 1, "false": 0}.get(x, x)) for x in rest)))
    return found


def _compiled():
    """Those that the library holds."""
    with open(_lib.LIB_PATH, "rb") as f:
        names = re.findall(rb"_ZN12_GLOBAL__N_1\d+q4_(?:stream|tile)_kernelI\w+?EEv", f.read())
    return _variants(name.decode() for name in set(names))


def test_every_compiled_kernel_is_reached(device):
    # a kernel that the calls above do not run is one that no test sees, or that no call needs
    from torch.profiler import ProfilerActivity, profile

    weights = {}

    def weight(N, K):
        if (N, K) not in weights:
            weights[N, K] = quantize_weight(_values((N, K), 1))
        return weights[N, K]

    with profile(activities=[ProfilerActivity.CPU, ProfilerActivity.CUDA]) as run:
        for dtype in TYPES:
            for M, N, K in FEW + MANY:
                quantized_linear(_values((M, K), 2, dtype), weight(N, K))
            for M, H, F in FFN_FEW + FFN_MANY:
                quantized_gated_ffn(_values((M, H), 2, dtype), weight(F, H), weight(F, H),
                                    weight(H, F))
        torch.cuda.synchronize()
    names = [e.name for e in run.events()]
    if not any("kernel" in name for name in names):
        pytest.skip("the profiler reports no kernels here")
    compiled = _compiled()
    assert len(compiled) > 100
    assert compiled - _variants(names) == set()


# rows for each tile of about 500 columns
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("factor", [1.0, 8.0])
@pytest.mark.parametrize("K, first", [(512, None), (504, 8), (500, 3)])
@pytest.mark.parametrize("M", [3000, 6000, 9000, 20000])
def test_many_rows_keep_every_bit_of_x(device, M, K, first, factor, dtype):
    # one weight in a row: y is x times it.  Its scale is 1/4 (of factor 8: 2, where rows of
    # fp16 go in pieces)
    g = torch.Generator().manual_seed(M + K)
    x = torch.randn(M, K, generator=g) * torch.exp(8 * torch.randn(M, K, generator=g))
    if dtype is F16:
        x = x.clamp(-65504 / factor, 65504 / factor)
    x = x.to(dtype).cuda()
    order = torch.randperm(K, generator=g).cuda()
    q = quantize_weight(torch.eye(K, device="cuda")[order] * factor)
    rows = x if first is None else _inside(x, first)
    assert torch.equal(quantized_linear(rows, q), x[:, order] * factor)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M, N, K", [(1, 90, 256), (40, 90, 300), (300, 90, 256)] + MANY)
def test_groups_that_are_not_numbers(device, M, N, K, dtype):
    w = _values((N, K), 31)
    w[7, 50] = float("nan")
    w[N - 3, K - 1] = float("inf")
    q, dense = _weight(w)
    x = _values((M, K), 32, dtype)
    out = quantized_linear(x, q)
    assert out[:, 7].isnan().all() and out[:, N - 3].isnan().all()
    _assert_linear(out, x, dense, columns=[n for n in range(N) if n not in (7, N - 3)])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M, H, F", [(1, 64, 100), (30, 72, 200)] + FFN_MANY)
def test_ffn_groups_that_are_not_numbers(device, M, H, F, dtype):
    gate, up, down = (_values(s, i) * s[1] ** -0.5 for i, s in enumerate(((F, H), (F, H), (H, F))))
    x = _values((M, H), 4, dtype)
    down[9, F - 1] = float("nan")
    (qg, g), (qu, u), (qd, d) = map(_weight, (gate, up, down))
    out = quantized_gated_ffn(x, qg, qu, qd)
    assert out[:, 9].isnan().all()
    _assert_ffn(out, x, g, u, d, columns=[n for n in range(H) if n != 9])
    # one of the middle product's columns is in all outputs
    for bad in (gate, up):
        kept = bad[F // 2, 3].clone()
        bad[F // 2, 3] = float("inf")
        assert quantized_gated_ffn(x, *map(quantize_weight, (gate, up, down))).isnan().all()
        bad[F // 2, 3] = kept


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M, H, F", [(1, 1024, 3584), (19, 2048, 5503), (256, 1024, 3584),
                                     (9000, 500, 300), (32768, 1024, 3584)])
def test_repeated_blocks_give_the_same_bits(device, M, H, F, dtype):
    weights = [quantize_weight(_values(s, i) * s[1] ** -0.5)
               for i, s in enumerate(((F, H), (F, H), (H, F)))]
    x = _values((M, H), 4, dtype)
    want = quantized_gated_ffn(x, *weights, residual=x)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(4):
        outs = [quantized_gated_ffn(x, *weights, residual=x)]
        for stream in streams:  # at the same time
            with torch.cuda.stream(stream):
                outs.append(quantized_gated_ffn(x, *weights, residual=x))
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for out in outs)


@pytest.mark.parametrize("dtype, first", [(BF, 8), (F16, 3), (F32, 8)])
def test_rows_past_32_bits(device, dtype, first):
    # 2^32 and more elements of x: the same 1024 rows again and again, the last of them fewer
    n, K, N = 1024, 4200, 40
    M = 2 ** 32 // K // n * n + n + 9
    part = _values((n, K), 1, dtype)
    q, dense = _weight(_values((N, K), 2) * K ** -0.5)
    x = torch.empty(M, K + 8, dtype=dtype, device="cuda")[:, first:first + K]
    assert M * K > 2 ** 32
    x[:M - 9].view(-1, n, K).copy_(part.expand(M // n, n, K))
    x[M - 9:] = part[:9]
    y = quantized_linear(x, q)
    del x
    _assert_linear(y[:n], part, dense)
    assert torch.equal(y[:M - 9].view(-1, n, N), y[:n].expand(M // n, n, N))
    assert torch.equal(y[M - 9:], y[:9])
    del y
    torch.cuda.empty_cache()
