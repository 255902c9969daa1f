"""4-bit weights on the GPU: quantising, reading back, and the products, against the
oracle in 64 bits.

Tolerances.  A product of a bf16 piece and a weight is exact in fp32; a sum of n
terms in any order is off by at most n 2^-24 of the sum of their magnitudes, twice that
where an add truncates.  A result is rounded once, by half a step of its type (fp16
below 2^-14: 2^-25).  The feed-forward block's middle product is off by its own
rounding, by its two sums' errors and by 2^-20 for its exponential."""

import pytest
import torch

from kadllm_amd.ops import (QuantizedWeight, dequantize_weight, quantize_weight,
                            quantized_gated_ffn, quantized_linear)
from oracle import quantized_ref as ref

pytestmark = pytest.mark.gpu

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U8 = torch.uint8
PIECES = {BF: 1, F16: 2, F32: 3}


def _values(shape, seed, dtype=F32, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.randn(shape[-1], generator=g).exp()
    return x.to(dtype).to(device)


def _check_parts(q, w):
    """q holds exactly the oracle's codes and scales of w."""
    codes, exps = ref.quantize(w)
    got = q.unpack()
    want = ref.parts(codes, exps)
    scales = got[1].view(U8).cpu()
    assert torch.equal(scales, want[1])
    ok = (exps != 128).repeat_interleave(32, 1)[:, :w.shape[1]]
    both = [torch.stack((c & 15, c >> 4), 2).flatten(1)[:, :w.shape[1]]
            for c in (got[0].cpu(), want[0])]
    assert torch.equal(both[0][ok], both[1][ok])
    return codes, exps


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("N, K", [(1, 1), (16, 128), (17, 129), (3, 512), (40, 1031), (130, 96),
                                  (64, 2050)])
def test_quantize_and_read_back(device, N, K, dtype):
    w = _values((N, K), N * K, dtype)
    q = quantize_weight(w)
    codes, exps = _check_parts(q, w)
    again = QuantizedWeight.pack(*q.unpack(), cols=K)
    assert torch.equal(again.codes, q.codes)  # the padding too
    assert torch.equal(again.scales.view(U8), q.scales.view(U8))
    exact = ref.dense(codes, exps)
    for out in (BF, F16, F32):
        assert torch.equal(dequantize_weight(q, out).cpu(), exact.to(out)), out


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("N, K", [(5, 2), (20, 7), (33, 8), (18, 9), (300, 131), (70, 260)])
def test_quantize_rows_that_begin_anywhere(device, N, K, dtype):
    # rows shorter and longer than what is loaded at once, each at another alignment
    w = _values((N, K + 5), N + K, dtype)[:, 3:3 + K]
    q = quantize_weight(w)
    codes, exps = _check_parts(q, w)
    exact = ref.dense(codes, exps)
    assert torch.equal(dequantize_weight(q, dtype).cpu(), exact.to(dtype))


def test_quantize_every_midpoint(device):
    # every code, every midpoint and its neighbours, for scales over the whole range
    a = torch.tensor([0, .25, .5, .75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7],
                     dtype=torch.float64)
    rows = []
    for e in [-101, -100, -99, -60, -24, -14, -1, 0, 1, 9, 60, 100, 124, 125]:
        base = a * 2.0 ** e
        up, down = (torch.nextafter(base.float(), torch.tensor(x)) for x in (1e38, 0.0))
        for part in (base.float(), up, down):
            part = part.clamp(max=torch.finfo(F32).max)
            rows.append(torch.cat((part[:-1], -part[:-1], part[-2:])))
            rows.append(torch.cat((part[:-1], -part[:-1], part[-1:], -part[:1])))
    w = torch.stack(rows)
    q = quantize_weight(w.cuda())
    codes, exps = _check_parts(q, w)
    assert torch.equal(dequantize_weight(q, F32).cpu(), ref.dense(codes, exps).float())


def test_quantize_extremes(device):
    big = torch.finfo(F32).max
    w = torch.zeros(8, 96)
    w[0, 3] = big
    w[1] = 1e-45
    w[2, 40] = float("inf")
    w[3, 70] = float("nan")
    w[4, :] = -big
    w[5, 0], w[5, 95] = -0.0, 2.0 ** -126
    w[6, 33] = 7.5 * 2.0 ** 125
    q = quantize_weight(w.cuda())
    codes, exps = _check_parts(q, w)
    back = dequantize_weight(q, F32).cpu()
    exact = ref.dense(codes, exps)
    assert torch.equal(back.isnan(), exact.isnan())
    assert back[2, 32:64].isnan().all() and back[3, 64:].isnan().all()
    assert torch.equal(back.nan_to_num(0), exact.nan_to_num(0).float())


@pytest.mark.parametrize("dtype", [BF, F32])
def test_quantize_strided(device, dtype):
    wide = _values((70, 301), 5, dtype)
    for w in (wide[3:60, 7:240], wide[:, 8:264], wide.T, wide[::2, :128], wide[:1, 3:5],
              wide[:, :1].expand(70, 40)):
        a, b = quantize_weight(w), quantize_weight(w.contiguous())
        assert torch.equal(a.codes, b.codes)
        assert torch.equal(a.scales.view(U8), b.scales.view(U8))


# ----------------------------------------------------------------------------
# products

def _weight(N, K, seed):
    """(QuantizedWeight, its values in float64 on the CPU)."""
    w = _values((N, K), seed) * K ** -0.5
    q = quantize_weight(w)
    return q, dequantize_weight(q, F32).cpu().double()


def _bound(y, size, terms, dtype):
    tiny = 2.0 ** -25 if dtype is F16 else 0.0
    return terms * 2.0 ** -23 * size + torch.finfo(dtype).eps / 2 * y.abs() * 1.01 + tiny


def _assert_linear(out, x, dense, residual=None):
    y, size = ref.linear(x, dense, residual)
    err = (out.double().cpu() - y).abs()
    bound = _bound(y, size, PIECES[x.dtype] * x.shape[-1] + 2, x.dtype)
    assert (err <= bound).all(), (err - bound).max().item()


SHAPES = [(1, 16, 128), (1, 1, 1), (1, 1024, 3584), (2, 33, 127), (7, 200, 1000), (15, 16, 2048),
          (16, 48, 384), (17, 1000, 129), (33, 31, 640), (50, 4001, 512), (64, 64, 64),
          (65, 130, 1030), (129, 257, 256), (300, 70, 2007), (513, 300, 130)]


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("M, N, K", SHAPES)
def test_linear(device, M, N, K, dtype):
    q, dense = _weight(N, K, M + N)
    x = _values((M, K), K, dtype)
    _assert_linear(quantized_linear(x, q), x, dense)
    r = _values((M, N), 7, dtype)
    _assert_linear(quantized_linear(x, q, residual=r), x, dense, r)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("M, N, K", [(1000, 130, 3000), (1100, 200, 2048), (530, 70, 5001),
                                     (37, 5001, 300), (100, 5000, 200), (200, 2700, 140)])
def test_linear_in_other_orders_of_workgroups(device, M, N, K, dtype):
    # rows of more bytes than an L2 holds, and than the weight; column tiles that are no
    # whole rounds of the 8 XCDs
    q, dense = _weight(N, K, M + N)
    x = _values((M, K), K, dtype)
    r = _values((M, N), 7, dtype)
    _assert_large(quantized_linear(x, q, residual=r), x, dense, r)


# one shape for each tile of the kernel of many rows, and for rows that it splits first
LARGE = [(700, 1900, 256), (1100, 3000, 300), (1100, 5000, 128), (4000, 8192, 130),
         (2000, 1030, 640), (25, 43000, 200), (1300, 2100, 328)]


def _assert_large(out, x, dense, residual=None):
    """_assert_linear in float64 on the GPU."""
    xd, w = x.double(), dense.cuda()
    y, size = xd @ w.T, xd.abs() @ w.abs().T
    if residual is not None:
        y, size = y + residual.double(), size + residual.double().abs()
    bound = _bound(y, size, PIECES[x.dtype] * x.shape[-1] + 2, x.dtype)
    err = (out.double() - y).abs()
    assert (err <= bound).all(), (err - bound).max().item()


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("M, N, K", LARGE)
def test_linear_of_many_rows(device, M, N, K, dtype):
    q, dense = _weight(N, K, M + N)
    x = _values((M, K), K, dtype)
    r = _values((M, N), 7, dtype)
    _assert_large(quantized_linear(x, q, residual=r), x, dense, r)
    # rows inside a wider buffer, at odd places of it
    wide = _values((M, K + 19), K + 1, dtype)
    for x in (wide[:, 8:8 + K], wide[:, 3:3 + K]):
        _assert_large(quantized_linear(x, q), x, dense)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("M, N, K", LARGE)
def test_many_rows_exactly(device, M, N, K, dtype):
    # whole numbers, every sum of which is one: nothing is lost or added
    g = torch.Generator().manual_seed(M)
    w = ref.values()[torch.randint(0, 16, (N, K), generator=g)].float()
    w[:, ::32] = 6.0
    q = quantize_weight(w.cuda())
    x = torch.randint(-4, 5, (M, K), generator=g).cuda()
    want = x.double() @ w.double().cuda().T
    got = quantized_linear(x.to(dtype), q)
    assert torch.equal(got, want.to(dtype))
    # a row that is not finite leaves the others alone
    y = x.to(dtype)
    y[M // 2, K - 1] = float("inf")
    y[M - 1, 0] = float("nan")
    out = quantized_linear(y, q)
    assert not out[M // 2].isfinite().any() and out[M - 1].isnan().all()
    rest = [m for m in range(M) if m not in (M // 2, M - 1)]
    assert torch.equal(out[rest], got[rest])


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("M, N, K", [(9, 100, 200), (700, 1900, 264), (1100, 3000, 8),
                                     (1100, 5000, 392), (4000, 8192, 72)])
def test_what_is_beside_the_rows_is_not_read(device, M, N, K, dtype):
    # rows at whole 16 bytes, which end inside a block of columns, in a buffer of NaN
    q, dense = _weight(N, K, M + N)
    wide = torch.full((M, K + 128), float("nan"), dtype=dtype, device="cuda")
    wide[:, 8:8 + K] = _values((M, K), K, dtype)
    x = wide[:, 8:8 + K]
    _assert_large(quantized_linear(x, q), x, dense)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("M, K", [(3, 40), (70, 200), (21000, 40)])
@pytest.mark.parametrize("N", [1, 2, 3, 4, 5])
def test_linear_of_few_columns(device, M, N, K, dtype):
    # fewer columns than are stored at once; a residual inside a wider buffer, at an odd place
    q, dense = _weight(N, K, M + N)
    x = _values((M, K), K, dtype)
    r = _values((M, N + 6), 7, dtype)[:, 3:3 + N]
    _assert_large(quantized_linear(x, q, residual=r), x, dense, r)
    _assert_large(quantized_linear(x, q), x, dense)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("M", [1, 3, 16, 40, 100, 260, 600])
def test_linear_whole_numbers_are_exact(device, M, dtype):
    # small whole numbers: every sum is one, in any order, so nothing may be lost
    g = torch.Generator().manual_seed(M)
    N, K = 150, 1500
    w = torch.tensor(ref.values().tolist())[torch.randint(0, 16, (N, K), generator=g)]
    w[:, ::32] = 6.0  # a scale of one for every group
    x = torch.randint(-4, 5, (M, K), generator=g).to(dtype)
    q = quantize_weight(w.cuda())
    assert torch.equal(dequantize_weight(q, F32).cpu(), w)
    want = (x.double() @ w.double().T).to(dtype)
    assert torch.equal(quantized_linear(x.cuda(), q).cpu(), want)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("M", [1, 30, 70, 300])
def test_linear_keeps_every_bit_of_x(device, M, dtype):
    # one weight of 1 in a row: y is x itself
    K = 256
    g = torch.Generator().manual_seed(M)
    x = torch.randn(M, K, generator=g, dtype=F32) * torch.exp(8 * torch.randn(M, K, generator=g))
    if dtype is F16:
        x = x.clamp(-65504, 65504)
    x = x.to(dtype).cuda()
    order = torch.randperm(K, generator=g)
    q = quantize_weight(torch.eye(K)[order].cuda())
    assert torch.equal(quantized_linear(x, q), x[:, order.cuda()])


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("M", [1, 20, 90, 300])
def test_linear_strided_rows(device, M, dtype):
    q, dense = _weight(100, 256, 3)
    wide = _values((M, 700), 4, dtype)
    odd = _values((M, 301), 5, dtype)
    rows = _values((2 * M, 256), 6, dtype)
    for x in (wide[:, 8:264], wide[:, 3:259], odd[:, 40:296], rows[::2], wide.T[:256].T,
              wide[:1, :256].expand(M, 256)):
        _assert_linear(quantized_linear(x, q), x, dense)
    out = torch.full((M, 300), 5.0, dtype=dtype, device="cuda")
    r = wide[:, 300:400]
    from kadllm_amd.quantized import _linear
    x = wide[:, 8:264]
    for first in (0, 3, 8):
        view = out[:, first:first + 100]
        _linear(x, q, view, r)
        _assert_linear(view, x, dense, r)
        assert bool((out[:, :first] == 5).all() and (out[:, first + 100:] == 5).all())
        out.fill_(5.0)
    # into the residual itself
    y = r.clone()
    want = quantized_linear(x, q, residual=r)
    _linear(x, q, y, y)
    assert torch.equal(y, want)


def test_linear_batched_shapes(device):
    q, dense = _weight(40, 200, 8)
    x = _values((3, 5, 200), 9, BF)
    out = quantized_linear(x, q)
    assert out.shape == (3, 5, 40) and out.dtype is BF
    assert torch.equal(out.view(15, 40), quantized_linear(x.view(15, 200), q))
    assert quantized_linear(x[0, 0], q).shape == (40,)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("M", [5, 40, 200, 300])
def test_linear_special_values(device, M, dtype):
    # a row with an infinity or NaN is what the definition gives, the others do not see it
    N, K = 90, 300
    q, dense = _weight(N, K, 21)
    x = _values((M, K), 22, dtype)
    clean = quantized_linear(x, q)
    x[1, 299] = float("inf")
    x[3, 0] = float("nan")
    out = quantized_linear(x, q).double().cpu()
    want = ref.linear(x[1:2], dense)[0][0]
    assert torch.equal(out[1].isnan(), want.isnan())
    assert torch.equal(out[1].isinf(), want.isinf())
    fine = want.isinf()
    assert torch.equal(out[1][fine], want[fine])
    assert out[3].isnan().all()
    rest = [m for m in range(M) if m not in (1, 3)]
    assert torch.equal(out[rest], clean[rest].double().cpu())


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("M", [1, 40, 300])
def test_a_group_that_is_not_a_number(device, M, dtype):
    w = _values((40, 200), 31)
    w[7, 50] = float("nan")
    w[20, 199] = float("inf")
    q = quantize_weight(w)
    out = quantized_linear(_values((M, 200), 32, dtype), q)
    assert out[:, 7].isnan().all() and out[:, 20].isnan().all()
    rest = [n for n in range(40) if n not in (7, 20)]
    assert out[:, rest].isfinite().all()


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("M, N", [(1, 50), (4, 50), (5, 300), (40, 300), (700, 1900), (1100, 3000),
                                  (1100, 5000), (4000, 8192)])
def test_scales_of_every_size(device, M, N, dtype):
    # most weights' scales are exact in fp16; here some groups' are far from it, in some row
    # blocks and columns of all
    K = 520
    w = _values((N, K), 41) * 0.04
    w[N // 3:N // 2, 130:250] *= 2.0 ** -25
    w[-7:, :32] *= 2.0 ** -60
    w[-1, 500:] *= 2.0 ** -100
    x = _values((M, K), 42, dtype)
    q = quantize_weight(w)
    dense = dequantize_weight(q, F32).cpu().double()
    _assert_large(quantized_linear(x, q), x, dense)
    # tiny weights alone: only their own products may be off, and only by a sum's rounding
    tiny = quantize_weight(w * 2.0 ** -25)
    big = (_values((M, K), 43) * 2.0 ** 7).clamp(-60000, 60000).to(dtype)
    _assert_large(quantized_linear(big, tiny), big, dequantize_weight(tiny, F32).cpu().double())
    # and huge ones
    huge = quantize_weight(w * 2.0 ** 20)
    small = (x.float() * 2.0 ** -19).to(dtype)
    _assert_large(quantized_linear(small, huge), small, dequantize_weight(huge, F32).cpu().double())


# ----------------------------------------------------------------------------
# the feed-forward block

def _assert_ffn(out, x, gate, up, down, residual=None):
    dtype, P = x.dtype, PIECES[x.dtype]
    (g, gs), (u, us) = ref.linear(x, gate), ref.linear(x, up)
    h = ref.silu(g) * u
    terms = (P * x.shape[-1] + 2) * 2.0 ** -23
    # |silu'| <= 1.1; the exponential, the quotient and the product; h's own rounding: a
    # bf16's step is 2^-7 of its leading bit, so rounding to one is off by 2^-8; what is
    # left behind a truncated piece is below 2^-7, of which the last piece's rounding
    # leaves 2^-8
    own = {BF: 2.0 ** -8, F16: 2.0 ** -15, F32: 2.0 ** -22}[dtype]
    err_h = 1.1 * terms * gs * u.abs() + terms * us * ref.silu(g).abs() + \
        (own + 2.0 ** -20) * h.abs() + 1.1 * terms ** 2 * gs * us
    y, size = ref.linear(h, down, residual)
    size_h = h.abs() + err_h
    n = (P * h.shape[1] + 2) * 2.0 ** -23
    size = size_h @ down.abs().T + (0 if residual is None else residual.double().cpu().abs())
    bound = err_h @ down.abs().T + n * size + torch.finfo(dtype).eps / 2 * y.abs() * 1.01
    bound = bound * 1.01 + (2.0 ** -25 if dtype is F16 else 0)
    err = (out.double().cpu() - y).abs()
    assert (err <= bound).all(), (err - bound).max().item()


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("M, H, F", [(1, 64, 128), (1, 1024, 3584), (3, 1, 1), (5, 100, 37),
                                     (16, 128, 200), (19, 333, 501), (40, 256, 1000),
                                     (70, 128, 129), (256, 128, 384), (300, 100, 77),
                                     (600, 256, 250)])
def test_ffn(device, M, H, F, dtype):
    (gate, g), (up, u), (down, d) = _weight(F, H, 1), _weight(F, H, 2), _weight(H, F, 3)
    x = _values((M, H), 4, dtype)
    _assert_ffn(quantized_gated_ffn(x, gate, up, down), x, g, u, d)
    r = _values((M, H), 5, dtype)
    _assert_ffn(quantized_gated_ffn(x, gate, up, down, residual=r), x, g, u, d, r)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("M, H, F", [(1000, 1100, 700), (1500, 256, 2000), (4000, 128, 4096)])
def test_ffn_of_many_rows(device, M, H, F, dtype):
    (gate, g), (up, u), (down, d) = _weight(F, H, 1), _weight(F, H, 2), _weight(H, F, 3)
    x = _values((M, H), 4, dtype)
    out = quantized_gated_ffn(x, gate, up, down, residual=x)
    # every tile of rows, the last ones among them
    rows = torch.cat((torch.arange(0, M, 37), torch.arange(M - 20, M)))
    _assert_ffn(out[rows.cuda()], x[rows.cuda()], g, u, d, x[rows.cuda()])


def test_ffn_strided_and_batched(device):
    H, F = 128, 96
    (gate, g), (up, u), (down, d) = _weight(F, H, 1), _weight(F, H, 2), _weight(H, F, 3)
    wide = _values((6, 300), 6, BF)
    for x in (wide[:, 8:136], wide[:, 5:133], wide.T[:128].T):
        _assert_ffn(quantized_gated_ffn(x, gate, up, down, residual=x), x, g, u, d, x)
    x = _values((2, 3, H), 7, BF)
    out = quantized_gated_ffn(x, gate, up, down, residual=x)
    assert torch.equal(out.view(6, H),
                       quantized_gated_ffn(x.view(6, H), gate, up, down, residual=x.view(6, H)))


def test_ffn_far_gates(device):
    # gates far below zero give zeros, far above the other projection; fp16 rows whose
    # middle product leaves their range
    H = 32
    one = quantize_weight(torch.eye(H, device="cuda"))
    x = torch.zeros(2, H, device="cuda", dtype=F32)
    x[0], x[1] = -1000.0, 1000.0
    out = quantized_gated_ffn(x, one, one, one)
    assert bool((out[0].abs() == 0).all()) and bool((out[1] == 1e6).all())
    small = quantize_weight(torch.eye(H, device="cuda") * 2.0 ** -10)
    out = quantized_gated_ffn(x.to(F16), one, one, small)
    assert bool((out[1] == 1e6 / 1024).all() | ((out[1] - 1e6 / 1024).abs() <= 0.5).all())


def test_ffn_row_with_an_infinity(device):
    (gate, g), (up, u), (down, d) = _weight(70, 40, 1), _weight(70, 40, 2), _weight(40, 70, 3)
    x = _values((9, 40), 8, BF)
    clean = quantized_gated_ffn(x, gate, up, down)
    x[4, 7] = float("nan")
    out = quantized_gated_ffn(x, gate, up, down)
    assert out[4].isnan().all()
    rest = [m for m in range(9) if m != 4]
    assert torch.equal(out[rest], clean[rest])


# ----------------------------------------------------------------------------
# as a program uses them

def _block(x, weights, head):
    """A tiny model: two residual feed-forward blocks and a head."""
    for gate, up, down in weights:
        x = quantized_gated_ffn(x, gate, up, down, residual=x)
    return quantized_linear(x, head)


def _model(dtype):
    H, F, V = 192, 320, 1001
    weights = [[quantize_weight(_values(s, i * 3 + j) * s[1] ** -0.5)
                for j, s in enumerate(((F, H), (F, H), (H, F)))] for i in range(2)]
    return weights, quantize_weight(_values((V, H), 11) * H ** -0.5), _values((24, H), 12, dtype)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
def test_a_model_of_blocks(device, dtype):
    weights, head, x = _model(dtype)
    out = _block(x, weights, head)
    y = x.double().cpu()
    for w in weights:
        y = ref.gated_ffn(y, *(dequantize_weight(q, F32).double() for q in w), residual=y)
        y = y.to(dtype).double()
    y = ref.linear(y, dequantize_weight(head, F32).double())[0]
    # the products of the second block reach 3.7e6 in most rows, past fp16: those rows
    # are infinite in the stream, and not numbers behind the head, where others pass it too
    fine = y.to(dtype).isfinite().all(1)
    assert fine.all() if dtype is not F16 else 0 < fine.sum() < 24
    out = out.double().cpu()
    assert torch.equal(out.isfinite().all(1), fine)
    # the stream is rounded three times and the middle products twice: relative to the
    # size of the whole output each adds at most half a step
    err = (out - y)[fine].norm() / y[fine].norm()
    assert err <= 5 * torch.finfo(dtype).eps / 2 + 2.0 ** -16


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("M", [1, 24, 300])
def test_captured_and_replayed(device, M, dtype):
    weights, head, x = _model(dtype)
    x = x[:1].expand(M, -1).contiguous() if M > 24 else x[:M].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _block(x, weights, head)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_block(x, weights, head))
        graphs.append(graph)
    for step in range(4):
        x.copy_(_values(tuple(x.shape), 40 + step, dtype))
        want = _block(x, weights, head)
        for graph, out in zip(graphs, outs):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out.nan_to_num(nan=7.0), want.nan_to_num(nan=7.0)), step


def test_streams(device):
    weights, head, x = _model(BF)
    want = _block(x, weights, head)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for s in streams:
        with torch.cuda.stream(s):
            outs.append(_block(x, weights, head))
    torch.cuda.synchronize()
    for out in outs:
        assert torch.equal(out, want)


def test_repeated_calls_give_the_same_bits(device):
    for M in (1, 40, 300, 2500):
        q, _ = _weight(1000, 3584, 1)
        x = _values((M, 3584), 2, BF)
        first = quantized_linear(x, q)
        for _ in range(3):
            assert torch.equal(quantized_linear(x, q), first)


def test_quantised_in_a_graph(device):
    w = _values((200, 1000), 1, BF)
    x = _values((30, 1000), 2, BF)
    quantize_weight(w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = quantize_weight(w)
        back, y = dequantize_weight(q), quantized_linear(x, q)
    for step in range(3):
        w.copy_(_values((200, 1000), 5 + step, BF))
        want = quantize_weight(w)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(q.codes, want.codes)
        assert torch.equal(q.scales.view(U8), want.scales.view(U8))
        assert torch.equal(back, dequantize_weight(want))
        assert torch.equal(y, quantized_linear(x, want))


def test_offsets_past_32_bits(device):
    # a weight of 2^33 and more elements: 16384 times the same 128 rows
    n, N, K = 128, 2**21, 4224
    part = _values((n, K), 1, BF)
    q1 = quantize_weight(part)
    w = part.expand(N // n, n, K).reshape(N, K)
    q = quantize_weight(w)
    del w
    codes = q.codes.view(N // n, -1)
    assert torch.equal(codes, q1.codes.view(1, -1).expand_as(codes))
    scales = q.scales.view(U8).view(N // n, -1)
    assert torch.equal(scales, q1.scales.view(U8).view(1, -1).expand_as(scales))
    back = dequantize_weight(q).view(N // n, n, K)
    assert torch.equal(back, dequantize_weight(q1).expand_as(back))
    del back
    for M in (2, 2100):  # and 2^32 outputs and residuals
        x = torch.randint(-2, 3, (M, K), device="cuda").to(BF)
        r = torch.randint(-2, 3, (M, n), device="cuda").to(BF)
        y = quantized_linear(x, q, residual=r.repeat(1, N // n)).view(M, N // n, n)
        assert torch.equal(y, y[:, -1:].expand_as(y))
        _assert_large(y[:, -1], x, dequantize_weight(q1, F32).double(), r)
    del y, q, codes, scales
    torch.cuda.empty_cache()
