"""4-bit weights on the GPU: rows of values that are no numbers, by every tile of the
products' kernels.

Where whole numbers or single products make a sum exact, outputs are compared bit for
bit with the definition in 64 bits."""

import pytest
import torch

from kadllm_amd.ops import (QuantizedWeight, dequantize_weight, quantize_weight,
                            quantized_gated_ffn, quantized_linear)

pytestmark = pytest.mark.gpu

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
TYPES = [BF, F16, F32]

# M, N, K: one for each tile, few rows among them
SHAPES = [(1, 90, 256), (40, 90, 300), (300, 90, 256), (700, 1900, 256), (1100, 3000, 300),
          (1100, 5000, 128), (1300, 2100, 328), (4000, 8192, 130)]


def _same(got, want):
    """The same numbers, infinities and NaN."""
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(nan=0.0, posinf=float("inf"), neginf=float("-inf")),
                       want.nan_to_num(nan=0.0, posinf=float("inf"), neginf=float("-inf")))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M, N, K", SHAPES)
def test_infinities_are_what_the_definition_gives(device, M, N, K, dtype):
    # weights of 4 and 6 times a power of two of the row's: every finite sum is exact
    g = torch.Generator().manual_seed(M)
    w = torch.tensor([4.0, 6.0])[torch.randint(0, 2, (N, K), generator=g)]
    w[:, ::32] = 6.0
    w *= torch.tensor([1.0, 2.0, 2.0 ** 20, 2.0 ** -18, 2.0 ** 100])[torch.arange(N) % 5][:, None]
    w[torch.arange(N) % 3 == 1] *= -1
    q, dense = quantize_weight(w.cuda()), w.double().cuda()
    assert torch.equal(dequantize_weight(q, F32).double(), dense)
    inf = float("inf")
    many = torch.randint(0, K, (K // 3,), generator=g)
    for first in range(0, 6, min(M, 6)):  # (one row has one of them at a time)
        x = torch.randint(1, 5, (M, K), generator=g).to(dtype)
        for kind in range(first, min(first + M, 6)):
            row = x[(kind * 37) % M if M > 222 else kind % M]
            if kind == 0:
                row[K - 1] = inf
            elif kind == 1:
                row[0] = -inf
            elif kind == 2:
                row[many] = inf
            elif kind == 3:
                row[many] = -inf
            elif kind == 4:
                row[1], row[K // 2] = inf, -inf
            else:
                row[K // 3] = float("nan")
        x = x.cuda()
        _same(quantized_linear(x, q), (x.double() @ dense.T).to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M, H, F", [(2, 64, 100), (30, 72, 200), (4000, 504, 200),
                                     (9000, 500, 300)])
def test_ffn_infinities(device, M, H, F, dtype):
    # positive weights, so that an infinity goes through both halves as one
    g = torch.Generator().manual_seed(M)

    def weight(*shape):
        w = torch.tensor([4.0, 6.0])[torch.randint(0, 2, shape, generator=g)]
        w[:, ::32] = 6.0
        return quantize_weight(w.cuda() * torch.tensor([2.0 ** -10, 2.0 ** 20]).cuda()[
            torch.arange(shape[0]).cuda() % 2][:, None])

    gate, up, down = weight(F, H), weight(F, H), weight(H, F)
    x = (torch.rand(M, H, generator=g) * 2.0 ** -40).to(dtype).cuda()
    clean = quantized_gated_ffn(x, gate, up, down)
    assert clean.isfinite().all()
    x[0, 3] = float("inf")
    x[M // 2, 5], x[M // 2, H - 1] = float("inf"), float("inf")
    out = quantized_gated_ffn(x, gate, up, down)
    assert bool((out[0] == float("inf")).all()) and bool((out[M // 2] == float("inf")).all())
    rest = [m for m in range(M) if m not in (0, M // 2)]
    assert torch.equal(out[rest], clean[rest])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M, N, K", SHAPES)
def test_signalling_nan(device, M, N, K, dtype):
    # of either sign (the second is negative as a whole number); in fp32 the leading half is an
    # infinity's
    bits = {BF: (0x7f81, -0x7f), F16: (0x7c01, -0x3ff), F32: (0x7f800001, -0x7f0001)}[dtype]
    q = quantize_weight(torch.ones(N, K, device="cuda"))
    x = torch.ones(M, K, dtype=dtype)
    rows = [0, M - 1][:M]
    for m, b in zip(rows, bits):
        x.view(torch.int32 if dtype is F32 else torch.int16)[m, K // 2] = b
    assert x[rows].isnan().any(1).all()
    out = quantized_linear(x.cuda(), q)
    assert out[rows].isnan().all()
    rest = [m for m in range(M) if m not in rows]
    assert bool((out[rest] == K).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M, N", [(1, 64), (40, 64), (300, 64), (3000, 512), (9000, 512)])
def test_rows_far_below_one(device, M, N, dtype):
    # one weight of 2^100 in a row: y is x times it.  The pieces of fp32 rows end at 2^-133, the
    # lowest step of bf16: values from 2^-110 are whole, others off by up to 2^-134
    K = 512
    g = torch.Generator().manual_seed(M)
    x = torch.randn(M, K, generator=g).double()
    order = torch.randperm(K, generator=g)[:N]
    q = quantize_weight((torch.eye(K)[order] * (1.0 if dtype is F16 else 2.0 ** 100)).cuda())
    for e in (-14, -20) if dtype is F16 else (-60, -100, -109, -118, -126):
        y = (x * 2.0 ** e).to(dtype)
        out = quantized_linear(y.cuda(), q).double().cpu()
        want = y[:, order].double() * (1.0 if dtype is F16 else 2.0 ** 100)
        if dtype is not F32:
            assert torch.equal(out, want), e
        else:
            whole = want.abs() >= 2.0 ** -10
            assert torch.equal(out[whole], want[whole]), e
            assert bool(((out - want).abs() <= 2.0 ** -34).all()), e


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [1, 40, 3000])
def test_stored_groups_of_zeros(device, M, dtype):
    # a weight with padding, as one is stored whose groups of zeros have the smallest scale
    N, K = 520, 300
    w = torch.randn(N, K, generator=torch.Generator().manual_seed(M))
    w[500:], w[:, 256:], w[::3, 32:64] = 0.0, 0.0, 0.0
    q = quantize_weight(w.cuda())
    codes, scales = q.unpack()
    groups = torch.nn.functional.pad(w, (0, -K % 32)).view(N, -1, 32)
    stored = scales.view(torch.uint8).masked_fill((groups == 0).all(2).cuda(), 0)
    p = QuantizedWeight.pack(codes, stored, cols=K)
    assert torch.equal(p.codes, q.codes)
    assert torch.equal(p.scales.view(torch.uint8), q.scales.view(torch.uint8))
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    assert torch.equal(quantized_linear(x, p), quantized_linear(x, q))
