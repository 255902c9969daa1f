"""Limits of the operators with 4-bit weights that are checked on the host (CPU only: no
launch is reached)."""

import pytest
import torch

from kadllm_amd import _lib, layers
from kadllm_amd.ops import QuantizedWeight
from oracle import quantized_ref as ref

U8, BF = torch.uint8, torch.bfloat16


def _zeros(N, K):
    return QuantizedWeight.pack(torch.zeros(N, -(-K // 2), dtype=U8),
                                torch.full((N, -(-K // 32)), 127, dtype=U8), cols=K)


@pytest.mark.parametrize("change, error", [
    (dict(a=torch.zeros(3, 1000, dtype=BF)), ValueError),  # past the weight's codes
    (dict(a=torch.zeros(3, 39, dtype=BF)), ValueError),
    (dict(a=torch.zeros(0, 40, dtype=BF)), ValueError),
    (dict(out=torch.zeros(3, 4, dtype=BF)), ValueError),
    (dict(out=torch.zeros(2, 5, dtype=BF)), ValueError),
    (dict(out=torch.zeros(5, 3, dtype=BF).T), ValueError),
    (dict(out=torch.zeros(1, 5, dtype=BF).expand(3, 5)), ValueError),
    (dict(a=torch.zeros(3, 40)), TypeError),  # four bytes an output
    (dict(a=torch.zeros(3, 40, dtype=torch.float16)), TypeError),
    (dict(out=torch.zeros(3, 5)), TypeError),
    (dict(residual=torch.zeros(3, 5)), TypeError),
    (dict(residual=torch.zeros(3, 4, dtype=BF)), ValueError),
    (dict(residual=torch.zeros(2, 5, dtype=BF)), ValueError),
    (dict(residual=None), ValueError),
    (dict(), RuntimeError),  # well-formed, but not on a ROCm device
])
def test_gemm_refusals(change, error):
    args = dict(a=torch.zeros(3, 40, dtype=BF), out=torch.zeros(3, 5, dtype=BF),
                residual=torch.zeros(3, 5, dtype=BF))
    args.update(change)
    with pytest.raises(error):
        layers.gemm(args.pop("a"), _zeros(5, 40), epilogue=layers.EPI_RESIDUAL, **args)


@pytest.mark.parametrize("N, K", [(1, 1), (3, 31), (5, 32), (4, 700), (20, 1001), (16, 1024)])
def test_groups_of_zeros_may_have_the_smallest_scale(N, K):
    # byte 0 is what a quantiser that clamps the exponent of an amax of 0 stores
    g = torch.Generator().manual_seed(K)
    w = torch.randn(N, K, generator=g)
    w[torch.rand(N, -(-K // 32), generator=g).repeat_interleave(32, 1)[:, :K] < 0.4] = 0.0
    w[N - 1] = 0.0  # a row of padding
    codes, exps = ref.quantize(w)
    zeros = torch.nn.functional.pad(w, (0, -K % 32)).view(N, -1, 32).abs().amax(2) == 0
    codes = codes | (torch.rand(N, K, generator=g) < 0.5) * 8 * (codes == 0)  # zeros of both signs
    parts, scales = ref.parts(codes, exps)
    stored = scales.masked_fill(zeros, 0)
    assert bool((stored == 0).any())
    if K % 2:
        parts[:, -1] |= 0x70  # what is behind the last column is not looked at
    q = QuantizedWeight.pack(parts, stored, cols=K)
    want = QuantizedWeight.pack(parts, scales, cols=K)
    assert torch.equal(q.codes, want.codes)
    assert torch.equal(q.scales.view(U8), want.scales.view(U8))
    assert bool((stored == 0).any()) and torch.equal(q.unpack()[1].view(U8), scales)
    # parts that are not contiguous
    q = QuantizedWeight.pack(parts.T.contiguous().T, stored.T.contiguous().T, cols=K)
    assert torch.equal(q.codes, want.codes)
    assert torch.equal(q.scales.view(U8), want.scales.view(U8))
    # NaN stays NaN
    nan = QuantizedWeight.pack(parts, scales.masked_fill(zeros, 255), cols=K).unpack()[1].view(U8)
    assert bool((nan[zeros] == 255).all())


@pytest.mark.parametrize("code, scale", [(1, 0), (7, 0), (9, 0), (0x10, 0), (0x70, 0), (0, 1),
                                         (0, 26), (0, 253), (8, 254), (1, 26)])
def test_other_scales_are_refused(code, scale):
    codes, scales = torch.zeros(3, 40, dtype=U8), torch.full((3, 3), 127, dtype=U8)
    codes[2, 39], scales[2, 2] = code, scale
    with pytest.raises(ValueError):
        QuantizedWeight.pack(codes, scales)


@pytest.mark.parametrize("N, K", [(8193 * 16, 8191 * 128),  # 2^26 - 1 blocks: 2^24 workgroups
                                  (2 ** 26 + 1, 128), (2 ** 26, 2048)])
def test_weights_past_a_grid_are_refused(N, K):
    P = 1 << 20  # an aligned address, which is not read
    lib = _lib.load()
    assert lib.kad_quantize_weight(P, K, 0, P, P, N, K, None) == -1
    assert lib.kad_dequantize_weight(P, P, P, K, 0, N, K, None) == -1
