"""Limits of the operators with 4-bit weights that are checked on the host (CPU only: no
launch is reached)."""

import pytest
import torch

from kadllm_amd import layers
from kadllm_amd.ops import QuantizedWeight

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
