"""4-bit weights and the products with them in plain torch, in 64 bits.

A weight is a table index (0 to 15) and a whole exponent for every 32 neighbours
of a row, so that nothing here depends on a library's conversion.
"""

import math

import torch

LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
GROUP = 32


def values():
    """The 16 values of a code."""
    return torch.tensor(LEVELS + tuple(-x for x in LEVELS), dtype=torch.float64)


def scale_exponent(amax):
    """The smallest e in [-100, 125] with amax <= 7 * 2^e; 0 for zeros."""
    if amax == 0:
        return 0
    frac, exp = math.frexp(amax)                    # frac in [1/2, 1)
    return min(max(exp - 3 + (frac > 7 / 8), -100), 125)


def quantize(w):
    """(codes [N, K] int64, exponents [N, ceil(K / 32)] int64, 128 for NaN) of w [N, K]."""
    w = w.detach().cpu().double()
    N, K = w.shape
    groups = torch.nn.functional.pad(w, (0, -K % GROUP)).view(N, -1, GROUP)
    amax = groups.abs().amax(2)
    finite = groups.isfinite().all(2)
    exps = torch.tensor([[scale_exponent(a) if ok else 128 for a, ok in zip(*row)]
                         for row in zip(amax.tolist(), finite.tolist())])
    powers = torch.ldexp(torch.ones_like(amax), torch.where(finite, exps, 0))
    y = torch.where(finite[..., None], groups / powers[..., None], 0.0)
    levels = torch.tensor(LEVELS, dtype=torch.float64)
    # the nearest level; of two equally near ones that of even number
    distance = (y.abs()[..., None] - levels).abs()
    near = distance == distance.amin(-1, keepdim=True)
    even = near & (torch.arange(8) % 2 == 0)
    codes = torch.where(even.any(-1), even.long().argmax(-1), near.long().argmax(-1))
    codes = codes + 8 * torch.signbit(y).long()
    return codes.view(N, -1)[:, :K], exps


def dense(codes, exps):
    """The values [N, K] in float64."""
    K = codes.shape[1]
    powers = torch.ldexp(torch.ones(exps.shape, dtype=torch.float64), exps)
    powers = torch.where(exps == 128, torch.nan, powers)
    return values()[codes] * powers.repeat_interleave(GROUP, 1)[:, :K]


def parts(codes, exps):
    """The row-major bytes: codes [N, ceil(K / 2)] and scales [N, ceil(K / 32)], uint8."""
    codes = torch.nn.functional.pad(codes, (0, codes.shape[1] % 2))
    return (codes[:, 0::2] + 16 * codes[:, 1::2]).to(torch.uint8), (exps + 127).to(torch.uint8)


def linear(x, w, residual=None):
    """(x w^T + residual, sum |x| |w| + |residual|) in float64."""
    x, w = x.detach().cpu().double(), w.cpu()
    y, size = x @ w.T, x.abs() @ w.abs().T
    if residual is not None:
        residual = residual.detach().cpu().double()
        y, size = y + residual, size + residual.abs()
    return y, size


def silu(x):
    return x * torch.sigmoid(x)


def gated_ffn(x, gate, up, down, residual=None):
    """The block's output in float64."""
    x = x.detach().cpu().double()
    h = silu(x @ gate.cpu().T) * (x @ up.cpu().T)
    return linear(h, down, residual)[0]
