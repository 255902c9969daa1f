"""Cases that time the products with 4-bit weights and check them.

A program that serves a model from 4-bit weights makes these calls:

  roundtrip  kadllm.ops.quantize_weight and dequantize_weight: a weight to 4
             bits as it is loaded, and the values that the codes stand for
  linear     kadllm.ops.quantized_linear: y = x W^T (+ residual)
  ffn        kadllm.ops.quantized_gated_ffn: y = (silu(x G^T) * (x U^T)) D^T
             (+ residual)

A case is a dict of plain values.  ``listed`` names the fixed ones, ``draw``
gives more of the same ranges, ``prepare`` makes on the GPU what the program
holds before the call, ``run`` makes one call (``own``) or computes the same
in elementary torch operations, ``work`` counts what the call cannot do
without, and ``exact`` computes the outputs in 64 bits from the definition.

A 4-bit weight [N, K] is e2m1 codes (0, 1/2, 1, 3/2, 2, 3, 4, 6 and their
negatives), two to a byte along K, and one e8m0 scale (a power of two) for
every 32 neighbours of a row.  Quantising takes the smallest scale 2^e, e from
-100 to 125, with amax <= 7 * 2^e, and rounds w / 2^e to the nearest code, ties
to the even one, at most 6.
"""

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
GROUP = 32


def listed():
    return [
        # one layer's gate projection of the 0.8B shape, as a checkpoint's tensor arrives
        {"name": "roundtrip_3584x1024", "kind": "roundtrip", "dtype": "bf16", "N": 3584, "K": 1024},
        # the vocabulary head of that model, the largest tensor of a load
        {"name": "roundtrip_248320x1024", "kind": "roundtrip", "dtype": "bf16", "N": 248320,
         "K": 1024},
        # one token's down projection into the residual stream: the smallest call, latency
        {"name": "linear_m1_1024x3584", "kind": "linear", "dtype": "bf16", "M": 1, "N": 1024,
         "K": 3584, "residual": True, "strided": False},
        # one token's logits over the full vocabulary: the longest read of a single decode step
        {"name": "linear_m1_248320x1024", "kind": "linear", "dtype": "bf16", "M": 1, "N": 248320,
         "K": 1024, "residual": False, "strided": False},
        # ten beams of one request through a GDN layer's input projection
        {"name": "linear_m10_8192x1024", "kind": "linear", "dtype": "bf16", "M": 10, "N": 8192,
         "K": 1024, "residual": False, "strided": False},
        # fifty beams' logits
        {"name": "linear_m50_248320x1024", "kind": "linear", "dtype": "bf16", "M": 50,
         "N": 248320, "K": 1024, "residual": False, "strided": False},
        # an fp16 model of odd sizes, rows inside a wider buffer
        {"name": "linear_fp16_m37_5001x2007", "kind": "linear", "dtype": "fp16", "M": 37,
         "N": 5001, "K": 2007, "residual": True, "strided": True},
        # an fp32 model's output projection for a short prompt
        {"name": "linear_fp32_m300_1024x2048", "kind": "linear", "dtype": "fp32", "M": 300,
         "N": 1024, "K": 2048, "residual": True, "strided": False},
        # one token through a layer's feed-forward block: latency
        {"name": "ffn_m1_1024x3584", "kind": "ffn", "dtype": "bf16", "M": 1, "H": 1024, "F": 3584,
         "residual": True, "strided": False},
        # the beams of one request of the headline search, 256 rows
        {"name": "ffn_m256_1024x3584", "kind": "ffn", "dtype": "bf16", "M": 256, "H": 1024,
         "F": 3584, "residual": True, "strided": False},
        # a wider fp16 block of odd width for a handful of rows
        {"name": "ffn_fp16_m19_2048x5503", "kind": "ffn", "dtype": "fp16", "M": 19, "H": 2048,
         "F": 5503, "residual": False, "strided": False},
        # the prefill of 32 prompts of 1024 tokens: bound by the matrix units
        {"name": "ffn_m32768_1024x3584", "kind": "ffn", "dtype": "bf16", "M": 32768, "H": 1024,
         "F": 3584, "residual": True, "strided": False},
    ]


def _log_int(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["roundtrip", "linear", "linear", "linear", "ffn", "ffn"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    step = rng.choice([1, 1, 16, 128])  # odd sizes and round ones

    def size(lo, hi):
        return -(-_log_int(rng, lo, hi) // step) * step

    if kind == "roundtrip":
        K = size(32, 16384)
        return {"kind": kind, "dtype": dtype, "N": size(1, min(248320, 200_000_000 // K)), "K": K}
    residual, strided = rng.random() < 0.5, rng.random() < 0.3
    if kind == "linear":
        K = size(16, 16384)
        N = size(16, min(248320, 200_000_000 // K))
        M = _log_int(rng, 1, max(1, min(8192, 200_000_000_000 // (2 * N * K), 10 ** 9 // N)))
        return {"kind": kind, "dtype": dtype, "M": M, "N": N, "K": K, "residual": residual,
                "strided": strided}
    H, F = size(64, 8192), size(64, 16384)
    M = _log_int(rng, 1, max(1, min(32768, 300_000_000_000 // (6 * H * F))))
    return {"kind": kind, "dtype": dtype, "M": M, "H": H, "F": F, "residual": residual,
            "strided": strided}


# ----------------------------------------------------------------------------
# inputs

def _weights(gen, N, K):
    """A weight's values, fp32: normal, columns of unlike magnitude."""
    w = torch.randn(N, K, generator=gen, device=DEVICE)
    return w.mul_(torch.randn(K, generator=gen, device=DEVICE).mul_(0.3).exp_().mul_(K ** -0.5))


def _power(exp):
    """2^exp in fp32 for whole exp from -126 to 127."""
    return ((exp + 127) << 23).view(torch.float32)


def _quantize(w):
    """(codes [N, ceil(K / 2)] uint8, scales [N, ceil(K / 32)] uint8) of w."""
    N, K = w.shape
    w = torch.nn.functional.pad(w.float(), (0, -K % GROUP)).view(N, -1, GROUP)
    frac, exp = torch.frexp(w.abs().amax(2))             # amax = frac 2^exp, frac in [1/2, 1)
    exp = (exp - 3 + (frac > 0.875).int()).clamp(-100, 125)
    y = (w * _power(-exp)[..., None]).view(N, -1)
    a = y.abs()
    # the midpoints between neighbours; a tie goes to the code of even number
    code = (a > 0.25).byte() + (a >= 0.75).byte() + (a > 1.25).byte() + (a >= 1.75).byte()
    code += (a > 2.5).byte() + (a >= 3.5).byte() + (a > 5.0).byte()
    code |= torch.signbit(y).byte() << 3
    codes = code[:, 0::2] | code[:, 1::2] << 4
    return codes[:, :-(-K // 2)].contiguous(), (exp + 127).to(torch.uint8)


class _Weight:
    """A quantised weight as its parts, and (own) as the framework holds it."""

    def __init__(self, gen, N, K):
        self.codes, self.scales = _quantize(_weights(gen, N, K))
        self.N, self.K = N, K
        self.packed = None
        if own:
            from kadllm.ops import QuantizedWeight

            self.packed = QuantizedWeight.pack(self.codes, self.scales, cols=K)


def _activations(gen, M, K, strided):
    """Rows as a norm leaves them: a few channels far larger than the rest, fp32."""
    x = torch.randn(M, K + (24 if strided else 0), generator=gen, device=DEVICE)
    big = torch.rand(x.shape[1], generator=gen, device=DEVICE) < 0.01
    return torch.where(big, 20.0, 1.0) * x


def _rows(x, K, dtype):
    """x in its type; the K columns behind the first eight where it is wider."""
    x = x.to(DTYPES[dtype])
    return x if x.shape[1] == K else x[:, 8:8 + K]


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    dtype = case["dtype"]
    if case["kind"] == "roundtrip":
        return {"case": case, "w": _weights(gen, case["N"], case["K"]).to(DTYPES[dtype])}
    M = case["M"]
    if case["kind"] == "linear":
        N, K = case["N"], case["K"]
        shapes = {"weight": (N, K)}
    else:
        N = K = case["H"]
        F = case["F"]
        shapes = {"gate": (F, K), "up": (F, K), "down": (K, F)}
    state = {"case": case, "x": _rows(_activations(gen, M, K, case["strided"]), K, dtype)}
    for name, shape in shapes.items():
        state[name] = _Weight(gen, *shape)
    state["residual"] = None
    if case["residual"]:
        state["residual"] = torch.randn(M, N, generator=gen, device=DEVICE).to(DTYPES[dtype])
    return state


# ----------------------------------------------------------------------------
# the plain forms

def _values(codes, scales, K):
    """The values that codes and scales stand for [N, K], fp32."""
    code = torch.stack((codes & 15, codes >> 4), 2).view(codes.shape[0], -1)[:, :K]
    m = (code & 7).int()
    # e2m1: exponent m >> 1 (0: subnormal), one fraction bit
    a = torch.where(m < 2, m * 0.5, (2 + (m & 1)) * _power(((m >> 1) - 2).clamp(min=-1)))
    a = torch.where(code > 7, -a, a)
    scale = _power(scales.int() - 127)
    return a * scale.repeat_interleave(GROUP, 1)[:, :K]


def _plain_roundtrip(s):
    w = s["w"]
    return _values(*_quantize(w), w.shape[1]).to(w.dtype)


def _dense(w):
    return _values(w.codes, w.scales, w.K)


def _plain_linear(s):
    y = s["x"].float() @ _dense(s["weight"]).T
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["x"].dtype)


def _plain_ffn(s):
    x = s["x"].float()
    g = x @ _dense(s["gate"]).T
    h = g / (1 + torch.exp(-g)) * (x @ _dense(s["up"]).T)
    y = h @ _dense(s["down"]).T
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["x"].dtype)


def run(state):
    kind = state["case"]["kind"]
    if not own:
        return {"roundtrip": _plain_roundtrip, "linear": _plain_linear,
                "ffn": _plain_ffn}[kind](state)
    from kadllm import ops

    if kind == "roundtrip":
        return ops.dequantize_weight(ops.quantize_weight(state["w"]), state["w"].dtype)
    if kind == "linear":
        return ops.quantized_linear(state["x"], state["weight"].packed,
                                    residual=state["residual"])
    return ops.quantized_gated_ffn(state["x"], *(state[n].packed for n in ("gate", "up", "down")),
                                   residual=state["residual"])


def work(case):
    """Bytes read and written once and flops of one call."""
    item = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "roundtrip":
        return {"bytes": 2 * item * case["N"] * case["K"], "flops": 0}
    M = case["M"]
    if case["kind"] == "linear":
        N, K, weights = case["N"], case["K"], case["N"] * case["K"]
    else:
        N = K = case["H"]
        weights = 3 * case["H"] * case["F"]
    rows = M * K + M * N * (2 if case["residual"] else 1)
    return {"bytes": rows * item + weights * 17 / 32, "flops": 2 * M * weights}


# ----------------------------------------------------------------------------
# the same outputs in 64 bits

_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _two_to(e):
    """2^e in float64 for whole e."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_roundtrip(w):
    N, K = w.shape
    levels = torch.tensor(_E2M1, dtype=torch.float64, device=DEVICE)
    out = torch.empty(N, K, dtype=torch.float64, device=DEVICE)
    rows = max(1, 2 ** 24 // K)
    for r in range(0, N, rows):
        part = torch.zeros(min(rows, N - r), -(-K // GROUP) * GROUP, dtype=torch.float64,
                           device=DEVICE)
        part[:, :K] = w[r:r + rows]
        part = part.view(-1, GROUP)
        amax = part.abs().amax(1)
        e = torch.ceil(torch.log2(amax / 7)).clamp(-100, 125)
        # (a logarithm next to a whole number may fall on its other side)
        e = torch.where(amax > 7 * _two_to(e), e + 1, e)
        e = torch.where(amax <= 7 * _two_to(e - 1), e - 1, e).clamp(-100, 125)
        scale = _two_to(e)[:, None]
        a = part.abs() / scale
        up = torch.bucketize(a, levels).clamp(max=7)                 # the first level >= a
        low = (up - 1).clamp(min=0)
        to_up, to_low = levels[up] - a, a - levels[low]
        index = torch.where((to_up < to_low) | ((to_up == to_low) & (up % 2 == 0)), up, low)
        q = levels[index] * scale
        out[r:r + rows] = torch.copysign(q, part).view(-1, -(-K // GROUP) * GROUP)[:, :K]
    return out


def _exact_dense(w):
    table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), dtype=torch.float64, device=DEVICE)
    out = torch.empty(w.N, w.codes.shape[1], 2, dtype=torch.float64, device=DEVICE)
    out[..., 0] = table[(w.codes % 16).long()]
    out[..., 1] = table[(w.codes // 16).long()]
    out = out.view(w.N, -1)[:, :w.K]
    scale = _two_to(w.scales.int() - 127)
    group = torch.arange(w.K, device=DEVICE) // GROUP
    return out * scale[:, group]


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "roundtrip":
        return _exact_roundtrip(state["w"])
    x = state["x"].double()
    if case["kind"] == "linear":
        y = torch.matmul(x, _exact_dense(state["weight"]).t())
    else:
        g, u = (torch.matmul(x, _exact_dense(state[n]).t()) for n in ("gate", "up"))
        y = torch.matmul(g * torch.sigmoid(g) * u, _exact_dense(state["down"]).t())
    return y if state["residual"] is None else y + state["residual"].double()
