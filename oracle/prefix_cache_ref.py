"""The 8-bit prefix cache in plain torch on the CPU, in 64 bits.

Codes are e4m3 values and scales powers of two, both as float64 tensors, so
that nothing here depends on a library's conversion.
"""

import math

import torch


def e4m3_values():
    """The 256 values an e4m3 byte stands for (NaN at 0x7f and 0xff)."""
    out = []
    for byte in range(256):
        sign, exp, frac = byte >> 7, byte >> 3 & 15, byte & 7
        x = math.ldexp(8 + frac, exp - 10) if exp else math.ldexp(frac, -9)
        out.append(math.nan if byte & 127 == 127 else -x if sign else x)
    return torch.tensor(out, dtype=torch.float64)


def decode(codes, scales):
    """(code values, scales) as float64 of float8_e4m3fn and float8_e8m0fnu tensors
    (NaN for the scale byte 255)."""
    table = e4m3_values()
    byte = scales.cpu().view(torch.uint8).long()
    powers = torch.ldexp(torch.ones((), dtype=torch.float64), byte - 127)
    return (table[codes.cpu().view(torch.uint8).long()],
            torch.where(byte == 255, torch.nan, powers))


def round_e4m3(x):
    """float64 x, |x| <= 448, to the nearest e4m3 value, ties to even; others NaN."""
    ok = x.isfinite()
    y = torch.where(ok, x, 0.0)
    _, e = torch.frexp(y)
    step = torch.ldexp(torch.ones_like(y), (e - 1).clamp(min=-6) - 3)
    return torch.where(ok, torch.round(y / step) * step, torch.nan)


def block_tables(lengths, free, block, max_length, starts=None, tables=None):
    width = -(-max_length // block)
    out, taken = [], 0
    for b, n in enumerate(lengths):
        held = -(-min(max(starts[b], 0), max_length) // block) if starts is not None else 0
        total = max(-(-min(max(n, 0), max_length) // block), held)
        row = [-1] * width
        for j in range(held):
            if tables is not None and j < len(tables[b]):
                row[j] = tables[b][j]
        for j in range(held, total):
            if taken < len(free):
                row[j] = free[taken]
            taken += 1
        out.append(row)
    return out, taken


def write(codes, scales, x, tables, lengths, starts, block):
    """Write x [B, N, HK, D] float64 into codes [pages, HK, block, D] and scales
    [pages, HK] (float64 tensors, changed in place)."""
    B, N, HK, _ = x.shape
    for b in range(B):
        start = max(starts[b], 0)
        stop = min(start + N, lengths[b], len(tables[b]) * block)
        for j in range(start // block, -(-stop // block) if stop > start else 0):
            page = tables[b][j]
            if not 0 <= page < codes.shape[0]:
                continue
            lo, hi = max(start - j * block, 0), min(stop - j * block, block)
            for h in range(HK):
                new = x[b, j * block + lo - start:j * block + hi - start, h]
                amax = torch.where(new.isfinite(), new.abs(), 0.0).max().item()
                e = -100
                while amax > 448 * 2.0 ** e:
                    e += 1
                s = 2.0 ** e
                before = scales[page, h].item()
                if lo and (before >= s or math.isnan(before)):
                    s = before
                elif lo:
                    codes[page, h, :lo] = round_e4m3(codes[page, h, :lo] * (before / s))
                codes[page, h, lo:hi] = round_e4m3(new / s)
                scales[page, h] = s


def attention(q, k_pool, v_pool, tables, lengths, suffix_k, suffix_v, beam_width, scale,
              gate=None):
    """(out, weight, slack), all [B*W, T, H, D] float64: the attention of
    kadllm.ops.block_prefix_attention, sum_j p_j |v_j| of its normalised
    weights (times the gate), and sum_j |v_j| / l over the cached keys (l the
    sum of exp(s_j - max s)).  k_pool, v_pool: (codes, scales) as decode gives."""
    BW, T, H, D = q.shape
    HK, block = k_pool[0].shape[1:3]
    G = H // HK
    out, weight, slack = (torch.zeros(BW, T, H, D, dtype=torch.float64) for _ in range(3))
    q = q.double().cpu()
    pages = k_pool[0].shape[0]
    for n in range(BW):
        b = n // beam_width
        keys = [(j // block, j % block) for j in range(min(lengths[b], len(tables[b]) * block))]
        keys = [(tables[b][j], r) for j, r in keys if 0 <= tables[b][j] < pages]
        page = torch.tensor([p for p, _ in keys], dtype=torch.long)
        row = torch.tensor([r for _, r in keys], dtype=torch.long)
        for h in range(H):
            kh = h // G
            k, v = (c[page, kh, row] * s[page, kh][:, None] for c, s in (k_pool, v_pool))
            for t in range(T):
                ka, va = k, v
                if suffix_k is not None:
                    see = suffix_k.shape[1] - T + t + 1
                    ka = torch.cat((k, suffix_k[n, :see, kh].double().cpu()))
                    va = torch.cat((v, suffix_v[n, :see, kh].double().cpu()))
                if not len(ka):
                    continue
                s = ka @ q[n, t, h] * scale
                p = torch.exp(s - s.max())
                g = 1.0
                if gate is not None:
                    g = torch.sigmoid(gate[n, t, h * D:(h + 1) * D].double().cpu())
                out[n, t, h] = (p / p.sum()) @ va * g
                weight[n, t, h] = (p / p.sum()) @ va.abs() * g
                slack[n, t, h] = v.abs().sum(0) / p.sum()
    return out, weight, slack
