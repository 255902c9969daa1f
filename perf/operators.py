"""Cases that time the operators of the 8-bit prefix cache and check them.

A serving program that keeps its requests' prefixes in 8 bits makes three
calls, and each is a kind of case here:

  tables     kadllm.ops.prefix_block_tables: the pages of a batch's requests
             from their lengths, for new prompts or for prompts that grow
  write      kadllm.ops.write_prefix_blocks: keys and values into the pages,
             e4m3 values with one power-of-two scale per page and KV head
  attention  kadllm.ops.block_prefix_attention: the beams' queries over the
             pages of their request, then over their own suffix

A case is a dict of plain values.  ``listed`` names the fixed ones, ``draw``
gives more of the same ranges, ``prepare`` makes on the GPU what the program
holds before the call, ``run`` makes one call (``own``) or computes the same
in elementary torch operations, ``work`` counts what the call cannot do
without, and ``exact`` computes the outputs in 64 bits from the definition.

A page holds ``block`` tokens: codes k, v [pages, HK, block, D] (e4m3) and
scales [pages, HK] (e8m0: powers of two).  The scale of a page and head is the
smallest power of two s with amax <= 448 s over the finite values written to it;
a page that is extended keeps the larger of its own scale and the new tokens'.
"""

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def listed():
    return [
        # a full serving batch of 1024-token prompts gets its pages
        {"name": "tables_b32_l1024", "kind": "tables", "requests": 32, "length": 1024, "block": 64,
         "grow": False, "ragged": False},
        # a large pool of long, unequal requests, each one token further
        {"name": "tables_b1000_l32768_grow", "kind": "tables", "requests": 1000, "length": 32768,
         "block": 64, "grow": True, "ragged": True},
        # one attention layer's keys and values of that full batch, as its prefill leaves them
        {"name": "write_b32_l1024", "kind": "write", "dtype": "bf16", "requests": 32,
         "length": 1024, "tokens": 1024, "kv_heads": 2, "dim": 256, "block": 64, "ragged": False},
        # a few long prompts of unequal length, eight KV heads of 128
        {"name": "write_b8_l20000", "kind": "write", "dtype": "fp16", "requests": 8,
         "length": 20000, "tokens": 20000, "kv_heads": 8, "dim": 128, "block": 128,
         "ragged": True},
        # 256 sequences in flight, each with one more token
        {"name": "write_b256_append", "kind": "write", "dtype": "bf16", "requests": 256,
         "length": 1000, "tokens": 1, "kv_heads": 2, "dim": 256, "block": 64, "ragged": True},
        # one layer of the full serving batch: 256 beams a request, third output token, gated
        {"name": "attention_b32_w256_l1024", "kind": "attention", "dtype": "bf16", "requests": 32,
         "beams": 256, "tokens": 1, "suffix": 2, "length": 1024, "heads": 8, "kv_heads": 2,
         "dim": 256, "block": 64, "gate": True, "ragged": False},
        # a small service with an odd beam width, unequal prompts and a replayed suffix
        {"name": "attention_b8_w50_l1000", "kind": "attention", "dtype": "bf16", "requests": 8,
         "beams": 50, "tokens": 3, "suffix": 3, "length": 1000, "heads": 8, "kv_heads": 2,
         "dim": 256, "block": 64, "gate": False, "ragged": True},
        # a single user's short prompt, first decode step of one sequence: latency
        {"name": "attention_b1_w1_l100", "kind": "attention", "dtype": "bf16", "requests": 1,
         "beams": 1, "tokens": 1, "suffix": 1, "length": 100, "heads": 8, "kv_heads": 2,
         "dim": 256, "block": 64, "gate": False, "ragged": False},
        # one token each for 16 long sequences whose every token is in the cache
        {"name": "attention_b16_l32768", "kind": "attention", "dtype": "bf16", "requests": 16,
         "beams": 1, "tokens": 1, "suffix": 0, "length": 32768, "heads": 8, "kv_heads": 2,
         "dim": 256, "block": 64, "gate": False, "ragged": False},
        # an fp16 model with 16 query and 4 KV heads of 128, ten beams on unequal prompts
        {"name": "attention_fp16_b4_w10_l5000", "kind": "attention", "dtype": "fp16",
         "requests": 4, "beams": 10, "tokens": 1, "suffix": 2, "length": 5000, "heads": 16,
         "kv_heads": 4, "dim": 128, "block": 128, "gate": False, "ragged": True},
        # many short beams on one request with heads of 64 (the small hybrid's four to one)
        {"name": "attention_b64_w4_l2000_d64", "kind": "attention", "dtype": "bf16",
         "requests": 64, "beams": 4, "tokens": 2, "suffix": 2, "length": 2000, "heads": 4,
         "kv_heads": 1, "dim": 64, "block": 32, "gate": False, "ragged": True},
        # one long prompt searched with 256 beams: few requests, many rows, many keys
        {"name": "attention_b1_w256_l8192", "kind": "attention", "dtype": "bf16", "requests": 1,
         "beams": 256, "tokens": 1, "suffix": 1, "length": 8192, "heads": 8, "kv_heads": 2,
         "dim": 256, "block": 64, "gate": True, "ragged": False},
    ]


def _log_int(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# (query heads, KV heads, head dim): the repository's two models' and generic ones
HEADS = [(8, 2, 256), (8, 2, 256), (4, 1, 64), (16, 4, 128), (8, 8, 64), (12, 2, 128)]


def draw(rng):
    kind = rng.choice(["tables", "write", "write", "attention", "attention", "attention"])
    block = rng.choice([32, 64, 64, 128])
    if kind == "tables":
        length = _log_int(rng, 16, 32768)
        return {"kind": kind, "requests": _log_int(rng, 1, max(1, min(4096, 2 ** 25 // length))),
                "length": length, "block": block, "grow": rng.random() < 0.5,
                "ragged": rng.random() < 0.7}
    heads, kv_heads, dim = rng.choice(HEADS)
    if kind == "write":
        most = 150_000_000 // (kv_heads * dim)  # tokens in all
        length = _log_int(rng, 1, 20000)
        requests = _log_int(rng, 1, max(1, min(512, most // length)))
        tokens = rng.choice([length, length, 1, rng.randint(1, length)])
        return {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                "requests": requests, "length": length, "tokens": tokens, "kv_heads": kv_heads,
                "dim": dim, "block": block, "ragged": rng.random() < 0.5}
    beams = _log_int(rng, 1, 256)
    tokens = rng.randint(1, 3)
    suffix = rng.choice([0, tokens, tokens, tokens + rng.randint(0, 5)])
    length = _log_int(rng, 1, 32768)
    # the flops of 32 requests of 256 beams over 1024 tokens, the bytes of 16 over 32768
    most = min(8 * 256 * 32 * 256 * 1024 // (heads * dim * beams * tokens),
               2 * 256 * 16 * 32768 // (kv_heads * dim))
    requests = _log_int(rng, 1, max(1, min(64, most // length)))
    length = max(1, min(length, most // requests))
    return {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "fp16"]), "requests": requests,
            "beams": beams, "tokens": tokens, "suffix": suffix, "length": length, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "block": block, "gate": rng.random() < 0.4,
            "ragged": rng.random() < 0.6}


# ----------------------------------------------------------------------------
# inputs

def _lengths(case, gen):
    """Tokens of each request [B] int32: all of them ``length``, or (ragged)
    spread evenly from none to ``length`` in an order of their own."""
    B, L = case["requests"], case["length"]
    if not case["ragged"] or B == 1:
        return torch.full((B,), L, dtype=torch.int32, device=DEVICE)
    even = (torch.arange(B, device=DEVICE, dtype=torch.float64) * L / (B - 1)).round().int()
    return even[torch.randperm(B, generator=gen, device=DEVICE)]


def _values(gen, shape):
    """Keys or values: each channel with a magnitude of its own, fp32."""
    x = torch.randn(shape, generator=gen, device=DEVICE)
    return x.mul_(torch.randn(shape[-1], generator=gen, device=DEVICE).mul(0.5).exp())


def _power(exp):
    """2^exp in fp32, exactly (exp2 and ldexp may be an ulp off on the GPU)."""
    return (exp + 127).to(torch.uint8).view(E8M0).float()


def _pool(gen, pages, kv_heads, block, dim):
    """Codes [pages, HK, block, D] e4m3 and scales [pages, HK] e8m0 of filled pages."""
    x = _values(gen, (pages, kv_heads, block, dim))
    frac, exp = torch.frexp(x.abs().amax((2, 3)) / 448.0)
    exp = torch.where(frac == 0.5, exp - 1, exp)
    codes = (x * _power(-exp)[..., None, None]).to(E4M3)
    return codes, (exp + 127).to(torch.uint8).view(E8M0)


def _tables(gen, lengths, block, width, pages):
    """Page numbers [B, width] int32 in an order of their own, -1 past a request's last page."""
    B = lengths.numel()
    order = torch.randperm(pages, generator=gen, device=DEVICE)[:B * width].view(B, width).int()
    held = (lengths + block - 1) // block
    return torch.where(torch.arange(width, device=DEVICE) < held[:, None], order, -1)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    B, L, block = case["requests"], case["length"], case["block"]
    width = -(-L // block)
    lengths = _lengths(case, gen)
    if case["kind"] == "tables":
        # the pool has a tenth more pages than the requests could fill
        pages = B * width + B * width // 10 + 1
        state = {"case": case, "lengths": lengths, "starts": None, "tables": None}
        if case["grow"]:
            state["starts"] = (lengths - 1).clamp(min=0)
            state["tables"] = _tables(gen, state["starts"], block, width, pages)
        free = torch.randperm(pages, generator=gen, device=DEVICE).int()
        if case["grow"]:
            held = torch.zeros(pages + 1, dtype=torch.bool, device=DEVICE)
            held[state["tables"].flatten().long()] = True  # -1 marks the last, unused place
            free = free[~held[free.long()]]
        state["free"] = free
        return state
    if case["kind"] == "write":
        HK, D, N = case["kv_heads"], case["dim"], case["tokens"]
        pages = B * width
        starts = (lengths - N).clamp(min=0) if N < L else None
        tables = _tables(gen, lengths, block, width, pages)
        # one page more than the requests hold: what another program's request would fill
        k, k_scale = _pool(gen, pages + 1, HK, block, D)
        v, v_scale = _pool(gen, pages + 1, HK, block, D)
        # heads first in memory, as a prefill leaves them; a step's rows as a projection does
        shape = (B, HK, N, D) if N > 1 else (B, N, HK, D)
        new = [_values(gen, shape).to(DTYPES[case["dtype"]]) for _ in range(2)]
        if N > 1:
            new = [x.transpose(1, 2) for x in new]
        return {"case": case, "pool": (k, v, k_scale, v_scale), "new": new, "tables": tables,
                "lengths": lengths, "starts": starts}
    W, T, Tk, H = case["beams"], case["tokens"], case["suffix"], case["heads"]
    HK, D, dt = case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    pages = B * width + 1
    k, k_scale = _pool(gen, pages, HK, block, D)
    v, v_scale = _pool(gen, pages, HK, block, D)
    q = torch.randn(B * W, T, H, D, generator=gen, device=DEVICE).to(dt)
    suffix = [_values(gen, (B * W, Tk, HK, D)).to(dt) if Tk else None for _ in range(2)]
    gate = None
    if case["gate"]:
        gate = torch.randn(B * W, T, H * D, generator=gen, device=DEVICE).to(dt)
    return {"case": case, "pool": (k, v, k_scale, v_scale), "q": q, "suffix": suffix,
            "gate": gate, "lengths": lengths, "tables": _tables(gen, lengths, block, width, pages)}


# ----------------------------------------------------------------------------
# the plain forms

def _plain_tables(s):
    case, block = s["case"], s["case"]["block"]
    B, L = case["requests"], case["length"]
    width = -(-L // block)
    lengths = s["lengths"].clamp(0, L)
    held = torch.zeros_like(lengths) if s["starts"] is None else (s["starts"] + block - 1) // block
    total = torch.maximum((lengths + block - 1) // block, held)
    need = total - held
    first = need.cumsum(0) - need
    col = torch.arange(width, device=DEVICE)
    at = first[:, None] + col - held[:, None]
    fresh = s["free"][at.clamp(0, s["free"].numel() - 1)]
    fresh = torch.where((col < total[:, None]) & (at < s["free"].numel()), fresh, -1)
    if s["tables"] is not None:
        fresh = torch.where(col < held[:, None], s["tables"], fresh)
    return fresh, need.sum(dtype=torch.int32).view(1)


def _plain_write(s):
    case = s["case"]
    B, L, N, block = case["requests"], case["length"], case["tokens"], case["block"]
    lengths = s["lengths"]
    starts = torch.zeros_like(lengths) if s["starts"] is None else s["starts"]
    width = s["tables"].shape[1]
    touched = min(width, (N + block - 2) // block + 1)  # pages that N tokens can reach into
    page = starts[:, None] // block + torch.arange(touched, device=DEVICE)  # [B, U]
    at = page[..., None] * block + torch.arange(block, device=DEVICE)       # [B, U, block]
    fresh = (at >= starts[:, None, None]) & (at < lengths[:, None, None])
    old = at < starts[:, None, None]
    ids = s["tables"].gather(1, page.clamp(max=width - 1).long()).long()
    spare = s["pool"][0].shape[0] - 1
    ids = torch.where(fresh.any(2) & (ids >= 0), ids, spare)     # the spare page takes the rest
    fresh = (fresh & (ids < spare)[..., None])[:, :, None, :, None]          # [B, U, 1, block, 1]
    keep = (old.any(2) & (ids < spare))[..., None]
    row = (at - starts[:, None, None]).clamp(0, N - 1)
    b = torch.arange(B, device=DEVICE)[:, None, None]
    for codes, scale, x in zip(s["pool"][:2], s["pool"][2:], s["new"]):
        x = x[b, row].transpose(2, 3).float()                    # [B, U, HK, block, D]
        amax = torch.where(fresh & x.isfinite(), x.abs(), 0.0).amax((3, 4))
        frac, exp = torch.frexp(amax / 448.0)
        exp = torch.where(frac == 0.5, exp - 1, exp).clamp(min=-100)
        before = scale.view(torch.uint8)[ids].int() - 127        # [B, U, HK]
        exp = torch.where(amax == 0, -100, exp)
        exp = torch.where(keep, torch.maximum(exp, before), exp)
        exp = torch.where((ids < spare)[..., None], exp, before)
        held = codes.view(torch.uint8)[ids].view(E4M3).float()
        moved = _power(torch.where(keep, before - exp, 0).clamp(min=-127))[..., None, None]
        held = torch.where(old[:, :, None, :, None], held * moved, held)
        x = x * _power(-exp)[..., None, None]
        codes.view(torch.uint8)[ids] = torch.where(fresh, x, held).to(E4M3).view(torch.uint8)
        scale.view(torch.uint8)[ids] = (exp + 127).to(torch.uint8)
    return s["pool"]


def _plain_attention(s):
    case = s["case"]
    B, W, T, Tk, H = (case[n] for n in ("requests", "beams", "tokens", "suffix", "heads"))
    HK, D = case["kv_heads"], case["dim"]
    G = H // HK
    k, v, k_scale, v_scale = s["pool"]
    ids = s["tables"].clamp(min=0).long()
    shape = (B, HK, ids.shape[1] * case["block"], D)
    seen = torch.arange(shape[2], device=DEVICE) < s["lengths"][:, None]          # [B, keys]
    k, v = ((c.view(torch.uint8)[ids].view(E4M3).float() * e.float()[ids][..., None, None])
            .transpose(1, 2).reshape(shape) for c, e in ((k, k_scale), (v, v_scale)))
    v = torch.where(seen[:, None, :, None], v, 0.0)
    q = s["q"].float().mul(D ** -0.5).view(B, W, T, HK, G, D).permute(0, 3, 1, 4, 2, 5)
    scores = q.reshape(B, HK, W * G * T, D) @ k.transpose(2, 3)
    scores = torch.where(seen[:, None, None], scores, -torch.inf).view(B, HK, W, G * T, -1)
    top = scores.amax(-1, keepdim=True)
    if Tk:
        ks, vs = (x.float().view(B, W, Tk, HK, D).permute(0, 3, 1, 2, 4) for x in s["suffix"])
        own_scores = q.reshape(B, HK, W, G * T, D) @ ks.transpose(3, 4)           # [.., G*T, Tk]
        t = torch.arange(T, device=DEVICE).repeat(G)
        causal = torch.arange(Tk, device=DEVICE) <= t[:, None] + (Tk - T)
        own_scores = torch.where(causal, own_scores, -torch.inf)
        top = torch.maximum(top, own_scores.amax(-1, keepdim=True))
    top = torch.where(top == -torch.inf, 0.0, top)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    out = (p.view(B, HK, W * G * T, -1) @ v).view(B, HK, W, G * T, D)
    if Tk:
        p = torch.exp(own_scores - top)
        total = total + p.sum(-1, keepdim=True)
        out = out + p @ vs
    out = torch.where(total > 0, out / total, 0.0)
    out = out.view(B, HK, W, G, T, D).permute(0, 2, 4, 1, 3, 5).reshape(B * W, T, H, D)
    if s["gate"] is not None:
        out = out * (1 / (1 + torch.exp(-s["gate"].float()))).view(out.shape)
    return out.to(s["q"].dtype)


def run(state):
    case = state["case"]
    if not own:
        return {"tables": _plain_tables, "write": _plain_write,
                "attention": _plain_attention}[case["kind"]](state)
    from kadllm import ops

    if case["kind"] == "tables":
        return ops.prefix_block_tables(state["lengths"], state["free"],
                                       block_size=case["block"], max_length=case["length"],
                                       starts=state["starts"], tables=state["tables"])
    blocks = ops.PrefixBlocks(*state["pool"])
    if case["kind"] == "write":
        return tuple(ops.write_prefix_blocks(blocks, *state["new"], state["tables"],
                                             state["lengths"], starts=state["starts"]))
    return ops.block_prefix_attention(state["q"], blocks, state["tables"], state["lengths"],
                                      *state["suffix"], beam_width=case["beams"],
                                      gate=state["gate"])


def work(case):
    """Bytes read and written once and flops of one call (ragged lengths: their mean)."""
    B, L, block = case["requests"], case["length"], case["block"]
    ragged = case["ragged"] and B > 1
    tokens = B * L // 2 if ragged else B * L
    width = -(-L // block)
    if case["kind"] == "tables":
        # lengths (and starts), the table out and its used part in (free pages or held ones)
        used = tokens / block
        return {"bytes": 4 * (B * (2 if case["grow"] else 1) + B * width + used), "flops": 0}
    HK, D = case["kv_heads"], case["dim"]
    if case["kind"] == "write":
        new = tokens if case["tokens"] >= L else B * min(L, case["tokens"])
        item = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": 2 * new * HK * D * (item + 1) + 8 * B, "flops": 0}
    H, Tk = case["heads"], case["suffix"]
    rows = B * case["beams"] * case["tokens"]
    bytes_ = 2 * tokens * HK * D + 2 * rows * H * D * (3 if case["gate"] else 2)
    bytes_ += 4 * B * case["beams"] * Tk * HK * D
    keys = tokens * case["beams"] * case["tokens"] + rows * max(0, Tk - (case["tokens"] - 1) / 2)
    return {"bytes": bytes_, "flops": 4 * keys * H * D}


# ----------------------------------------------------------------------------
# the same outputs in 64 bits

def _round_e4m3(y):
    """y (float64, at most 448) to the nearest e4m3 value, ties to the even one."""
    _, e = torch.frexp(y)                       # |y| in [2^(e-1), 2^e)
    step = (((e - 1).clamp(min=-6) - 3 + 1023).long() << 52).view(torch.float64)
    return torch.round(y / step) * step


def _exact_write(s):
    block = s["case"]["block"]
    lengths = s["lengths"].tolist()
    starts = [0] * len(lengths) if s["starts"] is None else s["starts"].tolist()
    out = []
    for codes, scale, x in zip(s["pool"][:2], s["pool"][2:], s["new"]):
        codes, scale = codes.double(), scale.double()
        for b, (lo, hi) in enumerate(zip(starts, lengths)):
            if hi <= lo:
                continue
            first, last = lo // block, -(-hi // block)
            ids = s["tables"][b, first:last].long()
            held = codes[ids].transpose(1, 2).flatten(0, 1)
            rows = (codes[ids] * scale[ids][..., None, None]).transpose(1, 2).flatten(0, 1)
            rows[lo - first * block:hi - first * block] = x[b, :hi - lo].double()
            new = torch.zeros(rows.shape[0], dtype=torch.bool, device=DEVICE)
            new[lo - first * block:hi - first * block] = True
            amax = torch.where(new[:, None, None], rows.abs(), 0.0)
            amax = amax.view(-1, block, *rows.shape[1:]).amax((1, 3))
            frac, e = torch.frexp(amax / 448)            # amax / 448 = frac 2^e, frac in [1/2, 1)
            e = torch.where(amax == 0, -100, torch.where(frac == 0.5, e - 1, e).clamp(min=-100))
            s_new = ((e + 1023).long() << 52).view(torch.float64)
            if lo % block:
                s_new[0] = torch.maximum(s_new[0], scale[ids[0]])
            rows = rows.view(-1, block, *rows.shape[1:]).transpose(1, 2)
            rows = _round_e4m3(rows / s_new[..., None, None]).transpose(1, 2).flatten(0, 1)
            rows[hi - first * block:] = held[hi - first * block:]   # past the request's end
            codes[ids] = rows.view(-1, block, *rows.shape[1:]).transpose(1, 2)
            scale[ids] = s_new
        out.append((codes, scale))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def _exact_attention(s):
    case = s["case"]
    B, W, T, Tk, H = (case[n] for n in ("requests", "beams", "tokens", "suffix", "heads"))
    HK, D = case["kv_heads"], case["dim"]
    G = H // HK
    out = torch.zeros(B * W, T, H, D, dtype=torch.float64, device=DEVICE)
    pool = [(s["pool"][i], s["pool"][i + 2]) for i in range(2)]
    for b, n in enumerate(s["lengths"].tolist()):
        ids = s["tables"][b, :-(-n // case["block"])].long()
        beams = slice(b * W, (b + 1) * W)
        for h in range(HK):
            heads = slice(h * G, (h + 1) * G)
            k, v = ((c.view(torch.uint8)[ids, h].view(E4M3).double()
                     * e.double()[ids, h][:, None, None]).reshape(-1, D)[:n] for c, e in pool)
            q = s["q"][beams, :, heads].double().reshape(-1, D)
            logits = [(q @ k.T) / math.sqrt(D)]
            if Tk:
                ks, vs = (x[beams, :, h].double() for x in s["suffix"])           # [W, Tk, D]
                own_logits = q.view(W, T * G, D) @ ks.mT / math.sqrt(D)
                step = torch.arange(T, device=DEVICE).repeat_interleave(G)[:, None]
                future = torch.arange(Tk, device=DEVICE) > step + Tk - T
                logits.append(own_logits.masked_fill(future, -torch.inf).view(W * T * G, Tk))
            logits = torch.cat(logits, 1)
            if not logits.shape[1]:
                continue
            weights = torch.softmax(logits, 1)
            y = weights[:, :n] @ v
            if Tk:
                y = y + (weights[:, n:].view(W, T * G, Tk) @ vs).view(-1, D)
            out[beams, :, heads] = y.view(W, T, G, D)
    if s["gate"] is not None:
        out = out * torch.sigmoid(s["gate"].double()).view(out.shape)
    return out


def exact(case, seed):
    if case["kind"] == "tables":
        return None                              # whole numbers
    state = prepare(case, seed)
    return _exact_write(state) if case["kind"] == "write" else _exact_attention(state)
