"""The 8-bit prefix cache's operators at the ends of what they accept: scores
that climb far above a row's first ones, values and queries of any magnitude.

The bounds are those of test_gpu_prefix_cache (derived there).
"""

import pytest
import torch

import test_gpu_prefix_cache as base
from kadllm_amd.ops import block_prefix_attention, write_prefix_blocks
from oracle import prefix_cache_ref as ref

pytestmark = pytest.mark.gpu


def _climbing(device, lengths, W, T, Tk, H, HK, D, block, dtype, key_bytes, seed, suffix=None):
    """A problem whose scores are near 11.5 * 2^(byte - 127) * f in log2 units: f is
    the row's own, 0.4 to 1, and byte the scale byte of the key's page (key_bytes,
    for every other request in reverse) or, for suffix key j, 127 + suffix(j)."""
    q, blocks, tables, lens, sk, sv, gate = base._problem(device, lengths, W, T, Tk, H, HK, D,
                                                          block, dtype, seed=seed)
    gen = torch.Generator().manual_seed(seed + 1)
    row = 0.4 + 0.6 * torch.rand(*q.shape[:3], 1, generator=gen)
    # q . k D^-0.5 = 8 f with keys near 1
    q = (row * 8 / D ** 0.5 * (1 + 0.05 * torch.randn(q.shape, generator=gen))).to(dtype)
    near_one = lambda shape: 1 + 0.125 * torch.randint(-1, 2, shape, generator=gen)  # noqa: E731
    blocks.k.copy_(near_one(blocks.k.shape).to(torch.float8_e4m3fn))
    scales = blocks.k_scale.view(torch.uint8)
    for b, pages in enumerate(tables.tolist()):
        for j, page in enumerate(pages):
            if page >= 0:
                scales[page] = key_bytes[j if b % 2 == 0 else len(key_bytes) - 1 - j]
    if suffix is not None:
        rise = torch.tensor([2.0 ** suffix(j) for j in range(Tk)]).view(1, Tk, 1, 1)
        sk = (near_one(sk.shape) * rise).to(dtype).to(device)
    return q.to(device), blocks, tables, lens, sk, sv, gate


def _attend_and_check(q, blocks, tables, lens, sk, sv, gate, W, times=1):
    """The attention of ``times`` copies against the oracle."""
    if times == 1:
        out = block_prefix_attention(q, blocks, tables, lens, sk, sv, beam_width=W, gate=gate)
    else:
        out = base._run_copies(times, W, q, blocks, tables, lens, sk, sv, gate)
    base._check_attention(out, q, blocks, tables.tolist(), lens.tolist(), sk, sv, W, gate)


# (lengths, copies, W, H, block): few rows, few rows in ranges, 128 rows that share
# tiles, and those in ranges
FORMS = [([160, 130], 1, 3, 2, 32), ([1500], 1, 1, 2, 64), ([160, 130], 72, 25, 5, 32),
         ([2000, 1921], 40, 97, 1, 64)]


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("lengths, times, W, H, block", FORMS)
@pytest.mark.parametrize("what", ["climb", "sum", "both"])
def test_values_near_the_largest(device, D, lengths, times, W, H, block, what):
    """Values of 2^100 and more under scores that climb by up to 35 (weights relative
    to the first score of up to 2^35), values whose plain sum passes fp32's
    largest, and both: the outputs, averages of the values, are finite."""
    pages = -(-max(lengths) // block)
    byte = [127 + 2 * (what != "sum" and j % 5 == 3) for j in range(pages)]
    q, blocks, tables, lens, sk, sv, gate = _climbing(device, lengths, W, 1, 1, H, 1, D, block,
                                                      torch.bfloat16, byte, seed=31,
                                                      suffix=lambda j: 0)
    blocks.v.view(torch.uint8).bitwise_and_(0x7f)
    blocks.v_scale.view(torch.uint8).fill_(220 if what == "climb" else 245)
    _attend_and_check(q, blocks, tables, lens, sk, sv, gate, W, times)


@pytest.mark.parametrize("lengths, times, W, H, block", [FORMS[0], FORMS[2]])
@pytest.mark.parametrize("T, Tk, climb", [(1, 40, True), (2, 33, False), (1, 4, True)])
def test_suffix_values_near_the_largest(device, lengths, times, W, H, block, T, Tk, climb):
    byte = [127] * -(-max(lengths) // block)
    q, blocks, tables, lens, sk, sv, gate = _climbing(
        device, lengths, W, T, Tk, H, 1, 64, block, torch.bfloat16, byte, seed=32,
        suffix=lambda j: 2 * (climb and j % 4 == 3))
    sv = sv.abs() * 2.0 ** 125
    _attend_and_check(q, blocks, tables, lens, sk, sv, gate, W, times)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("lengths, times, W, H, block", FORMS)
@pytest.mark.parametrize("exponent", [-95, -108, -119, -126])
def test_queries_of_any_magnitude(device, D, lengths, times, W, H, block, exponent):
    """Queries down to bf16's smallest numbers, under keys as much larger."""
    q, blocks, tables, lens, sk, sv, gate = base._problem(device, lengths, W, 1, 0, H, 1, D, block,
                                                          torch.bfloat16, seed=33)
    q = (q.double() * 2.0 ** exponent).bfloat16()
    blocks.k_scale.view(torch.uint8).sub_(exponent % 256)
    _attend_and_check(q, blocks, tables, lens, sk, sv, gate, W, times)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("byte", [252, 253, 254, 255])
def test_pages_of_the_largest_scales_are_extended(device, dtype, byte):
    """Pages whose scale is 2^125 to 2^127, and pages that are not numbers (255): the
    earlier tokens stay what they are, new ones are codes of that scale."""
    blocks = base._pool(device, 3, 2, 32, 64, 36)
    blocks.k_scale.view(torch.uint8)[:2] = byte
    blocks.v_scale.view(torch.uint8)[1:] = byte
    before = base._clone(blocks)
    gen = torch.Generator().manual_seed(36)
    k, v = (torch.randn(3, 9, 2, 64, generator=gen).mul(2.0 ** 125).to(dtype) for _ in range(2))
    tables, starts, lengths = [[0], [1], [2]], [20, 1, 31], [29, 10, 32]
    write_prefix_blocks(blocks, k.to(device), v.to(device), base._ints(tables, device),
                        base._ints(lengths, device), starts=base._ints(starts, device))
    for x, now, was in ((k, (blocks.k, blocks.k_scale), (before.k, before.k_scale)),
                        (v, (blocks.v, blocks.v_scale), (before.v, before.v_scale))):
        codes, scales = ref.decode(*was)
        ref.write(codes, scales, x.double(), tables, lengths, starts, 32)
        got_codes, got_scales = ref.decode(*now)
        assert torch.equal(got_scales.isnan(), scales.isnan())
        assert torch.equal(got_scales.nan_to_num(0), scales.nan_to_num(0))
        # a token's value: of a page that is not a number, none
        got, want = (c * s[..., None, None] for c, s in ((got_codes, got_scales), (codes, scales)))
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.nan_to_num(0), want.nan_to_num(0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("lengths, times, W, H, block", FORMS)
def test_scores_that_climb_past_the_first_walk(device, dtype, D, lengths, times, W, H, block):
    """Scores up to 174 above the first ones: past 2^60 in some rows and not in others, so
    that some take their weights from a second walk.  Every output is held to its bound."""
    pages = -(-max(lengths) // block)
    _attend_and_check(*_climbing(device, lengths, W, 1, 1, H, 1, D, block, dtype,
                                 [127 + j % 5 for j in range(pages)], seed=34), W, times)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("lengths, times, W, H, block", [FORMS[0], FORMS[2]])
@pytest.mark.parametrize("T, Tk", [(1, 33), (3, 50)])
def test_suffix_scores_that_climb_past_the_first_walk(device, dtype, D, lengths, times, W, H, block,
                                                      T, Tk):
    """Suffix scores that lie up to 12 above the first ones from key 16 on and up to 81
    from key 32 on (a first walk holds fp16 suffix weights up to 2^14, bf16 ones up to
    2^60)."""
    byte = [127] * -(-max(lengths) // block)
    _attend_and_check(*_climbing(device, lengths, W, T, Tk, H, 1, D, block, dtype, byte, seed=35,
                                 suffix=lambda j: j // 16 + (j >= 32)), W, times)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lengths, times, W, T, Tk, H, D", [
    ([100], 1, 1, 1, 1, 2, 256), ([1, 0, 33, 700], 1, 5, 2, 2, 4, 64),
    ([100, 0], 40, 97, 1, 2, 1, 128), ([65, 1], 40, 97, 1, 0, 1, 256)])
def test_tables_much_wider_than_the_lengths(device, dtype, lengths, times, W, T, Tk, H, D):
    """Tables of 4096 tokens over short requests: most of the ranges that the prefix is
    split into hold no keys, some requests none at all."""
    q, blocks, tables, lens, sk, sv, gate = base._problem(device, lengths, W, T, Tk, H, 1, D, 64,
                                                          dtype, gated=True, seed=37)
    wide = torch.full((len(lengths), 64), 10**6, dtype=torch.int32, device=device)
    wide[:, ::3] = -1
    wide[:, :tables.shape[1]] = tables
    _attend_and_check(q, blocks, wide, lens, sk, sv, gate, W, times)
    if times == 1:      # what lies in the columns behind the lengths does not matter
        other = wide.clone()
        other[:, tables.shape[1]:] = 0
        a, b = (block_prefix_attention(q, blocks, t, lens, sk, sv, beam_width=W, gate=gate)
                for t in (wide, other))
        assert torch.equal(a, b)
