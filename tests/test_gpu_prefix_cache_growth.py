"""Requests that grow in the 8-bit prefix cache: pages out of one list over many
calls, counted on the GPU."""

import pytest
import torch

import test_gpu_prefix_cache as base
from kadllm_amd import _lib
from kadllm_amd.ops import block_prefix_attention, prefix_block_tables, write_prefix_blocks
from oracle import prefix_cache_ref as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("taken", [-3, 0, 1, 7, 11, 12, 2**31 - 1])
def test_tables_behind_the_pages_taken(device, taken):
    """The same tables as from the rest of the list, and a count that goes on."""
    lengths, starts = [70, 64, 1, 33, 0], [64, 64, 0, 1, 0]
    held = [[30, 31, -1], [32, 33, -1], [-1] * 3, [34, -1, -1], [-1] * 3]
    free = list(range(12))
    skip = max(taken, 0)
    want, n = ref.block_tables(lengths, free[skip:], 32, 96, starts, held)
    got, used = prefix_block_tables(base._ints(lengths, device), base._ints(free, device),
                                    block_size=32, max_length=96, starts=base._ints(starts, device),
                                    tables=base._ints(held, device),
                                    taken=base._ints([taken], device))
    assert got.tolist() == want and used.tolist() == [min(skip + n, 2**31 - 1)]


def test_the_entry_point_without_a_count(device):
    """kad_prefix_block_tables: the list from its front."""
    lengths, free = base._ints([70, 0, 32], device), base._ints([5, 6, 7, 8, 9], device)
    out, used = base._ints([[0] * 3] * 3, device), base._ints([0], device)
    _lib.call("kad_prefix_block_tables", lengths.data_ptr(), None, None, 0, free.data_ptr(), 5,
              out.data_ptr(), 3, used.data_ptr(), 3, 32, 96, _lib.stream_of(out))
    assert out.tolist() == [[5, 6, 7], [-1] * 3, [8, -1, -1]] and used.tolist() == [4]


def test_a_captured_growth_step_gives_out_no_page_twice(device):
    """One captured step of one token for each request, replayed past several pages'
    ends with tables, lengths and the count carried along: pages of their own for
    every request, and the cache and attention of the same steps made one by one."""
    B, W, H, HK, D, block, most = 3, 2, 4, 2, 64, 32, 160
    gen = torch.Generator(device=device).manual_seed(40)
    rand = lambda *s: torch.randn(*s, generator=gen, device=device).bfloat16()  # noqa: E731
    free = torch.randperm(15, generator=gen, device=device).int()
    prompt = [rand(B, 70, HK, D) for _ in range(2)]
    first = base._ints([70, 31, 1], device)

    def start():
        blocks = base._pool(device, 15, HK, block, D, 40)
        tables, taken = prefix_block_tables(first, free, block_size=block, max_length=most)
        write_prefix_blocks(blocks, *prompt, tables, first)
        return blocks, tables, taken, first.clone()

    def step(blocks, tables, taken, lengths, k1, v1, q):
        longer = lengths + 1
        new_tables, new_taken = prefix_block_tables(longer, free, block_size=block,
                                                    max_length=most, starts=lengths, tables=tables,
                                                    taken=taken)
        write_prefix_blocks(blocks, k1, v1, new_tables, longer, starts=lengths)
        out = block_prefix_attention(q, blocks, new_tables, longer, beam_width=W)
        tables.copy_(new_tables)
        taken.copy_(new_taken)
        lengths.copy_(longer)
        return out

    new = lambda: [rand(B, 1, HK, D), rand(B, 1, HK, D), rand(B * W, 1, H, D)]  # noqa: E731
    inputs = new()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*start(), *inputs)
    torch.cuda.current_stream().wait_stream(side)
    state, eager = start(), start()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*state, *inputs)
    for n in range(1, 71):
        for dst, src in zip(inputs, new()):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, step(*eager, *inputs))
        for x, y in zip((*state[0], *state[1:]), (*eager[0], *eager[1:])):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
        lengths = [70 + n, 31 + n, 1 + n]
        assert state[3].tolist() == lengths
        pages = [p for row in state[1].tolist() for p in row if p >= 0]
        assert len(pages) == sum(-(-m // block) for m in lengths) == state[2].item()
        assert len(set(pages)) == len(pages) and set(pages) <= set(range(15))
