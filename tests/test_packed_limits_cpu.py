"""Sizes that the operators over a cache of 4 bits and of log probabilities choose by themselves, and what they refuse, without a GPU."""

import math

import pytest


def test_what_lies_beyond_a_sample_fits_the_lists():
    """Whatever the vocabulary and the alternatives: fewer than one row of a million overflows, and the sample has enough tokens."""
    from pagedserve_b200.kernels.ops import MOST_ALTERNATIVES, Ops

    for top in range(1, MOST_ALTERNATIVES + 1):
        for V in (8192, 9000, 20000, 32000, 40001, 50257, 65536, 100003, 128256, 151936, 200064, 262144, 10 ** 6, 10 ** 7):
            every = Ops.sample_every(V, top)
            assert every >= 1 and -(-V // every) >= top
            # the list's length over `every`: a sum of `top` waits, exponential ones of mean 1 (Gamma); above its mean P(sum > x) <= e^(top - x) (x / top)^top
            x = Ops.HEAD_LIST / every
            assert x > top and top - x + top * math.log(x / top) < math.log(1e-6)
    assert Ops.sample_every(50257, 32) == 25 and Ops.sample_every(20000, 5) == 10           # (as many as ever where they are enough)


def test_unpacked_rows_have_a_place_for_every_position():
    """Prompts in float32 read position p of an item in page p // 64 of that item's row: within the row for any context up to the bound given, however few pages
    the request's own table has."""
    from pagedserve_b200.kernels.ops import Ops

    for longest in (1, 63, 64, 65, 100, 1000, 4097, 32768):
        span = Ops.unpacked_span(longest)
        assert span % 64 == 0 and (longest - 1) // 64 < span // 64 and span < longest + 64


@pytest.mark.parametrize("kv_heads,dim,longest,portion", [(25, 64, 32768, 512), (12, 64, 1024, 128), (8, 128, 131072, 4096)])
def test_unpacked_rows_of_a_growing_context(kv_heads, dim, longest, portion):
    """A step's arena keeps what it was ever asked for: a prompt that runs in portions must not ask for a little more with each of them."""
    import torch

    from pagedserve_b200.cache.budget import unpacking_reserve
    from pagedserve_b200.cache.manager import KVNeed
    from pagedserve_b200.kernels.ops import Ops, StepArena

    def grown(asked):
        arena = StepArena()
        for end in range(portion, longest + 1, portion):
            arena.reset()
            arena.empty((asked(Ops.unpacked_span(end) * 2 * kv_heads * dim * 4) // 4,), torch.float32, torch.device("meta"))
        return sum(chunk.numel() - StepArena.ALIGN for chunk in arena.chunks)

    largest = longest * 2 * kv_heads * dim * 4
    reserve = unpacking_reserve([KVNeed(kv_heads, dim)], longest, 64)
    assert grown(Ops.unpacked_bytes) <= max(reserve, StepArena.CHUNK_BYTES)
    assert largest <= reserve <= 4 * max(largest, Ops.UNPACKED_BYTES)
    if largest > 4 * StepArena.CHUNK_BYTES:
        assert grown(lambda needed: needed) > 4 * reserve                  # (as it would be otherwise)


def test_what_is_kept_for_unpacked_rows():
    from pagedserve_b200.cache.budget import unpacking_reserve
    from pagedserve_b200.cache.manager import KVNeed

    assert unpacking_reserve([], 1024, 8) == 0
    assert unpacking_reserve([KVNeed(12, 64)], 1024, 1) == 2 * (1 << 23)                   # 6 MB of one request
    assert unpacking_reserve([KVNeed(12, 64), KVNeed(25, 64)], 1024, 8) == 2 * (1 << 27)   # 8 requests of 13 MB
    assert unpacking_reserve([KVNeed(25, 64)], 1024, 1000) == 2 * (1 << 29)
    assert unpacking_reserve([KVNeed(32, 128)], 10 ** 5, 8) == 2 * (1 << 32)               # one request's rows, whatever they need


def test_tables_of_more_positions_than_are_counted_are_refused():
    """(single tokens over a table of 2^31 positions saw none of them)"""
    import torch

    from pagedserve_b200.kernels.ops import KernelError, Ops, packed_slab_bytes

    ops, page, dim = Ops(torch.bfloat16), 64, 64
    slab = packed_slab_bytes(page, dim)
    pool = torch.empty((2, 2, 1, slab), dtype=torch.uint8)
    ask = lambda width: ops._packed_pools("packed_attention_tokens", pool[:, 0], pool[:, 1], 2 * slab, 1, dim, page, torch.empty((1, width), dtype=torch.int32, device="meta"))
    with pytest.raises(KernelError, match="positions"):
        ask(2 ** 25)
    with pytest.raises(KernelError, match="CUDA device"):
        ask(2 ** 25 - 2 ** 10)
