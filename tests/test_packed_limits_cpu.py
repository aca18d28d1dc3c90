"""Sizes that the operators over a cache of 4 bits and of log probabilities choose by themselves, and what they refuse, without a GPU."""

import math


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
