"""Attention over a cache held in 4 bits where numbers of very different sizes meet: groups, rows and weights far below others."""

import pytest
import torch

from plain_packed import PackedCase, attention
from test_packed_gpu import BF16, DEV, F32, bound_of, ints, on_device, ops_for

pytestmark = pytest.mark.gpu


def prompts(ops, case, planes, q, new, heads, scale, shares=0, window=None, softcap=None, sink=None):
    length, kv_heads, dim = case.lengths[0], case.kv_heads, case.dim
    out = torch.full((new, heads * dim), 7.0, dtype=q.dtype, device=DEV)
    ops.packed_attention_prompts(q.to(DEV), out, *planes, ints([0, new]), ints([length]), case.table.to(DEV), ints([0]), 0, 1, -(-new // 64), length, heads, kv_heads, dim,
                                 case.page, window, scale, softcap=softcap, sink=None if sink is None else sink.to(DEV), shares=shares)
    return out.cpu().double().view(new, heads, dim)


def tokens(ops, case, planes, q, positions, heads, scale, shares=0, window=None, softcap=None, sink=None):
    kv_heads, dim = case.kv_heads, case.dim
    out = torch.full((len(positions), heads * dim), 7.0, dtype=q.dtype, device=DEV)
    ops.packed_attention_tokens(q.to(DEV), out, *planes, ints([0] * len(positions)), ints(positions), case.table.to(DEV), heads, kv_heads, dim, case.page, window, scale,
                                case.lengths[0], softcap=softcap, sink=None if sink is None else sink.to(DEV), shares=shares)
    return out.cpu().double().view(len(positions), heads, dim)


def limit_of(found, scale, dtype, dim):
    """(bfloat16: keys, values and weights of prompts in float16, half a step of 2^-11 each; weights times steps of single tokens likewise)"""
    return bound_of(*found, scale, dtype, *((2.0 ** -10, dim, 2.0 ** -11) if dtype == BF16 else (2.0 ** -20, dim)))


def agrees(got, found, limit):
    off = ((got - found[0]).abs() / limit).max()
    assert off <= 1, float(off)


def shrunk(case, what, size):
    """Numbers of ``size`` beside ordinary ones; what the queries are to be multiplied by, or None."""
    if what == "a group of values":
        case.v[:, 0, :32] *= size
    elif what == "a group of one value":
        case.v[:, -1, :32] = size
    elif what == "the first rows' values":
        case.v[:40] *= size
    elif what == "a channel":
        case.v[:, 0, :32] = case.v[:, 0, :32].abs() + 0.125
        case.v[:, 0, 5] = size                                             # the least of its group: code 0
    elif what == "a group of keys":
        case.k[:, 0, :32] *= size
        return 1 / size
    elif what == "the last values":
        case.v[-20:] *= size
    return None


def beside_ordinary_ones(dtype, size, what, heads, kv_heads, dim, new):
    length = new if what == "the first rows' values" else 700             # (so that some queries see nothing else)
    case = PackedCase([length], kv_heads, dim, 16, dtype, seed=dim)
    grown = shrunk(case, what, size)
    _, planes = on_device(case)
    k, v = (x.double() for x in case.held())
    q = torch.randn(new, heads, dim, generator=torch.Generator().manual_seed(3))
    if grown is not None:
        q[:, :heads // kv_heads, :32] *= grown
    q = q.flatten(1).to(dtype)
    positions, scale = torch.arange(length - new, length), dim ** -0.5
    return ops_for(dtype), case, planes, q, positions, scale, attention(q.double().view(new, heads, dim), k, v, positions, scale)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("size", [1e-4, 1e-5, 1e-6, 3e-8, 1e-12])
@pytest.mark.parametrize("what", ["a group of values", "a group of one value", "the first rows' values", "a channel", "a group of keys", "the last values"])
@pytest.mark.parametrize("heads,kv_heads,dim,shares", [(2, 2, 64, 1), (4, 2, 128, 8), (3, 1, 40, 1), (2, 2, 96, 2)])
def test_small_numbers_in_prompts(dtype, size, what, heads, kv_heads, dim, shares):
    """What is held of a small group, row or channel reaches the result to the same relative error as ordinary numbers."""
    new = 300
    ops, case, planes, q, positions, scale, found = beside_ordinary_ones(dtype, size, what, heads, kv_heads, dim, new)
    agrees(prompts(ops, case, planes, q, new, heads, scale, shares=shares if dtype == BF16 else 0), found, limit_of(found, scale, dtype, dim))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shares", [1, 4])
@pytest.mark.parametrize("sink", [10.0, 15.0, 20.0, 40.0])
@pytest.mark.parametrize("window,softcap", [(None, None), (50, None), (None, 3.0)])
def test_sinks_far_above_the_scores(dtype, shares, sink, window, softcap):
    """A sink takes nearly all of a row's weight: what is left for the values is small, and right."""
    ops, heads, dim, page, length, new = ops_for(dtype), 2, 64, 16, 600, 300
    case = PackedCase([length], heads, dim, page, dtype, seed=5)
    _, planes = on_device(case)
    k, v = (x.double() for x in case.held())
    q = torch.randn(new, heads * dim, generator=torch.Generator().manual_seed(3)).to(dtype)
    sinks, positions = torch.tensor([sink, 0.5]), torch.arange(length - new, length)
    found = attention(q.double().view(new, heads, dim), k, v, positions, 0.125, window, softcap, sinks)
    limit = limit_of(found, 0.125, dtype, dim)
    extras = dict(window=window, softcap=softcap, sink=sinks, shares=shares if dtype == BF16 else 0)
    agrees(tokens(ops, case, planes, q, positions.tolist(), heads, 0.125, **extras), found, limit)
    agrees(prompts(ops, case, planes, q, new, heads, 0.125, **extras), found, limit)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("size", [1e-4, 1e-5, 1e-6, 3e-8, 1e-12])
@pytest.mark.parametrize("what", ["a group of values", "a group of one value", "the first rows' values", "a channel", "a group of keys", "the last values"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 2, 64), (4, 2, 128), (3, 1, 40), (20, 2, 96)])
def test_small_numbers_of_single_tokens(dtype, size, what, heads, kv_heads, dim):
    """As in prompts."""
    ops, case, planes, q, positions, scale, found = beside_ordinary_ones(dtype, size, what, heads, kv_heads, dim, 300)
    if what == "a channel":
        # Single tokens form a group's part of the result as a sum of step * (code - 8) and one of low + 8 * step, both of the group's size whatever the number
        # itself: their roundings, counted by a channel's own numbers in the limit, count by the largest channel's of the group here.
        groups = torch.arange(dim) // 32
        found = found[0], torch.stack([found[1][..., groups == g].amax(-1) for g in groups], -1), found[2]
    some = [0, 1, 39, 150, 299]
    found = [x[some] for x in found]
    agrees(tokens(ops, case, planes, q[some], positions[some].tolist(), heads, scale), found, limit_of(found, scale, dtype, dim))


def heavy_key(dtype, heads, kv_heads, dim, length, place, gap, seed):
    """Queries that one key, at ``place``, answers with a score about ``gap`` above all others'."""
    g = torch.Generator().manual_seed(seed)
    case = PackedCase([length], kv_heads, dim, 16, dtype, seed=seed, mean=0.0)
    along = torch.randn(kv_heads, dim, generator=g)
    along /= along.norm(dim=1, keepdim=True)
    case.k = (case.k.float() * 0.25 - (case.k.float() * 0.25 * along).sum(-1, keepdim=True) * along).to(dtype)
    case.k[place] = (8 * along).to(dtype)
    q = (along.repeat_interleave(heads // kv_heads, 0) * (gap * dim ** 0.5 / 8))[None] + 0.05 * torch.randn(6, heads, dim, generator=g)
    return case, q.flatten(1).to(dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 2, 64), (4, 1, 128), (20, 2, 32), (2, 1, 96)])
@pytest.mark.parametrize("shrink", [10, 16, 18, 20, 24, 30, 60])
@pytest.mark.parametrize("place", [0, 150, 690])
def test_the_key_that_carries_the_weight_has_small_values(dtype, heads, kv_heads, dim, shrink, place):
    """The result is that key's values, however much larger those of the keys are that have no weight."""
    ops, length = ops_for(dtype), 700
    case, q = heavy_key(dtype, heads, kv_heads, dim, length, place, 60.0, dim)
    case.v[place] = (case.v[place].float() * 2.0 ** -shrink).to(dtype)
    if shrink == 20:
        case.v[place, :, :16] *= 64.0                                     # (a step and a low that are not alike)
    _, planes = on_device(case)
    k, v = (x.double() for x in case.held())
    positions, scale = torch.arange(length - 6, length), dim ** -0.5
    found = attention(q.double().view(6, heads, dim), k, v, positions, scale)
    limit = limit_of(found, scale, dtype, dim)
    for shares in (0, 1, 8):
        agrees(tokens(ops, case, planes, q, positions.tolist(), heads, scale, shares=shares), found, limit)
    agrees(prompts(ops, case, planes, q, 6, heads, scale), found, limit)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 2, 64), (4, 1, 128)])
@pytest.mark.parametrize("gap", [6.0, 10.0, 12.0, 16.0, 20.0])
def test_the_key_that_carries_the_weight_has_no_values(dtype, heads, kv_heads, dim, gap):
    """A key whose values are zeros takes the weight: the others' small weights make the result."""
    ops, length = ops_for(dtype), 300
    case, q = heavy_key(dtype, heads, kv_heads, dim, length, 3, gap, dim)
    case.v[3] = 0
    _, planes = on_device(case)
    k, v = (x.double() for x in case.held())
    positions, scale = torch.arange(length - 6, length), dim ** -0.5
    found = attention(q.double().view(6, heads, dim), k, v, positions, scale)
    limit = limit_of(found, scale, dtype, dim)
    agrees(tokens(ops, case, planes, q, positions.tolist(), heads, scale), found, limit)
    agrees(prompts(ops, case, planes, q, 6, heads, scale), found, limit)


@pytest.mark.parametrize("heads,kv_heads,dim", [(12, 12, 64), (8, 2, 128)])
def test_results_repeat_bit_by_bit(heads, kv_heads, dim):
    ops, length, new = ops_for(BF16), 900, 300
    case = PackedCase([length], kv_heads, dim, 16, BF16, seed=1)
    _, planes = on_device(case)
    q = torch.randn(new, heads * dim, generator=torch.Generator().manual_seed(3)).bfloat16()
    for shares in (0, 1, 4):
        one, two = (prompts(ops, case, planes, q, new, heads, 0.125, shares=shares) for _ in range(2))
        assert torch.equal(one, two)
        at = list(range(length - 8, length))
        one, two = (tokens(ops, case, planes, q[:8], at, heads, 0.125, shares=shares) for _ in range(2))
        assert torch.equal(one, two)


def test_contexts_longer_than_their_table_in_float32():
    """What has no place in the table is a key of zeros, as a key without a page is: the kernels stay inside the unpacked rows."""
    ops, heads, dim, page, width = ops_for(F32), 2, 64, 16, 5
    case = PackedCase([width * page, width * page], heads, dim, page, F32, seed=3)
    _, planes = on_device(case)
    lengths, new = [600, 333], [200, 333]
    q = torch.randn(sum(new), heads * dim, generator=torch.Generator().manual_seed(3))
    out = torch.full((sum(new), heads * dim), 7.0, device=DEV)
    ops.packed_attention_prompts(q.to(DEV), out, *planes, ints([0, 200, 533]), ints(lengths), case.table.to(DEV), ints([0, 1]), 0, 2, 4 + 6, max(lengths), heads, heads, dim,
                                 page, None, 0.125)
    for item, rows in enumerate((slice(0, 200), slice(200, 533))):
        k, v = (torch.cat([case.context(item, x), torch.zeros(lengths[item] - width * page, heads, dim, dtype=torch.float64)]) for x in case.held())
        found = attention(q[rows].double().view(-1, heads, dim), k, v, torch.arange(lengths[item] - new[item], lengths[item]), 0.125)
        agrees(out[rows].cpu().double().view(-1, heads, dim), found, limit_of(found, 0.125, F32, dim))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_results_in_the_queries_place(dtype):
    """Single tokens read a head's query before its result is written, done again or not; prompts refuse it."""
    from pagedserve_b200.kernels.ops import KernelError

    ops, case, planes, q, positions, scale, found = beside_ordinary_ones(dtype, 1e-12, "a group of keys", 4, 2, 64, 300)
    limit, some = limit_of(found, scale, dtype, 64), [0, 17, 299]
    rows = q[some].to(DEV)
    ops.packed_attention_tokens(rows, rows, *planes, ints([0] * 3), ints(positions[some].tolist()), case.table.to(DEV), 4, 2, 64, 16, None, scale, 700)
    agrees(rows.cpu().double().view(3, 4, 64), [x[some] for x in found], limit[some])
    rows = q.to(DEV)
    with pytest.raises(KernelError, match="place"):
        ops.packed_attention_prompts(rows, rows, *planes, ints([0, 300]), ints([700]), case.table.to(DEV), ints([0]), 0, 1, 5, 700, 4, 2, 64, 16, None, scale)
    assert torch.equal(rows.cpu(), q)


@pytest.mark.parametrize("heads,kv_heads,dim,page", [(4, 2, 64, 16), (20, 2, 33, 1), (3, 3, 128, 64), (6, 1, 20, 4)])
@pytest.mark.parametrize("window,softcap,with_sink", [(None, None, True), (70, 5.0, False), (-128, None, True)])
@pytest.mark.parametrize("out_dtype", [BF16, F32])
@pytest.mark.parametrize("shares", [1, 8])
def test_rows_that_are_formed_again(heads, kv_heads, dim, page, window, softcap, with_sink, out_dtype, shares):
    """In float32 from the codes, under masks, caps and sinks, in rows of a wider buffer, with pages that are missing, beside rows that are not formed again."""
    ops, lengths, new = ops_for(BF16), [300, 200, 1], [150, 200, 1]
    case = PackedCase(lengths, kv_heads, dim, page, BF16, seed=dim, width=1)
    case.k[:300, 0, :16] *= 1e-12                                          # request 0, the first key head
    _, planes = on_device(case)
    table = case.table.clone()
    gone = 40 // page                                                      # request 1: one page of it, of every head
    table[1, gone] = -1
    k, v = case.held()
    g = torch.Generator().manual_seed(4)
    q = torch.randn(sum(new), heads, dim, generator=g)
    q[:150, :heads // kv_heads, :16] *= 1e12
    q = q.flatten(1).to(BF16)
    sink = torch.randn(heads, generator=g) if with_sink else None
    scale, starts = dim ** -0.5, [0, 150, 350, 351]
    wide = torch.zeros(351, heads * dim + 3, dtype=BF16, device=DEV)
    wide[:, 3:] = q.to(DEV)
    sinks = None if sink is None else sink.to(DEV)
    rows = torch.full((351, heads * dim + 5), 9.0, dtype=out_dtype, device=DEV)
    ops.packed_attention_prompts(wide[:, 3:], rows[:, :heads * dim], *planes, ints(starts), ints(lengths), table.to(DEV), ints([0, 1, 2]), 0, 3, 3 + 4 + 1, 300, heads, kv_heads,
                                 dim, page, window, scale, softcap=softcap, sink=sinks, shares=shares)
    single = torch.full((351, heads * dim + 5), 9.0, dtype=out_dtype, device=DEV)
    positions = [*range(150, 300), *range(200), 0]
    ops.packed_attention_tokens(wide[:, 3:], single[:, :heads * dim], *planes, ints([0] * 150 + [1] * 200 + [2]), ints(positions), table.to(DEV), heads, kv_heads, dim, page,
                                window, scale, 300, softcap=softcap, sink=sinks, shares=shares)
    for out in (rows, single):
        assert (out[:, heads * dim:] == 9.0).all()
        got = out[:, :heads * dim].cpu().double().view(351, heads, dim)
        for item in (0, 2):
            part = slice(starts[item], starts[item + 1])
            found = attention(q[part].double().view(-1, heads, dim), case.context(item, k), case.context(item, v), torch.arange(lengths[item] - new[item], lengths[item]), scale,
                              window, softcap, sink)
            agrees(got[part], found, limit_of(found, scale, BF16, dim))
        keys, values = case.context(1, k), case.context(1, v)
        for at in (0, 39, 63, 64, 128, 199):
            seen = torch.tensor([i for i in range(at + 1) if i // page != gone
                                 and (not window or (at - i < window if window > 0 else i // -window == at // -window))], dtype=torch.long)
            if not len(seen):
                assert (got[150 + at] == 0).all()
                continue
            found = attention(q[150 + at:151 + at].double().view(1, heads, dim), keys[seen], values[seen], torch.tensor([len(seen) - 1]), scale, None, softcap, sink)
            agrees(got[150 + at:151 + at], found, limit_of(found, scale, BF16, dim))


@pytest.mark.parametrize("dim", [20, 64, 128])
@pytest.mark.parametrize("k_scale,v_scale,q_scale", [(1.0, 3e30, 1.0), (3e5, 1.0, 2e5), (1.0, 1e-3, 1e20)])
def test_large_numbers_in_prompts_in_float32(dim, k_scale, v_scale, q_scale):
    ops, heads, length, new = ops_for(F32), 2, 200, 150
    case = PackedCase([length], heads, dim, 16, F32, seed=4)
    case.k, case.v = case.k * k_scale, case.v * v_scale
    _, planes = on_device(case)
    k, v = (x.double() for x in case.held())
    q = torch.randn(new, heads * dim, generator=torch.Generator().manual_seed(2)) * q_scale
    scale = 0.125 / max(1.0, k_scale * q_scale)
    found = attention(q.double().view(new, heads, dim), k, v, torch.arange(length - new, length), scale)
    agrees(prompts(ops, case, planes, q, new, heads, scale), found, limit_of(found, scale, F32, dim))
