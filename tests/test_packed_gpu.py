"""A cache held in 4 bits (csrc/packed_cache.cu, attention_packed.cu) against the format written out number by number and 64-bit attention."""

import pytest
import torch

from plain_packed import PackedCase, attention, held

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32


def ops_for(dtype):
    from test_kernels_gpu import ops_for as make

    return make(dtype)


def ints(values):
    return torch.as_tensor(values, dtype=torch.int32).to(DEV)


def on_device(case):
    """The written pool's planes and the page stride."""
    pool = case.filled().to(DEV)
    return pool, (pool[:, 0], pool[:, 1], pool.stride(0))


# ------------------------------------------------------------------------------------------------ rows in and out
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kv_heads,dim,page", [(1, 64, 16), (3, 128, 8), (2, 16, 1), (2, 48, 4), (1, 80, 32), (2, 33, 2), (1, 256, 64), (5, 96, 16), (1, 1, 1)])
def test_written_bytes(dtype, kv_heads, dim, page):
    """Every byte of the pool: the written rows' as the format says, all others as they were."""
    ops = ops_for(dtype)
    case = PackedCase([1, page, page + 1, 3 * page + 2, 17], kv_heads, dim, page, dtype, seed=dim, width=2)
    want = case.filled()
    got = case.pool.to(DEV)
    # rows of a wider buffer whose start is no multiple of 16 bytes where the head size is odd
    rows = torch.zeros((len(case.positions), 3 * kv_heads * dim + 5), dtype=dtype)
    rows[:, kv_heads * dim:2 * kv_heads * dim] = case.k.flatten(1)
    rows[:, 2 * kv_heads * dim:3 * kv_heads * dim] = case.v.flatten(1)
    rows = rows.to(DEV)
    ops.kv_append_packed(rows[:, kv_heads * dim:2 * kv_heads * dim], rows[:, 2 * kv_heads * dim:3 * kv_heads * dim], case.token_row.to(DEV),
                         case.positions.to(DEV), case.table.to(DEV), got[:, 0], got[:, 1], got.stride(0), kv_heads, dim, page)
    # (a padding byte of a slab is nobody's)
    groups = -(-dim // 32)
    assert torch.equal(got.cpu()[..., :page * groups * 20], want[..., :page * groups * 20])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kv_heads,dim,page", [(25, 64, 16), (3, 33, 4), (8, 128, 64)])
def test_written_bytes_of_many_tokens(dtype, kv_heads, dim, page):
    """Tokens enough that a CTA takes several, a number of them that is no multiple of four, some without a place."""
    ops, case = ops_for(dtype), PackedCase([1501, 700, 3], kv_heads, dim, page, dtype, seed=dim)
    got = case.pool.to(DEV)
    positions = case.positions.clone()
    positions[5::7] = -1
    ops.kv_append_packed(case.k.flatten(1).to(DEV), case.v.flatten(1).to(DEV), case.token_row.to(DEV), positions.to(DEV), case.table.to(DEV), got[:, 0],
                         got[:, 1], got.stride(0), kv_heads, dim, page)
    keep = torch.ones(len(positions), dtype=torch.bool)
    keep[5::7] = False
    case.k, case.v, case.token_row, case.positions = case.k[keep], case.v[keep], case.token_row[keep], case.positions[keep]
    groups = -(-dim // 32)
    assert torch.equal(got.cpu()[..., :page * groups * 20], case.filled()[..., :page * groups * 20])


def special_rows(dim):
    g = torch.Generator().manual_seed(5)
    rows = [torch.zeros(dim), torch.full((dim,), 3.25), torch.full((dim,), -1.0000001), torch.randn(dim, generator=g) * 1e-30,
            torch.randn(dim, generator=g) * 1e30, torch.randn(dim, generator=g) * 1e-42, torch.arange(dim).float(),
            torch.where(torch.arange(dim) == 3, 1e4, 0.0), torch.where(torch.arange(dim) == 3, float("nan"), 1.0),
            torch.where(torch.arange(dim) == 40, float("inf"), 1.0), torch.where(torch.arange(dim) == 0, float("-inf"), 1.0),
            torch.where(torch.arange(dim) % 2 == 0, 3e38, -3e38), torch.full((dim,), -3.4e38)]
    return torch.stack(rows)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_unusual_numbers_and_reading_back(dtype):
    """Rows of zeros, of one number, of denormals, with NaN, infinities and ranges beyond float32; a number is within half a step of what is held."""
    ops, dim, page = ops_for(dtype), 64, 16
    rows = special_rows(dim).to(dtype)
    case = PackedCase([len(rows)], 1, dim, page, dtype)
    case.k, case.v = rows[:, None], rows.flip(0)[:, None]
    pool = case.pool.to(DEV)
    planes = (pool[:, 0], pool[:, 1], pool.stride(0))
    ops.kv_append_packed(case.k.flatten(1).to(DEV), case.v.flatten(1).to(DEV), case.token_row.to(DEV), case.positions.to(DEV), case.table.to(DEV),
                         *planes, 1, dim, page)
    assert torch.equal(pool.cpu(), case.filled())
    out = torch.full((1, 2, 1, 16, dim), 7.0, dtype=dtype, device=DEV)
    ops.kv_unpack(*planes, ints([len(rows)]), case.table.to(DEV), ints([0]), 0, 1, 16, out, 1, dim, page)
    want = torch.from_numpy(held(rows.float().numpy()))
    assert torch.equal(torch.nan_to_num(out[0, 0, 0, :len(rows)].float().cpu(), nan=123.0), torch.nan_to_num(want.to(dtype).float(), nan=123.0))
    assert (out[0, :, 0, len(rows):] == 7.0).all()                       # rows behind the last one stay as they were
    finite = rows[:8].float()
    for part in (slice(0, 32), slice(32, 64)):
        x, y = finite[:, part], want[:8, part]
        step = (x.amax(1, keepdim=True) - x.amin(1, keepdim=True)) / 15
        # low is down by at most 2^-7 of itself, step up by as much: half of a step that spans both
        bound = 0.5 * (step + x.amin(1, keepdim=True).abs() * 2.0 ** -7 / 15) * (1 + 2.0 ** -7) + 2.0 ** -133 + x.abs() * 2.0 ** -22
        assert ((x - y).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_tokens_that_have_no_place(dtype):
    """Positions below 0, pages that are missing or outside the pool, positions beyond the table: nothing is written for them."""
    ops, case = ops_for(dtype), PackedCase([40], 2, 64, 16, dtype)
    pool = case.pool.to(DEV)
    before = pool.clone()
    table = case.table.clone()
    table[0, 0], table[0, 1], table[0, 2] = -1, case.pages, 2 ** 30
    positions = torch.tensor([-1, 3, 17, 40, 48, 10 ** 6, -2 ** 31, 2 ** 31 - 1], dtype=torch.int32)
    rows = torch.ones((8, 128), dtype=dtype, device=DEV)
    ops.kv_append_packed(rows, rows, ints([0] * 8), positions.to(DEV), table.to(DEV), pool[:, 0], pool[:, 1], pool.stride(0), 2, 64, 16)
    assert torch.equal(pool, before)
    out = torch.full((3, 2, 2, 16, 64), 5.0, dtype=dtype, device=DEV)
    ops.kv_unpack(pool[:, 0], pool[:, 1], pool.stride(0), ints([40]), table.to(DEV), ints([0]), 0, 1, 48, out, 2, 64, 16)
    assert (out == 5.0).all()


def test_one_plane_at_a_time():
    ops, case = ops_for(BF16), PackedCase([20], 2, 64, 16, BF16)
    pool = case.pool.to(DEV)
    place = (case.token_row.to(DEV), case.positions.to(DEV), case.table.to(DEV), pool[:, 0], pool[:, 1], pool.stride(0), 2, 64, 16)
    ops.kv_append_packed(None, case.v.flatten(1).to(DEV), *place)
    want = case.filled()
    assert torch.equal(pool.cpu()[:, 1], want[:, 1]) and (pool[:, 0] == 0xA5).all()
    ops.kv_append_packed(case.k.flatten(1).to(DEV), None, *place)
    assert torch.equal(pool.cpu(), want)


def test_unpacked_pages_of_another_size():
    ops, case = ops_for(F32), PackedCase([5, 70, 33], 2, 96, 8, F32, seed=3)
    _, planes = on_device(case)
    out = torch.zeros((2 * 2, 2, 2, 64, 96), device=DEV)
    ops.kv_unpack(*planes, ints([33, 70, 5]), case.table.to(DEV), ints([2, 1, 0]), 1, 2, 128, out, 2, 96, 8)     # requests 1 and 0, as items 1 and 2
    for plane, rows in enumerate(case.held()):
        for item, request in ((0, 1), (1, 0)):
            length = case.lengths[request]
            flat = out[2 * item:2 * item + 2, plane].transpose(1, 2).flatten(0, 1).cpu()
            assert torch.equal(flat[:length], case.context(request, rows)[:length].float())
            assert (flat[length:] == 0).all()


# ------------------------------------------------------------------------------------------------ single tokens
def bound_of(want, weighted, sizes, scale, out_dtype, softmax_step, dim, key_step=0.0):
    """How far a result may be off: scores formed in float32 from sums of up to ``dim`` products (and numbers about 8 steps in size beside them),
    2^-24 each, keys rounded by ``key_step`` (a score is then off by that much of the sum of |q| |k|), weights by ``softmax_step``, sums over the keys in
    float32, one rounding of the result."""
    score = ((dim + 64) * 2.0 ** -24 * 4 + key_step) * scale * sizes[..., None]
    return (2 * score + softmax_step + 2.0 ** -18) * 4 * weighted + torch.finfo(out_dtype).eps / 2 * want.abs() + 1e-30


MASKS = [(None, None, False), (70, 5.0, True), (-128, None, True)]
SHAPES = [(12, 12, 64, 16), (6, 2, 48, 8), (8, 1, 40, 64), (4, 2, 128, 32), (16, 2, 96, 1), (10, 5, 80, 4), (4, 4, 160, 16), (32, 2, 64, 16), (2, 1, 256, 16), (6, 6, 20, 2)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,kv_heads,dim,page", SHAPES)
@pytest.mark.parametrize("window,softcap,with_sink", MASKS)
def test_single_tokens(dtype, heads, kv_heads, dim, page, window, softcap, with_sink):
    ops = ops_for(dtype)
    lengths = [1, 2, 15, 16, 17, 31, 33, 64, 127, 129, 300, 520]
    case = PackedCase(lengths, kv_heads, dim, page, dtype, seed=dim + heads, width=1)
    _, planes = on_device(case)
    k, v = case.held()
    g = torch.Generator().manual_seed(9)
    # the last token of every request, an older one of the longest, and one that stands nowhere
    rows = list(range(len(lengths))) + [11, 11]
    positions = [length - 1 for length in lengths] + [77, -1]
    q = torch.randn(len(rows), heads * dim + 8, generator=g).to(dtype)
    sink = torch.randn(heads, generator=g) if with_sink else None
    scale = dim ** -0.5
    for out_dtype in {dtype, F32}:
        out = torch.full((len(rows), heads * dim + 8), 9.0, dtype=out_dtype, device=DEV)
        ops.packed_attention_tokens(q.to(DEV)[:, :heads * dim], out[:, :heads * dim], *planes, ints(rows), ints(positions), case.table.to(DEV), heads,
                                    kv_heads, dim, page, window, scale, max(lengths), softcap=softcap, sink=None if sink is None else sink.to(DEV))
        assert (out[:, heads * dim:] == 9.0).all()
        got = out[:, :heads * dim].cpu().double().view(-1, heads, dim)
        assert (got[-1] == 0).all()
        for i, (row, position) in enumerate(zip(rows[:-1], positions)):
            want, weighted, sizes = attention(q[i:i + 1, :heads * dim].double().view(1, heads, dim), case.context(row, k), case.context(row, v),
                                              torch.tensor([position]), scale, window, softcap, sink)
            # (bfloat16: a weight times its step is rounded to float16, 2^-11, before it meets the codes)
            assert ((got[i:i + 1] - want).abs() <= bound_of(want, weighted, sizes, scale, out_dtype, 2.0 ** -11 if dtype == BF16 else 0.0, dim)).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("tokens,length", [(1, 5000), (3, 2049), (40, 700), (1, 1)])
def test_long_contexts_and_many_tokens(dtype, tokens, length):
    """Keys shared out over CTAs, and tokens enough that they are not."""
    ops, heads, kv_heads, dim, page = ops_for(dtype), 4, 2, 64, 16
    case = PackedCase([length], kv_heads, dim, page, dtype, seed=length)
    _, planes = on_device(case)
    k, v = (x.double() for x in case.held())
    q = torch.randn(tokens, heads * dim, generator=torch.Generator().manual_seed(1)).to(dtype)
    positions = [length - 1 - i * (length // (tokens + 1)) for i in range(tokens)]
    out = torch.empty((tokens, heads * dim), dtype=dtype, device=DEV)
    for bound in (length, 4 * length + 1000):                            # what a graph passes is longer than any context
        ops.packed_attention_tokens(q.to(DEV), out, *planes, ints([0] * tokens), ints(positions), case.table.to(DEV), heads, kv_heads, dim, page, None,
                                    0.125, bound)
        want, weighted, sizes = attention(q.double().view(tokens, heads, dim), k, v, torch.tensor(positions), 0.125)
        limit = bound_of(want, weighted, sizes, 0.125, dtype, 2.0 ** -11 if dtype == BF16 else 0.0, dim)
        assert ((out.cpu().double().view(tokens, heads, dim) - want).abs() <= limit).all()


@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("heads,kv_heads", [(6, 2), (8, 2), (5, 1)])
@pytest.mark.parametrize("window,softcap,with_sink", [(None, None, False), (20, 3.0, True)])
def test_many_tokens_of_grouped_heads_in_float32(dim, heads, kv_heads, window, softcap, with_sink):
    """Two query heads of a key head at a time, and one that is left."""
    ops, page, tokens = ops_for(F32), 16, 30
    lengths = [1 + 13 * i % 90 for i in range(tokens)]
    case = PackedCase(lengths, kv_heads, dim, page, F32, seed=dim)
    _, planes = on_device(case)
    g = torch.Generator().manual_seed(heads)
    q = torch.randn(tokens, heads * dim, generator=g)
    sink = torch.randn(heads, generator=g) if with_sink else None
    out = torch.full((tokens, heads * dim), 7.0, device=DEV)
    at = [length - 1 for length in lengths]
    ops.packed_attention_tokens(q.to(DEV), out, *planes, ints(range(tokens)), ints(at), case.table.to(DEV), heads, kv_heads, dim, page, window, 0.125, 90,
                                softcap=softcap, sink=None if sink is None else sink.to(DEV))
    held_k, held_v = case.held()
    for i in range(tokens):
        want, weighted, sizes = attention(q[i:i + 1].double().view(1, heads, dim), case.context(i, held_k), case.context(i, held_v), torch.tensor([at[i]]), 0.125,
                                          window, softcap, sink)
        assert ((out[i:i + 1].cpu().double().view(1, heads, dim) - want).abs() <= bound_of(want, weighted, sizes, 0.125, F32, 0.0, dim)).all()


@pytest.mark.parametrize("shares,warps", [(1, 4), (1, 8), (2, 8), (4, 8), (8, 4), (8, 8)])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 4, 32), (6, 2, 64), (3, 3, 96), (8, 1, 128), (20, 2, 128)])
def test_shares_and_warps_of_single_tokens(shares, warps, heads, kv_heads, dim):
    """Contexts of fewer keys than warps, of one, of none."""
    ops, page, lengths = ops_for(BF16), 16, [1200, 17, 1, 333]
    case = PackedCase(lengths, kv_heads, dim, page, BF16, seed=dim)
    _, planes = on_device(case)
    q = torch.randn(5, heads * dim, generator=torch.Generator().manual_seed(1)).bfloat16()
    out = torch.full((5, heads * dim), 7.0, device=DEV)
    at = [1199, 16, 0, 332, -1]
    ops.packed_attention_tokens(q.to(DEV), out, *planes, ints([0, 1, 2, 3, 0]), ints(at), case.table.to(DEV), heads, kv_heads, dim, page, None, 0.125, 1200,
                                shares=shares, warps=warps)
    assert (out[4] == 0).all()
    held_k, held_v = case.held()
    for i in range(4):
        want, weighted, sizes = attention(q[i:i + 1].double().view(1, heads, dim), case.context(i, held_k), case.context(i, held_v), torch.tensor([at[i]]), 0.125)
        limit = bound_of(want, weighted, sizes, 0.125, F32, 2.0 ** -11, dim)
        assert ((out[i:i + 1].cpu().double().view(1, heads, dim) - want).abs() <= limit).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("k_scale,v_scale,q_scale", [(1e4, 1e6, 1e-4), (1e-6, 1e-9, 1e3), (1.0, 3e30, 1.0), (1.0, 1e-30, 1.0), (3e5, 1.0, 2e5), (0.0, 0.0, 1.0)])
def test_sizes_of_numbers(dtype, k_scale, v_scale, q_scale):
    """Keys, values and queries far from 1 in size."""
    ops, heads, dim, page, length = ops_for(dtype), 2, 64, 16, 150
    case = PackedCase([length], heads, dim, page, dtype, seed=4)
    case.k, case.v = (case.k.float() * k_scale).to(dtype), (case.v.float() * v_scale).to(dtype)
    _, planes = on_device(case)
    k, v = (x.double() for x in case.held())
    q = (torch.randn(20, heads * dim, generator=torch.Generator().manual_seed(2)) * q_scale).to(dtype)
    positions = list(range(130, 150))
    scale = 0.125 / max(1.0, k_scale * q_scale)                          # (so that the softmax is not of one key)
    want, weighted, sizes = attention(q.double().view(20, heads, dim), k, v, torch.tensor(positions), scale)
    limit = bound_of(want, weighted, sizes, scale, dtype, 2.0 ** -10 if dtype == BF16 else 0.0, dim)
    out = torch.empty((20, heads * dim), dtype=dtype, device=DEV)
    ops.packed_attention_tokens(q.to(DEV), out, *planes, ints([0] * 20), ints(positions), case.table.to(DEV), heads, heads, dim, page, None, scale, length)
    assert ((out.cpu().double().view(20, heads, dim) - want).abs() <= limit).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_nan_and_infinity(dtype):
    """A NaN among a request's keys or values reaches the tokens that see its row, and no other; an infinite query is NaN."""
    ops, heads, dim, page = ops_for(dtype), 2, 64, 16
    case = PackedCase([100, 100, 100], heads, dim, page, dtype, seed=6)
    case.k[50, 0, 3] = float("nan")                                     # request 0, head 0
    case.v[150, 1, 40] = float("inf")                                   # request 1, head 1, second group
    _, planes = on_device(case)
    q = torch.randn(6, heads * dim, generator=torch.Generator().manual_seed(3)).to(dtype)
    q[5, 0] = float("inf")
    out = torch.empty((6, heads * dim), dtype=dtype, device=DEV)
    ops.packed_attention_tokens(q.to(DEV), out, *planes, ints([0, 0, 1, 1, 2, 2]), ints([49, 50, 49, 50, 99, 99]), case.table.to(DEV), heads, heads, dim,
                                page, None, 0.125, 100)
    bad = out.isnan().cpu().view(6, heads, 2, 32)
    want = torch.zeros_like(bad)
    want[1, 0] = True
    want[3, 1, 1] = True
    want[5, 0] = True
    assert torch.equal(bad, want)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_missing_pages_are_not_seen(dtype):
    ops, heads, dim, page = ops_for(dtype), 2, 64, 16
    case = PackedCase([64], heads, dim, page, dtype, seed=8)
    _, planes = on_device(case)
    table = case.table.clone()
    table[0, 1], table[0, 3] = -1, case.pages + 5
    q = torch.randn(2, heads * dim, generator=torch.Generator().manual_seed(3)).to(dtype)
    out = torch.empty((2, heads * dim), dtype=dtype, device=DEV)
    ops.packed_attention_tokens(q.to(DEV), out, *planes, ints([0, 0]), ints([63, 500]), table.to(DEV), heads, heads, dim, page, None, 0.125, 600)
    k, v = case.held()
    kept = torch.cat([torch.arange(16), torch.arange(32, 48)])
    want, weighted, sizes = attention(q.double().view(2, heads, dim), k[kept].double(), v[kept].double(), torch.tensor([31, 31]), 0.125)
    limit = bound_of(want, weighted, sizes, 0.125, dtype, 2.0 ** -11 if dtype == BF16 else 0.0, dim)
    assert ((out.cpu().double().view(2, heads, dim) - want).abs() <= limit).all()


# ------------------------------------------------------------------------------------------------ portions of prompts
PROMPT_SHAPES = [(4, 4, 64, 16), (8, 2, 128, 16), (3, 3, 64, 64), (4, 2, 64, 8), (6, 3, 96, 16), (4, 4, 48, 4), (5, 1, 80, 1), (2, 2, 128, 32), (3, 3, 20, 2)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,kv_heads,dim,page", PROMPT_SHAPES)
@pytest.mark.parametrize("window,softcap,with_sink", MASKS)
def test_prompt_portions(dtype, heads, kv_heads, dim, page, window, softcap, with_sink):
    """Whole prompts and portions behind a context, of lengths around a tile's; the items in front and the rows of other tokens stay as they are."""
    ops = ops_for(dtype)
    lengths, new = [40, 16, 129, 300, 200, 517], [1, 16, 129, 77, 200, 128]
    case = PackedCase(lengths, kv_heads, dim, page, dtype, seed=dim, width=1)
    _, planes = on_device(case)
    k, v = case.held()
    g = torch.Generator().manual_seed(5)
    starts = [0]
    for count in new:
        starts.append(starts[-1] + count)
    q = torch.randn(starts[-1] + 3, heads * dim, generator=g).to(dtype)
    sink = torch.randn(heads, generator=g) if with_sink else None
    scale = dim ** -0.5
    blocks = sum(-(-count // 64) for count in new[1:])
    for out_dtype in {dtype, F32}:
        out = torch.full((starts[-1] + 3, heads * dim), 9.0, dtype=out_dtype, device=DEV)
        ops.packed_attention_prompts(q.to(DEV), out, *planes, ints(starts), ints(lengths), case.table.to(DEV), ints(range(6)), 1, 5, blocks, max(lengths),
                                     heads, kv_heads, dim, page, window, scale, softcap=softcap, sink=None if sink is None else sink.to(DEV))
        assert (out[:1] == 9.0).all() and (out[starts[-1]:] == 9.0).all()
        got = out.cpu().double().view(-1, heads, dim)
        for item in range(1, 6):
            rows = slice(starts[item], starts[item + 1])
            want, weighted, sizes = attention(q[rows].double().view(-1, heads, dim), case.context(item, k), case.context(item, v),
                                              torch.arange(lengths[item] - new[item], lengths[item]), scale, window, softcap, sink)
            # (bfloat16: keys, values and weights are rounded to float16, half a step of 2^-11 each)
            limit = bound_of(want, weighted, sizes, scale, out_dtype, *((2.0 ** -10, dim, 2.0 ** -11) if dtype == BF16 else (2.0 ** -20, dim)))
            assert ((got[rows] - want).abs() <= limit).all(), (item, float(((got[rows] - want).abs() / limit).max()))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("k_scale,v_scale,q_scale", [(1e4, 1e6, 1e-4), (1e-6, 1e-9, 1e3), (1.0, 3e30, 1.0), (1.0, 1e-30, 1.0), (3e5, 1.0, 2e5), (0.0, 0.0, 1.0),
                                                     (1.0, 1e-3, 1e20), (1e-4, 1.0, 1e-20)])
def test_sizes_of_numbers_in_prompts(dtype, k_scale, v_scale, q_scale):
    """Keys, values and queries far from 1 in size: beyond float16's range on either side."""
    ops, heads, dim, page, length, new = ops_for(dtype), 2, 64, 16, 200, 150
    if dtype == F32 and (v_scale > 1e7 or k_scale * q_scale > 1e7):
        pytest.skip("the kernel over float32 pages has bounds of its own")
    case = PackedCase([length], heads, dim, page, dtype, seed=4)
    case.k, case.v = (case.k.float() * k_scale).to(dtype), (case.v.float() * v_scale).to(dtype)
    _, planes = on_device(case)
    k, v = (x.double() for x in case.held())
    q = (torch.randn(new, heads * dim, generator=torch.Generator().manual_seed(2)) * q_scale).to(dtype)
    scale = 0.125 / max(1.0, k_scale * q_scale)
    want, weighted, sizes = attention(q.double().view(new, heads, dim), k, v, torch.arange(length - new, length), scale)
    limit = bound_of(want, weighted, sizes, scale, dtype, *((2.0 ** -10, dim, 2.0 ** -11) if dtype == BF16 else (2.0 ** -20, dim)))
    out = torch.empty((new, heads * dim), dtype=dtype, device=DEV)
    ops.packed_attention_prompts(q.to(DEV), out, *planes, ints([0, new]), ints([length]), case.table.to(DEV), ints([0]), 0, 1, 3, length, heads, heads, dim,
                                 page, None, scale)
    assert ((out.cpu().double().view(new, heads, dim) - want).abs() <= limit).all()


def test_nan_and_missing_pages_in_prompts():
    """A NaN among the values reaches the rows that see it and no other; keys without a page are not seen."""
    ops, heads, dim, page, length = ops_for(BF16), 2, 64, 16, 160
    case = PackedCase([length, length], heads, dim, page, BF16, seed=6)
    case.v[100, 1, 40] = float("nan")                                   # request 0, head 1, second group
    _, planes = on_device(case)
    table = case.table.clone()
    table[1, 2], table[1, 5] = -1, case.pages
    q = torch.randn(2 * length, heads * dim, generator=torch.Generator().manual_seed(3)).bfloat16()
    out = torch.empty((2 * length, heads * dim), dtype=BF16, device=DEV)
    ops.packed_attention_prompts(q.to(DEV), out, *planes, ints([0, length, 2 * length]), ints([length, length]), table.to(DEV), ints([0, 1]), 0, 2, 6, length,
                                 heads, heads, dim, page, None, 0.125)
    got = out.cpu().double().view(2, length, heads, dim)
    bad = got[0].isnan()
    assert bad[100:, 1, 32:].all() and bad.sum() == 60 * 32
    k, v = (case.context(1, rows) for rows in case.held())
    kept = torch.tensor([i for i in range(length) if i // page not in (2, 5)])
    for i in (31, 40, 79, 90, 159):
        mine = kept[kept <= i]
        want, weighted, sizes = attention(q[length + i:length + i + 1].double().view(1, heads, dim), k[mine], v[mine], torch.tensor([len(mine) - 1]), 0.125)
        assert ((got[1, i:i + 1] - want).abs() <= bound_of(want, weighted, sizes, 0.125, BF16, 2.0 ** -10, dim, 2.0 ** -11)).all()


@pytest.mark.parametrize("shares", [1, 2, 4, 8])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window,softcap,with_sink", [(None, None, False), (150, None, True), (None, 3.0, True)])
def test_shares_of_the_keys_of_a_block(shares, dim, window, softcap, with_sink):
    """More shares than tiles of keys, shares whose keys a query tile does not see, rows of fewer than a block."""
    ops, heads, kv_heads, page = ops_for(BF16), 4, 2, 16
    news, lengths = [300, 5, 129, 1, 256], [1500, 700, 129, 1, 900]
    case = PackedCase(lengths, kv_heads, dim, page, BF16, seed=9)
    _, planes = on_device(case)
    starts = [0]
    for new in news:
        starts.append(starts[-1] + new)
    g = torch.Generator().manual_seed(dim)
    q = torch.randn(starts[-1], heads * dim, generator=g).bfloat16()
    sink = torch.randn(heads, generator=g) if with_sink else None
    out = torch.full((starts[-1] + 3, heads * dim), 7.0, dtype=BF16, device=DEV)
    ops.packed_attention_prompts(q.to(DEV), out[:-3], *planes, ints(starts), ints(lengths), case.table.to(DEV), ints(range(5)), 0, 5, 5 + 1 + 3 + 1 + 4, 1500,
                                 heads, kv_heads, dim, page, window, 0.125, softcap=softcap, sink=None if sink is None else sink.to(DEV), shares=shares)
    assert (out[-3:] == 7.0).all()
    for i in range(5):
        k, v = (case.context(i, held_rows) for held_rows in case.held())
        mine = slice(starts[i], starts[i + 1])
        positions = torch.arange(lengths[i] - news[i], lengths[i])
        want, weighted, sizes = attention(q[mine].double().view(-1, heads, dim), k, v, positions, 0.125, window=window, softcap=softcap, sink=sink)
        got = out[mine].cpu().double().view(-1, heads, dim)
        assert ((got - want).abs() <= bound_of(want, weighted, sizes, 0.125, BF16, 2.0 ** -10, dim, 2.0 ** -11)).all()


def test_shares_and_rows_that_are_formed_again():
    """A NaN in one share's keys is met by all of them."""
    ops, heads, dim, page, length = ops_for(BF16), 2, 64, 16, 1100
    case = PackedCase([length], heads, dim, page, BF16, seed=6)
    case.v[900, 1, 40] = float("nan")                                   # head 1, second group
    _, planes = on_device(case)
    q = torch.randn(300, heads * dim, generator=torch.Generator().manual_seed(3)).bfloat16().to(DEV)
    arguments = (ints([0, 300]), ints([length]), case.table.to(DEV), ints([0]), 0, 1, 5, length, heads, heads, dim, page, None, 0.125)
    once = ops.packed_attention_prompts(q, torch.empty_like(q), *planes, *arguments, shares=1)
    bad = once.view(300, heads, dim).isnan()
    assert bad[100:, 1, 32:].all() and bad.sum() == 200 * 32            # (queries from position 800 on)
    for shares in (2, 4, 8):
        shared = ops.packed_attention_prompts(q, torch.empty_like(q), *planes, *arguments, shares=shares)
        assert torch.equal(shared.isnan(), once.isnan())
        assert torch.equal(shared.view(300, heads, dim)[:, 1].nan_to_num(), once.view(300, heads, dim)[:, 1].nan_to_num())


def test_prompts_in_several_rounds():
    """Unpacked rows of some items at a time."""
    ops, heads, dim, page = ops_for(F32), 2, 64, 16
    lengths = [100, 30, 70, 129]
    case = PackedCase(lengths, heads, dim, page, F32, seed=2)
    _, planes = on_device(case)
    starts = [0, 100, 130, 200, 329]
    q = torch.randn(329, heads * dim, generator=torch.Generator().manual_seed(5))
    arguments = (ints(starts), ints(lengths), case.table.to(DEV), ints(range(4)), 0, 4, 2 + 1 + 2 + 3, 129, heads, heads, dim, page, None, 0.125)
    once = ops.packed_attention_prompts(q.to(DEV), torch.empty(329, 128, device=DEV), *planes, *arguments).clone()
    kept = ops.UNPACKED_BYTES
    ops.UNPACKED_BYTES = 1
    try:
        assert torch.equal(ops.packed_attention_prompts(q.to(DEV), torch.empty(329, 128, device=DEV), *planes, *arguments), once)
    finally:
        ops.UNPACKED_BYTES = kept


# ------------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_captured_step(dtype):
    """Rows written and attended to on a side stream, captured and replayed with other rows and lengths."""
    ops, heads, dim, page = ops_for(dtype), 4, 64, 16
    case = PackedCase([70, 200, 33], heads, dim, page, dtype, seed=12)
    pool = case.pool.to(DEV)
    planes = (pool[:, 0], pool[:, 1], pool.stride(0))
    token_row, positions, table = case.token_row.to(DEV), case.positions.to(DEV), case.table.to(DEV)
    k, v = case.k.flatten(1).to(DEV), case.v.flatten(1).to(DEV)
    q = torch.randn(3, heads * dim, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    out, at = torch.empty_like(q), ints([69, 199, 32])

    def step():
        ops.kv_append_packed(k, v, token_row, positions, table, *planes, heads, dim, page)
        ops.packed_attention_tokens(q, out, *planes, ints_row, at, table, heads, heads, dim, page, None, 0.125, 256)

    ints_row = ints([0, 1, 2])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        graph.capture_begin()
        step()
        graph.capture_end()
    side.synchronize()
    case.k, case.v = case.k.flip(0).contiguous(), case.v.flip(0).contiguous()
    k.copy_(case.k.flatten(1))
    v.copy_(case.v.flatten(1))
    at.copy_(ints([50, 120, 2]))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(pool.cpu(), case.filled())
    held_k, held_v = case.held()
    for i, position in enumerate((50, 120, 2)):
        want, weighted, sizes = attention(q[i:i + 1].cpu().double().view(1, heads, dim), case.context(i, held_k), case.context(i, held_v),
                                          torch.tensor([position]), 0.125)
        limit = bound_of(want, weighted, sizes, 0.125, dtype, 2.0 ** -11 if dtype == BF16 else 0.0, dim)
        assert ((out[i:i + 1].cpu().double().view(1, heads, dim) - want).abs() <= limit).all()
    del graph


def test_pages_that_are_missing_may_unpack_as_zeros():
    ops, heads, dim, page, length = ops_for(F32), 2, 64, 16, 160
    case = PackedCase([length], heads, dim, page, F32, seed=6)
    _, planes = on_device(case)
    table = case.table.clone()
    table[0, 2], table[0, 5] = -1, case.pages
    out = torch.full((3, 2, heads, 64, dim), 7.0, device=DEV)
    ops.kv_unpack(*planes, ints([length]), table.to(DEV), ints([0]), 0, 1, 192, out, heads, dim, page, fill=True)
    place = torch.arange(192)
    gone = (place // page == 2) | (place // page == 5)
    for plane, rows in enumerate(case.held()):
        flat = out[:, plane].transpose(1, 2).flatten(0, 1).cpu()
        want = torch.full((192, heads, dim), 7.0)
        want[:length] = case.context(0, rows)[:length].float()
        want[gone] = 0.0
        assert torch.equal(flat, want)


def test_prompts_in_float32_first_met_under_capture():
    """What a captured call needs is its own: an eager call on another stream, before and after the graph is replayed, does not read it."""
    ops, heads, dim, page, length = ops_for(F32), 2, 64, 16, 150
    case = PackedCase([length], heads, dim, page, F32, seed=4)
    _, planes = on_device(case)
    q = torch.randn(length, heads * dim, generator=torch.Generator().manual_seed(5)).to(DEV)
    arguments = (ints([0, length]), ints([length]), case.table.to(DEV), ints([0]), 0, 1, 3, length, heads, heads, dim, page, None, 0.125)
    run = lambda into: ops.packed_attention_prompts(q, into, *planes, *arguments)
    first, second, third = (torch.zeros_like(q) for _ in range(3))
    ops._tc_library(), ops._packed_library(), ops.status_flag(q.device)
    torch.cuda.synchronize()
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        graph.capture_begin()
        run(first)
        graph.capture_end()
    assert ops._ramps == {}
    with torch.cuda.stream(other):
        run(second)
    run(third)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(first, second) and torch.equal(first, third) and first.abs().sum() > 0
    del graph


def test_refusals_on_the_device():
    from pagedserve_b200.kernels.ops import KernelError

    ops, case = ops_for(BF16), PackedCase([20], 2, 64, 16, BF16)
    pool = case.pool.to(DEV)
    row, at, table = case.token_row.to(DEV), case.positions.to(DEV), case.table.to(DEV)
    k = case.k.flatten(1).to(DEV)
    planes = (pool[:, 0], pool[:, 1], pool.stride(0))
    good = dict(k_src=k, v_src=k, token_row=row, positions=at, block_table=table, k_pool=planes[0], v_pool=planes[1], page_stride=planes[2], n_kv_heads=2,
                head_dim=64, page_size=16)
    for change in (dict(k_src=None, v_src=None), dict(k_src=k.float()), dict(k_src=k[:, :100]), dict(k_src=k.t()), dict(token_row=row.long()),
                   dict(positions=at[:5]), dict(block_table=table.long()), dict(block_table=table[0]), dict(k_pool=planes[0].float()),
                   dict(page_stride=planes[2] + 16), dict(n_kv_heads=1), dict(head_dim=32), dict(page_size=8), dict(page_size=12), dict(head_dim=0),
                   dict(head_dim=257), dict(v_pool=planes[1][:1]), dict(k_src=k.cpu()), dict(positions=at.cpu()), dict(block_table=table.cpu())):
        with pytest.raises(KernelError):
            ops.kv_append_packed(**{**good, **change})
    q, out = torch.zeros(3, 256, dtype=BF16, device=DEV), torch.zeros(3, 256, dtype=BF16, device=DEV)
    tokens = dict(q=q, out=out, k_pool=planes[0], v_pool=planes[1], page_stride=planes[2], token_row=row, positions=at, block_table=table, n_heads=4,
                  n_kv_heads=2, head_dim=64, page_size=16, window=None, scale=0.1, max_kv_len=20)
    for change in (dict(n_heads=3), dict(q=q.float()), dict(out=out.half()), dict(out=out[:2]), dict(out=out[:, ::2]), dict(sink=torch.zeros(3, device=DEV)),
                   dict(sink=torch.zeros(4)), dict(softcap=-1.0), dict(softcap=0.0), dict(scale=-0.1), dict(scale=float("nan")), dict(token_row=row[:2]), dict(n_kv_heads=0)):
        with pytest.raises(KernelError):
            ops.packed_attention_tokens(**{**tokens, **change})
    prompts = dict(q=q, out=out, k_pool=planes[0], v_pool=planes[1], page_stride=planes[2], q_start=ints([0, 3]), kv_len=ints([20]), block_table=table,
                   item_row=ints([0]), first_item=0, n_items=1, max_blocks=1, max_kv_len=20, n_heads=4, n_kv_heads=2, head_dim=64, page_size=16,
                   window=None, scale=0.1)
    for change in (dict(n_items=2), dict(first_item=1), dict(first_item=-1), dict(kv_len=ints([20]).long()), dict(q_start=ints([0]))):
        with pytest.raises(KernelError):
            ops.packed_attention_prompts(**{**prompts, **change})
    assert (out == 0).all()
