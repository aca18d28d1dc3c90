"""The operators of a cache held in 4 bits and of log probabilities, as cases that can be timed and checked.

A cache held in 4 bits: what a step writes is rounded and packed (``store``), single tokens (``tokens``) and portions of prompts
(``prompts``) attend to it.  Log probabilities of given tokens, with the entropy of the distribution and its largest
members: from logits that a step returned (``logits``), and from the rows in front of the head, whose logits nobody
needs (``head``).

A cached row of one key/value head is cut into groups of 32 numbers.  A group keeps ``low``, its minimum rounded down to
bfloat16, ``step``, (maximum - low) / 15 rounded up to bfloat16, and 16 codes of 4 bits a word of two: code = (x - low) / step
rounded to the nearest whole number (ties to even), and it reads as low + code * step.  A page of a head holds the codes of its
rows, then a 32-bit word a group (step in the lower half, low in the upper one), rounded up to 16 bytes.  The part ``t``
(numbers 8t to 8t + 7) of group ``j`` of ``n`` is word t * n + j of its row; the lower four codes of a word are the even numbers, the
upper four the odd ones.

``exact`` states the operators in 64 bits with code of its own.
"""

import math
import random

import numpy as np
import torch

own = False                    # whether ``run`` calls the framework's operators or computes their plain forms

DEVICE = "cuda:0"
GROUP = 32
VOCAB = 50257                  # GPT-2's
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
ORDER = (0, 2, 4, 6, 1, 3, 5, 7)          # which number of a part each code of its word is


# ------------------------------------------------------------------------------------------------ the cases
def _attend(name, kind, dtype, requests, longest, heads, kv_heads, dim, new=1, page=16, window=0, softcap=0.0, sink=False):
    return dict(name=name, kind=kind, dtype=dtype, requests=requests, longest=longest, new=new, heads=heads, kv_heads=kv_heads,
                dim=dim, page=page, window=window, softcap=softcap, sink=sink)


def listed():
    return [
        # a decode step of a few users, GPT-2 124M: one row a request is written, the smallest call
        _attend("store-8-bf16", "store", "bfloat16", 8, 100, 12, 12, 64),
        # long prompts of the 1.5B model in the engine's default precision, every row of them written
        _attend("store-prompts-float32", "store", "float32", 5, 1023, 25, 25, 64, new=1023),
        # one user, a short chat, GPT-2 124M: latency
        _attend("tokens-1-bf16", "tokens", "bfloat16", 1, 129, 12, 12, 64),
        # a few users with a full context: the batch of the engine's headline benchmark
        _attend("tokens-8-bf16", "tokens", "bfloat16", 8, 1024, 12, 12, 64),
        # a busy server with long contexts, heads of 128 in groups of four
        _attend("tokens-64-bf16", "tokens", "bfloat16", 64, 4099, 32, 8, 128),
        # windowed attention with capped scores and sinks in the default precision
        _attend("tokens-5-float32", "tokens", "float32", 5, 777, 16, 16, 64, window=512, softcap=50.0, sink=True),
        # two whole prompts in one step, GPT-2 124M
        _attend("prompts-2048-bf16", "prompts", "bfloat16", 2, 1024, 12, 12, 64, new=1024),
        # portions of long documents behind a cached context, heads of 128 in groups of four
        _attend("prompts-portions-bf16", "prompts", "bfloat16", 3, 8192, 16, 4, 128, new=683),
        # the logits of a decode step of 8 users and their most likely tokens
        dict(name="logits-8", kind="logits", rows=8, vocab=VOCAB, top=5),
        # scoring: the logits of a long step
        dict(name="logits-2047", kind="logits", rows=2047, vocab=VOCAB, top=20),
        # scoring a text of two prompts with the head of GPT-2 124M
        dict(name="head-2047-bf16", kind="head", dtype="bfloat16", rows=2047, width=768, vocab=VOCAB, top=5),
        # a short text in the default precision
        dict(name="head-33-float32", kind="head", dtype="float32", rows=33, width=768, vocab=VOCAB, top=1),
    ]


def _spread(rng, low, high):
    """A whole number, even over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """Another case of the same ranges."""
    kind = rng.choice(("store", "tokens", "tokens", "tokens", "prompts", "prompts", "logits", "head", "head"))
    dtype = rng.choice(("bfloat16", "bfloat16", "float32"))
    if kind == "logits":
        return dict(kind=kind, rows=_spread(rng, 1, 2000), vocab=rng.choice((VOCAB, 32000, _spread(rng, 500, 50000))), top=rng.choice((0, 1, 5, 20)))
    if kind == "head":
        width = rng.choice((768, 1024, 1600))
        return dict(kind=kind, dtype=dtype, rows=_spread(rng, 1, (2000 if dtype == "bfloat16" else 300) * 768 // width), width=width,
                    vocab=rng.choice((VOCAB, 32000, _spread(rng, 500, 50000))), top=rng.choice((0, 1, 5, 20)))
    heads, kv_heads, dim = rng.choice(((12, 12, 64), (25, 25, 64), (16, 16, 128), (32, 8, 128), (16, 2, 64), (8, 8, 80), (6, 3, 96)))
    page = rng.choice((16, 16, 16, 8, 32, 64))
    extras = dict(window=rng.choice((0, 0, 256, 1000)), softcap=rng.choice((0.0, 0.0, 50.0)), sink=rng.choice((False, False, True)))
    if kind == "tokens":
        requests = _spread(rng, 1, 64)
        return dict(kind=kind, dtype=dtype, requests=requests, longest=_spread(rng, 1, min(32768, 65536 // requests)), new=1, heads=heads,
                    kv_heads=kv_heads, dim=dim, page=page, **extras)
    requests = _spread(rng, 1, 8)
    new = _spread(rng, 16, (2048 if dtype == "bfloat16" else 1024) // requests)
    longest = new + rng.choice((0, _spread(rng, 1, 3000 // requests)))
    if kind == "store":
        extras = dict(window=0, softcap=0.0, sink=False)
        new = rng.choice((1, new))
    return dict(kind=kind, dtype=dtype, requests=requests, longest=max(longest, new), new=new, heads=heads, kv_heads=kv_heads, dim=dim, page=page, **extras)


# ------------------------------------------------------------------------------------------------ sizes and inputs
def _lengths(case):
    """Cached tokens of each request after the step and how many of them the step brings: the longest request, and others with
    between a third and all of both."""
    rng = random.Random(case["longest"] * 1009 + case["requests"])
    longest, new = case["longest"], case["new"]
    lengths, brought = [longest], [new]
    for _ in range(case["requests"] - 1):
        share = rng.uniform(0.33, 1.0)
        brought.append(max(1, int(new * share)))
        lengths.append(max(brought[-1], int(longest * share)))
    return lengths, brought


def _slab(page, dim):
    """Bytes of one head's rows in a page."""
    groups = -(-dim // GROUP)
    return -(-page * groups * 20 // 16) * 16


def _generator(seed, salt):
    return torch.Generator(device=DEVICE).manual_seed(int(seed) * 16 + salt)


def _normal(g, shape, std=1.0, mean=0.0):
    return torch.empty(shape, dtype=torch.float32, device=DEVICE).normal_(mean, std, generator=g)


def _round_down(x):
    """float32 to the bfloat16 number at or below it (as float32)."""
    near = x.bfloat16().float()
    below = (near.view(torch.int32) + torch.where(near > 0, -65536, 65536).int()).view(torch.float32)
    below = torch.where(near == 0, torch.full_like(x, -2.0 ** -133), below)
    return torch.where(near > x, below, near)


def _pack(x):
    """Rows [..., dim] float32 -> codes as bytes [..., 16 * groups] and words [..., groups] (int32)."""
    dim = x.shape[-1]
    groups = -(-dim // GROUP)
    lead = x.shape[:-1]
    if dim % GROUP:                                        # numbers that are not there: as the last group's first one
        first = dim // GROUP * GROUP
        x = torch.cat([x, x[..., first:first + 1].expand(*lead, groups * GROUP - dim)], dim=-1)
    x = x.reshape(*lead, groups, GROUP)
    low = _round_down(x.amin(-1))
    step = -_round_down(-((x.amax(-1) - low) / torch.full_like(low, 15.0)))
    bad = ~(torch.isfinite(low) & torch.isfinite(step))
    low, step = (torch.where(bad, torch.full_like(v, float("nan")), v) for v in (low, step))
    code = torch.round((x - low[..., None]) / torch.where(step == 0, torch.ones_like(step), step)[..., None])
    code = torch.where(bad[..., None], torch.zeros_like(code), code).clamp(0, 15).to(torch.uint8)
    code = code.reshape(*lead, groups * GROUP)
    code[..., dim:] = 0
    code = code.reshape(*lead, groups, 4, 8)[..., list(ORDER)].transpose(-3, -2)       # [..., part, group, code of the word]
    data = (code[..., 0::2] | (code[..., 1::2] << 4)).reshape(*lead, groups * 16)
    halves = torch.stack([step, low], dim=-1).bfloat16().contiguous()
    return data, halves.view(torch.int32).squeeze(-1)


def _unpack(data, words, dim):
    """The inverse: [..., 16 * groups] bytes and [..., groups] words -> float32 [..., dim]."""
    groups = words.shape[-1]
    lead = words.shape[:-1]
    code = torch.stack([data & 15, data >> 4], dim=-1).reshape(*lead, 4, groups, 8)
    back = [ORDER.index(i) for i in range(8)]
    code = code[..., back].transpose(-3, -2).reshape(*lead, groups, GROUP).float()
    halves = words.contiguous().view(torch.bfloat16).reshape(*lead, groups, 2).float()
    return (halves[..., 1:] + code * halves[..., :1]).reshape(*lead, groups * GROUP)[..., :dim]


def _page_parts(pool, page, dim):
    """Views of a plane [pages, kv heads, slab]: codes [pages, kv heads, page, 16 * groups] and words [pages, kv heads, page, groups]."""
    groups = -(-dim // GROUP)
    codes = pool[..., :page * groups * 16].unflatten(-1, (page, groups * 16))
    words = pool[..., page * groups * 16:page * groups * 20].unflatten(-1, (page, groups * 4))
    return codes, words


def _rows(pool, pages, page, dim):
    """The rows of the listed pages [...] in order: float32 [..., page, kv heads, dim]."""
    codes, words = _page_parts(pool, page, dim)
    return _unpack(codes[pages], words[pages].contiguous().view(torch.int32), dim).transpose(-3, -2)


def _filled_pool(g, pages, case, keys):
    """A plane of rows as a model leaves them: keys with a bias for each channel, which they have in earnest, values without."""
    page, dim, kv_heads = case["page"], case["dim"], case["kv_heads"]
    pool = torch.zeros((pages, kv_heads, _slab(page, dim)), dtype=torch.uint8, device=DEVICE)
    codes, words = _page_parts(pool, page, dim)
    bias = _normal(g, (kv_heads, 1, dim)) if keys else 0.0
    at_once = max(1, (1 << 25) // (kv_heads * page * dim))
    for start in range(0, pages, at_once):
        end = min(pages, start + at_once)
        data, word = _pack(_normal(g, (end - start, kv_heads, page, dim)) + bias)
        codes[start:end] = data
        words[start:end] = word.contiguous().view(torch.uint8).reshape(words[start:end].shape)
    return pool


def prepare(case, seed):
    state = dict(case)
    if case["kind"] == "logits":
        g = _generator(seed, 1)
        # a few tokens stand out, as they do behind a trained head
        logits = _normal(g, (case["rows"], case["vocab"]), 2.0)
        likely = torch.randint(case["vocab"], (case["rows"], 8), generator=g, device=DEVICE)
        logits.scatter_add_(1, likely, _normal(g, likely.shape, 3.0, 6.0))
        state["logits"] = logits
        state["targets"] = likely[:, 0].int()
    elif case["kind"] == "head":
        g = _generator(seed, 2)
        dtype = DTYPES[case["dtype"]]
        # On a grid on which float32 sums are exact in any order, so that which tokens are the most likely is a fact: hidden numbers
        # are multiples of 1/8, the table's of 1/512.
        table = (_normal(g, (case["vocab"], case["width"]), 0.04) * 512).round() / 512
        likely = torch.randint(case["vocab"], (case["rows"],), generator=g, device=DEVICE)
        hidden = _normal(g, (case["rows"], case["width"])) + table[likely] * (6.0 * 768 / case["width"])
        state["hidden"] = ((hidden * 8).round() / 8).clamp(-6, 6).to(dtype)
        state["table"] = table.clamp(-0.49, 0.49).to(dtype)
        state["targets"] = likely.int()
    else:
        _prepare_cache(case, seed, state)
    if own:
        from pagedserve_b200.kernels.ops import Ops

        state["ops"] = Ops(DTYPES[case.get("dtype", "float32")])
    return state


def _prepare_cache(case, seed, state):
    g = _generator(seed, 3)
    lengths, brought = _lengths(case)
    page, kv_heads, dim, heads = case["page"], case["kv_heads"], case["dim"], case["heads"]
    dtype = DTYPES[case["dtype"]]
    counts = [-(-length // page) for length in lengths]
    total = sum(counts)
    shuffled = np.random.default_rng(int(seed)).permutation(total)
    table = np.full((len(lengths), max(counts)), -1, dtype=np.int32)
    taken = 0
    for row, count in enumerate(counts):
        table[row, :count] = shuffled[taken:taken + count]
        taken += count
    device = lambda values: torch.as_tensor(np.asarray(values), dtype=torch.int32, device=DEVICE)
    starts = np.concatenate([[0], np.cumsum(brought)])
    state.update(lengths=lengths, brought=brought, tokens=int(starts[-1]), table=device(table),
                 token_row=device(np.repeat(np.arange(len(lengths)), brought)),
                 positions=device(np.concatenate([np.arange(length - new, length) for length, new in zip(lengths, brought)])),
                 q_start=device(starts), kv_len=device(lengths), item_row=device(np.arange(len(lengths))))
    pool = torch.empty((total, 2, kv_heads, _slab(page, dim)), dtype=torch.uint8, device=DEVICE)
    for plane in (0, 1):
        pool[:, plane] = _filled_pool(g, total, case, keys=plane == 0)
    state["k_pool"], state["v_pool"], state["page_stride"] = pool[:, 0], pool[:, 1], pool.stride(0)
    if case["kind"] == "store":
        # the projection's rows: queries, keys and values side by side
        width = (heads + 2 * kv_heads) * dim
        rows = _normal(g, (state["tokens"], width)).to(dtype)
        state["k"] = rows[:, heads * dim:(heads + kv_heads) * dim]
        state["v"] = rows[:, (heads + kv_heads) * dim:]
        span = max(counts) * page
        state["read"] = torch.zeros((len(lengths) * max(counts), 2, kv_heads, page, dim), dtype=dtype, device=DEVICE)
        state["span"] = span
    else:
        state["q"] = _normal(g, (state["tokens"], heads * dim)).to(dtype)
        state["out"] = torch.empty_like(state["q"])
        state["scale"] = dim ** -0.5
        state["sinks"] = _normal(g, (heads,)) if case["sink"] else None


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    ops, kind = state["ops"], state["kind"]
    if kind == "logits":
        return tuple(ops.token_logprobs(state["logits"], state["targets"], top=state["top"]))
    if kind == "head":
        return tuple(ops.head_logprobs(state["hidden"], state["table"], state["targets"], top=state["top"]))
    pools = (state["k_pool"], state["v_pool"], state["page_stride"])
    sizes = (state["kv_heads"], state["dim"], state["page"])
    if kind == "store":
        ops.kv_append_packed(state["k"], state["v"], state["token_row"], state["positions"], state["table"], *pools, *sizes)
        # what the cache then holds, as values, page by page
        ops.kv_unpack(*pools, state["kv_len"], state["table"], state["item_row"], 0, state["requests"], state["span"], state["read"], *sizes)
        return state["read"]
    extras = dict(softcap=state["softcap"] or None, sink=state["sinks"])
    if kind == "tokens":
        return ops.packed_attention_tokens(state["q"], state["out"], *pools, state["token_row"], state["positions"], state["table"], state["heads"],
                                           *sizes, state["window"] or None, state["scale"], max(state["lengths"]), **extras)
    blocks = sum(-(-new // 64) for new in state["brought"])
    return ops.packed_attention_prompts(state["q"], state["out"], *pools, state["q_start"], state["kv_len"], state["table"], state["item_row"],
                                        0, state["requests"], blocks, max(state["lengths"]), state["heads"], *sizes, state["window"] or None,
                                        state["scale"], **extras)


def _plain_logprobs(logits, targets, top):
    largest = logits.amax(1, keepdim=True)
    shifted = logits - largest
    weights = shifted.exp()
    total = weights.sum(1, keepdim=True)
    log_total = total.log()
    logprobs = shifted - log_total
    given = logprobs.gather(1, targets.long()[:, None])[:, 0]
    entropy = log_total[:, 0] - (weights * shifted).sum(1) / total[:, 0]
    # (of equal ones the lowest index comes first: a number's order and its index as one whole number)
    bits = (logits + 0.0).view(torch.int32)
    ordered = torch.where(bits < 0, bits ^ 0x7fffffff, bits).long()
    backwards = torch.arange(logits.shape[1] - 1, -1, -1, device=logits.device)
    order = logits.shape[1] - 1 - ((ordered << 32) + backwards).topk(top, dim=1)[0] % (1 << 32)
    return given, entropy, logprobs.gather(1, order), order.int()


def _run_plain(state):
    kind = state["kind"]
    if kind in ("logits", "head"):
        logits = state["logits"] if kind == "logits" else state["hidden"].float() @ state["table"].float().t()
        return _plain_logprobs(logits, state["targets"], state["top"])
    if kind == "store":
        return _plain_store(state)
    return (_plain_tokens if kind == "tokens" else _plain_prompts)(state)


def _plain_store(state):
    page, kv_heads, dim = state["page"], state["kv_heads"], state["dim"]
    positions = state["positions"].long()
    pages = state["table"][state["token_row"].long(), positions // page].long()
    for rows, pool in ((state["k"], state["k_pool"]), (state["v"], state["v_pool"])):
        codes, words = _page_parts(pool, page, dim)
        data, word = _pack(rows.float().unflatten(1, (kv_heads, dim)))
        codes[pages, :, positions % page] = data
        words[pages, :, positions % page] = word.contiguous().view(torch.uint8).reshape(*word.shape[:-1], -1)
    read = state["read"].unflatten(0, state["table"].shape)                # [requests, pages, 2, kv heads, page, dim]
    place = torch.arange(state["span"], device=DEVICE).view(1, -1, 1, page, 1)
    inside = place < state["kv_len"].view(-1, 1, 1, 1, 1)
    for plane, pool in enumerate((state["k_pool"], state["v_pool"])):
        values = _rows(pool, state["table"].long().clamp(min=0), page, dim).transpose(2, 3).to(read.dtype)
        read[:, :, plane] = torch.where(inside, values, read[:, :, plane])
    return state["read"]


def _plain_weights(scores, key, position, state, sinks):
    """softmax over the last axis of the keys that a query at ``position`` sees."""
    if state["softcap"]:
        scores = state["softcap"] * torch.tanh(scores / state["softcap"])
    seen = key <= position
    if state["window"]:
        seen = seen & (key > position - state["window"])
    scores = torch.where(seen, scores, torch.full_like(scores, float("-inf")))
    largest = scores.amax(-1, keepdim=True)
    if sinks is not None:
        largest = torch.maximum(largest, sinks)
    weights = (scores - largest).exp()
    total = weights.sum(-1, keepdim=True)
    if sinks is not None:
        total = total + (sinks - largest).exp()
    return weights / total


def _plain_tokens(state):
    page, kv_heads, dim, heads = state["page"], state["kv_heads"], state["dim"], state["heads"]
    tables = state["table"][state["token_row"].long()].long().clamp(min=0)
    tokens, width = tables.shape
    group = heads // kv_heads
    q = state["q"].float().view(tokens, kv_heads, group, dim)
    key = torch.arange(width * page, device=DEVICE)
    sinks = state["sinks"].view(1, kv_heads, group, 1) if state["sinks"] is not None else None
    at_once = max(1, (1 << 29) // (width * page * kv_heads * dim))
    for start in range(0, tokens, at_once):
        end = min(tokens, start + at_once)
        k, v = (_rows(pool, tables[start:end], page, dim).flatten(1, 2) for pool in (state["k_pool"], state["v_pool"]))
        scores = torch.einsum("tgrd,tlgd->tgrl", q[start:end], k) * state["scale"]
        position = state["positions"][start:end].view(-1, 1, 1, 1)
        weights = _plain_weights(scores, key, position, state, sinks)
        # (rows behind a token's own hold what is in the pages: their weight is zero)
        state["out"][start:end] = torch.einsum("tgrl,tlgd->tgrd", weights, v).reshape(end - start, heads * dim).to(state["out"].dtype)
    return state["out"]


def _plain_prompts(state):
    page, kv_heads, dim, heads = state["page"], state["kv_heads"], state["dim"], state["heads"]
    group = heads // kv_heads
    first = 0
    for row, (length, new) in enumerate(zip(state["lengths"], state["brought"])):
        pages = state["table"][row, :-(-length // page)].long()
        k, v = (_rows(pool, pages, page, dim).flatten(0, 1)[:length] for pool in (state["k_pool"], state["v_pool"]))
        key = torch.arange(length, device=DEVICE)
        sinks = state["sinks"].view(kv_heads, group, 1, 1) if state["sinks"] is not None else None
        q = state["q"][first:first + new].float().view(new, kv_heads, group, dim)
        scores = torch.einsum("ngrd,lgd->grnl", q, k) * state["scale"]
        position = torch.arange(length - new, length, device=DEVICE)[:, None]
        weights = _plain_weights(scores, key, position, state, sinks)
        state["out"][first:first + new] = torch.einsum("grnl,lgd->ngrd", weights, v).reshape(new, heads * dim).to(state["out"].dtype)
        first += new
    return state["out"]


# ------------------------------------------------------------------------------------------------ what it cannot do without
def _visible(state_or_case, length, new):
    """Pairs of a query of the step and a key that it sees, and the keys that any of them sees."""
    window = state_or_case["window"]
    pairs = 0
    if not window:
        pairs = new * (length - new) + new * (new + 1) // 2
        return pairs, length
    first = length - new
    full = max(0, length - max(first, window))             # queries that see a whole window
    pairs = full * window
    rest = new - full
    pairs += rest * first + rest * (rest + 1) // 2
    return pairs, min(length, new + window - 1)


def work(case):
    if case["kind"] == "logits":
        count = case["rows"] * case["vocab"]
        return dict(bytes=4 * count + case["rows"] * (12 + 8 * case["top"]), flops=6 * count)
    if case["kind"] == "head":
        size = 2 if case["dtype"] == "bfloat16" else 4
        return dict(bytes=size * case["width"] * (case["vocab"] + case["rows"]) + case["rows"] * (12 + 8 * case["top"]),
                    flops=2 * case["rows"] * case["width"] * case["vocab"])
    lengths, brought = _lengths(case)
    size = 2 if case["dtype"] == "bfloat16" else 4
    packed = 2 * case["kv_heads"] * -(-case["dim"] // GROUP) * 20             # bytes of a token's rows
    plain = 2 * case["kv_heads"] * case["dim"] * size
    if case["kind"] == "store":
        return dict(bytes=sum(brought) * (plain + packed) + sum(lengths) * (packed + plain), flops=4 * sum(brought) * plain // size)
    pairs = keys = 0
    for length, new in zip(lengths, brought):
        more_pairs, more_keys = _visible(case, length, new)
        pairs, keys = pairs + more_pairs, keys + more_keys
    return dict(bytes=keys * packed + 2 * sum(brought) * case["heads"] * case["dim"] * size, flops=4 * case["heads"] * case["dim"] * pairs)


# ------------------------------------------------------------------------------------------------ the definition, in 64 bits
def _exact_halves(words):
    """The two bfloat16 numbers of a group's words, as float64: step and low."""
    bits = words.to(torch.int64) & 0xFFFFFFFF
    low = (bits >> 16) << 16
    step = (bits & 0xFFFF) << 16
    as_float = lambda value: torch.where(value >= 2 ** 31, value - 2 ** 32, value).to(torch.int32).view(torch.float32).double()
    return as_float(step), as_float(low)


def _exact_context(pool, table_row, length, case):
    """What the cache holds of one request: float64 [length, kv heads, dim], read number by number from the bytes."""
    page, dim, kv_heads = case["page"], case["dim"], case["kv_heads"]
    groups = (dim + GROUP - 1) // GROUP
    place = torch.arange(length, device=DEVICE)
    slabs = pool[table_row.long()[place // page]]                             # [length, kv heads, slab]
    number = torch.arange(dim, device=DEVICE)
    group, part, inner = number // 32, number % 32 // 8, number % 8
    nibble = inner // 2 + 4 * (inner % 2)
    at = (place % page)[:, None] * (groups * 16) + (part * groups + group)[None, :] * 4 + (nibble // 2)[None, :]
    byte = slabs.gather(2, at[:, None, :].expand(length, kv_heads, dim)).long()
    code = torch.where(nibble % 2 == 1, byte // 16, byte % 16).double()
    base = page * groups * 16 + (place % page)[:, None] * (groups * 4) + group[None, :] * 4
    word = torch.zeros((length, kv_heads, dim), dtype=torch.int64, device=DEVICE)
    for i in range(4):
        word += slabs.gather(2, (base + i)[:, None, :].expand(length, kv_heads, dim)).long() << (8 * i)
    step, low = _exact_halves(word)
    return low + code * step


def _exact_stored(x):
    """Rows [tokens, kv heads, dim] as the format holds them.  The format says where it rounds: differences and quotients to float32
    (in 64 bits first, which changes neither), low down and step up to bfloat16, codes to the nearest whole number."""
    x = x.double()
    out = torch.empty_like(x)
    to32 = lambda value: value.float().double()

    def towards(value, up):
        magnitude = value.abs().float().view(torch.int32)
        cut = magnitude & ~0xFFFF
        grows = (cut != magnitude) & ((value > 0) if up else (value < 0))
        return torch.sign(value) * (cut + grows.int() * 0x10000).view(torch.float32).double()

    for first in range(0, x.shape[-1], GROUP):
        part = x[..., first:first + GROUP]
        low = towards(part.min(-1, keepdim=True)[0], up=False)
        step = towards(to32(to32(part.max(-1, keepdim=True)[0] - low) / 15.0), up=True)
        code = torch.zeros_like(part)
        held = step > 0
        code = torch.where(held, to32(to32(part - low) / torch.where(held, step, 1.0)).round().clamp(0, 15), code)
        out[..., first:first + GROUP] = low + code * step
    return out


def _exact_cache(case, state):
    kind, kv_heads, dim, page, heads = (case[name] for name in ("kind", "kv_heads", "dim", "page", "heads"))
    if kind == "store":
        result = torch.zeros(state["read"].shape, dtype=torch.float64, device=DEVICE)
        pages_each = state["table"].shape[1]
        done = 0
        for row, (length, new) in enumerate(zip(state["lengths"], state["brought"])):
            for plane, (rows, pool) in enumerate(((state["k"], state["k_pool"]), (state["v"], state["v_pool"]))):
                held = _exact_context(pool, state["table"][row], length, case)
                held[length - new:] = _exact_stored(rows[done:done + new].reshape(new, kv_heads, dim))
                for p in range(-(-length // page)):
                    some = held[p * page:(p + 1) * page]
                    result[row * pages_each + p, plane, :, :some.shape[0]] = some.transpose(0, 1)
            done += new
        return result
    out = torch.empty(state["out"].shape, dtype=torch.float64, device=DEVICE)
    done, group = 0, heads // kv_heads
    for row, (length, new) in enumerate(zip(state["lengths"], state["brought"])):
        keys, values = (_exact_context(pool, state["table"][row], length, case) for pool in (state["k_pool"], state["v_pool"]))
        place = torch.arange(length, device=DEVICE)
        for start in range(0, new, 256):
            some = min(256, new - start)
            here = torch.arange(length - new + start, length - new + start + some, device=DEVICE)[:, None]
            hidden = place[None, :] > here
            if case["window"]:
                hidden |= here - place[None, :] >= case["window"]
            for h in range(heads):
                q = state["q"][done + start:done + start + some, h * dim:(h + 1) * dim].double()
                s = (q @ keys[:, h // group].t()) * state["scale"]
                if case["softcap"]:
                    s = case["softcap"] * torch.tanh(s / case["softcap"])
                s = s.masked_fill(hidden, float("-inf"))
                if state["sinks"] is not None:
                    s = torch.cat([s, state["sinks"][h].double().expand(some, 1)], dim=1)
                p = torch.softmax(s, dim=1)[:, :length]
                out[done + start:done + start + some, h * dim:(h + 1) * dim] = p @ values[:, h // group]
        done += new
    return out


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] not in ("logits", "head"):
        return _exact_cache(case, state)
    given, entropy, best, ids = [], [], [], []
    for start in range(0, case["rows"], 256):
        end = min(case["rows"], start + 256)
        if case["kind"] == "logits":
            x = state["logits"][start:end].double()
        else:
            x = torch.matmul(state["hidden"][start:end].double(), state["table"].double().transpose(0, 1))
        log = torch.log_softmax(x, dim=1)
        given.append(log[torch.arange(end - start, device=DEVICE), state["targets"][start:end].long()])
        entropy.append(torch.special.entr(log.exp()).sum(1))
        index = torch.argsort(-x, dim=1, stable=True)[:, :case["top"]]
        best.append(torch.take_along_dim(log, index, dim=1))
        ids.append(index.int())
    return tuple(torch.cat(column) for column in (given, entropy, best, ids))
