"""A cache held in 4 bits and log probabilities, plainly: the format number by number, attention and softmax in 64 bits."""

import numpy as np
import torch

GROUP = 32


def slab_bytes(page, dim):
    return -(-page * -(-dim // GROUP) * 20 // 16) * 16


def _bf16(x, up):
    """float32 to the bfloat16 numbers at or above (``up``) or below them."""
    bits = x.view(np.uint32)
    cut = bits & np.uint32(0xFFFF0000)
    return (cut + np.where((bits != cut) & ((x > 0) == up), np.uint32(0x10000), np.uint32(0))).view(np.float32)


def pack_groups(x):
    """float32 [rows, up to 32] -> steps and lows [rows], codes [rows, up to 32]."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        low = _bf16(x.min(1), up=False)
        step = _bf16((x.max(1) - low) / np.float32(15), up=True)
        good = np.isfinite(x).all(1) & np.isfinite(low) & np.isfinite(step)
        codes = np.clip(np.rint((x - low[:, None]) / step[:, None]), 0, 15)
    codes = np.where((good & (step > 0))[:, None], codes, 0).astype(np.uint32)
    nan = np.float32(np.nan)
    return np.where(good, step, nan), np.where(good, low, nan), codes


def held(rows):
    """Rows of one head [..., dim] as the cache holds them: float32 numbers low + code * step."""
    rows = np.asarray(rows, dtype=np.float32)
    flat = rows.reshape(-1, rows.shape[-1])
    out = np.empty_like(flat)
    for first in range(0, flat.shape[1], GROUP):
        step, low, codes = pack_groups(flat[:, first:first + GROUP])
        out[:, first:first + GROUP] = low.astype(np.float64)[:, None] + codes * step.astype(np.float64)[:, None]
    return out.reshape(rows.shape)


def packed_rows(rows):
    """Rows of one head [n, dim] -> the words of their codes [n, 4 * groups] and of their scales [n, groups]."""
    count, dim = rows.shape
    groups = -(-dim // GROUP)
    words, scales = np.zeros((count, groups * 4), dtype=np.uint32), np.zeros((count, groups), dtype=np.uint32)
    half = lambda v: np.where(np.isfinite(v), v.astype(np.float32).view(np.uint32) >> 16, 0x7FFF).astype(np.uint32)
    for j in range(groups):
        step, low, codes = pack_groups(rows[:, j * GROUP:(j + 1) * GROUP])
        for i in range(codes.shape[1]):
            part, inner = i // 8, i % 8
            words[:, part * groups + j] |= codes[:, i] << np.uint32(4 * (inner // 2 + 4 * (inner % 2)))
        scales[:, j] = half(step) | half(low) << np.uint32(16)
    return words, scales


class PackedCase:
    """Requests with cached rows in shuffled pages of a pool that starts as a pattern of bytes, on the CPU."""

    def __init__(self, lengths, kv_heads, dim, page, dtype, seed=0, spare=3, width=0, mean=1.0, std=1.0):
        g = torch.Generator().manual_seed(seed)
        self.lengths, self.kv_heads, self.dim, self.page = lengths, kv_heads, dim, page
        counts = [-(-length // page) for length in lengths]
        self.pages = sum(counts) + spare
        order = torch.randperm(self.pages, generator=g)[:sum(counts)].int()
        self.table = torch.full((len(lengths), max(max(counts), 1) + width), -1, dtype=torch.int32)
        done = 0
        for row, count in enumerate(counts):
            self.table[row, :count] = order[done:done + count]
            done += count
        total = sum(lengths)
        self.k = (torch.randn(total, kv_heads, dim, generator=g) * std + mean * torch.randn(1, kv_heads, dim, generator=g)).to(dtype)
        self.v = (torch.randn(total, kv_heads, dim, generator=g) * std).to(dtype)
        self.slab = slab_bytes(page, dim)
        self.token_row = torch.repeat_interleave(torch.arange(len(lengths)), torch.tensor(lengths)).int()
        self.positions = torch.cat([torch.arange(length) for length in lengths]).int()
        self.pool = torch.full((self.pages, 2, kv_heads, self.slab), 0xA5, dtype=torch.uint8)

    def filled(self):
        """The pool once every row has been written."""
        pool = self.pool.clone().numpy()
        page, groups = self.page, -(-self.dim // GROUP)
        place = self.positions.numpy()
        at = self.table.numpy()[self.token_row.numpy(), place // page]
        for plane, rows in enumerate((self.k, self.v)):
            for head in range(self.kv_heads):
                slabs = pool[:, plane, head]
                words = slabs[:, :page * groups * 16].copy().view(np.uint32).reshape(len(pool), page, groups * 4)
                scales = slabs[:, page * groups * 16:page * groups * 20].copy().view(np.uint32).reshape(len(pool), page, groups)
                words[at, place % page], scales[at, place % page] = packed_rows(rows[:, head].float().numpy())
                slabs[:, :page * groups * 16] = words.reshape(len(pool), -1).view(np.uint8)
                slabs[:, page * groups * 16:page * groups * 20] = scales.reshape(len(pool), -1).view(np.uint8)
        return torch.from_numpy(pool)

    def held(self):
        """Keys and values as the cache holds them, [tokens, kv heads, dim]."""
        return tuple(torch.from_numpy(held(rows.float().numpy())) for rows in (self.k, self.v))

    def context(self, request, rows):
        first = sum(self.lengths[:request])
        return rows[first:first + self.lengths[request]].double()


def attention(q, k, v, positions, scale, window=None, softcap=None, sink=None):
    """q [n, heads, dim], k / v [length, kv heads, dim], float64 -> results [n, heads, dim], and for bounds the weighted sizes of the values
    [n, heads, dim] and the sums of |q| |k| [n, heads].  ``window``: > 0 the last keys, < 0 chunks of -window."""
    heads, length = q.shape[1], k.shape[0]
    k, v = (x.repeat_interleave(heads // k.shape[1], 1) for x in (k, v))
    at, key = positions.long()[:, None], torch.arange(length)[None]
    seen = key <= at
    if window:
        seen = seen & ((at - key < window) if window > 0 else (at // -window == key // -window))
    s = torch.einsum("ihd,jhd->hij", q, k) * scale
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    s = s.masked_fill(~seen, float("-inf"))
    if sink is not None:
        s = torch.cat([s, sink.double()[:, None, None].expand(heads, len(positions), 1)], -1)
    top = s.amax(-1, keepdim=True)
    w = torch.exp(s - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    total = w.sum(-1, keepdim=True)
    w = (w / torch.where(total == 0, torch.ones_like(total), total))[..., :length]
    sizes = torch.einsum("ihd,jhd->hij", q.abs(), k.abs()).masked_fill(~seen, 0).amax(-1).T if length else torch.zeros(len(positions), heads)
    return torch.einsum("hij,jhd->ihd", w, v), torch.einsum("hij,jhd->ihd", w, v.abs()), sizes


def logprobs(logits, targets, top):
    """float64 rows -> log probabilities of the targets (-1: 0), entropies, the largest with their indices."""
    largest = logits.amax(1, keepdim=True)
    log = logits - largest - torch.log(torch.exp(logits - largest).sum(1, keepdim=True))
    given = torch.stack([log[r, y] if y >= 0 else log.new_zeros(()) for r, y in enumerate(targets.tolist())])
    p = torch.exp(log)
    entropy = -torch.where(p > 0, p * log, torch.zeros_like(p)).sum(1)
    order = torch.sort(logits, dim=1, descending=True, stable=True)[1][:, :top]
    return given, entropy, torch.gather(log, 1, order), order.int()
