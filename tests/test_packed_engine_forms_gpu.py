"""What the engine's own steps hand to the kernels over a cache of 4 bits, against 64-bit attention over the bytes of its pool; scores read inside the head's product."""

import dataclasses

import numpy as np
import pytest
import torch

from plain_packed import attention, logprobs
from test_packed_engine_gpu import engine_for
from test_packed_sizes_gpu import agrees, limit_of

pytestmark = pytest.mark.gpu
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def numbers_of(plane, page, dim):
    """A plane of a pool, bytes [pages, kv heads, slab] -> what its rows hold, float64 [pages, page, kv heads, dim]."""
    pages, heads, _ = plane.shape
    groups = -(-dim // 32)
    raw = plane.cpu().contiguous().numpy()
    words = raw[..., :page * groups * 16].copy().view(np.uint32).reshape(pages, heads, page, 4, groups)
    scales = raw[..., page * groups * 16:page * groups * 20].copy().view(np.uint32).reshape(pages, heads, page, groups)
    half = lambda bits: (bits.astype(np.uint32) << np.uint32(16)).view(np.float32).astype(np.float64)
    step, low = half(scales & np.uint32(0xFFFF)), half(scales >> np.uint32(16))
    out = np.empty((pages, page, heads, groups * 32))
    for j in range(groups):
        for part in range(4):
            for i in range(8):
                code = words[:, :, :, part, j] >> np.uint32(4 * (i // 2 + 4 * (i % 2))) & np.uint32(15)
                out[..., 32 * j + 8 * part + i] = (low[..., j] + code * step[..., j]).transpose(0, 2, 1)
    return torch.from_numpy(out[..., :dim].copy())


class Watched:
    """An engine whose attention over packed pages is noted: queries, results, and the pool as it was then."""

    def __init__(self, engine):
        self.engine, self.calls, self.plain = engine, [], engine.ops._packed_attention
        engine.ops._packed_attention = self

    def __call__(self, q, k, v, out, ctx, layer, heads, kv_heads, dim, window, scale, write_cache, softcap, sink, mix):
        before = out.clone() if not torch.cuda.is_current_stream_capturing() else None
        result = self.plain(q, k, v, out, ctx, layer, heads, kv_heads, dim, window, scale, write_cache, softcap, sink, mix)
        if before is not None:
            copy = lambda x: x.detach().clone() if isinstance(x, torch.Tensor) else x
            self.calls.append(dict(q=copy(q), out=copy(out), k=copy(layer.k_pool), v=copy(layer.v_pool), table=copy(layer.block_table), slots=copy(ctx.token_slot),
                                   positions=copy(ctx.positions), tokens=ctx.num_tokens, page=layer.page_size, sizes=(heads, kv_heads, dim),
                                   mask=(window, softcap, copy(sink)), scale=scale, long=ctx.num_items - ctx.num_short_items))
        return result

    def check(self, dtype):
        """Every noted token of a request; the number of them that stood in a prompt portion's step."""
        scratch, seen = self.engine.cache.scratch_slot, 0
        for call in self.calls:
            heads, kv_heads, dim = call["sizes"]
            window, softcap, sink = call["mask"]
            k, v = (numbers_of(call[name], call["page"], dim) for name in ("k", "v"))
            slots, positions, table = (call[name].cpu().long() for name in ("slots", "positions", "table"))
            for slot in sorted(set(slots[:call["tokens"]].tolist()) - {scratch}):
                mine = (slots[:call["tokens"]] == slot).nonzero()[:, 0]
                at = positions[mine]
                pages = table[slot][:int(at.max()) // call["page"] + 1]
                keys, values = (x[pages.clamp(min=0)].flatten(0, 1)[:int(at.max()) + 1] for x in (k, v))
                gone = (pages < 0).repeat_interleave(call["page"])[:len(keys)]
                keys[gone] = values[gone] = 0.0                            # (given back: behind the window)
                q = call["q"][mine.to(call["q"].device)].cpu().double().view(-1, heads, dim)
                got = call["out"][mine.to(call["out"].device)].cpu().double().view(-1, heads, dim)
                found = attention(q, keys, values, at, call["scale"], window, softcap, None if sink is None else sink.cpu())
                agrees(got, found, limit_of(found, call["scale"], call["out"].dtype if dtype == torch.bfloat16 else dtype, dim)
                       + (limit_of(found, call["scale"], dtype, dim) if call["out"].dtype != dtype else 0))
                seen += len(mine) if call["long"] else 0
        self.calls.clear()
        return seen


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("name", ["tiny-b", "zositar-tiny", "tefopel-tiny"])
def test_steps_against_the_bytes_of_the_pool(name, dtype):
    """Prompts, portions, short portions and single tokens of several requests in one step, padded as the engine pads them."""
    engine = engine_for(name, dtype, "int4", num_blocks=128, max_num_seqs=6)
    watched, vocab = Watched(engine), engine.vocab_size
    text = lambda start, count: [(7 * i + 3 * start + 1) % vocab for i in range(start, start + count)]
    portions = 0
    for entries in ([("a", text(0, 150), [149])], [("a", text(150, 1), [0]), ("b", text(5, 70), [69]), ("c", text(9, 17), [])],
                    [("a", text(151, 1), [0]), ("b", text(75, 1), [0]), ("c", text(26, 100), [99]), ("d", text(2, 5), [4])],
                    [("a", text(152, 40), [39]), ("b", text(76, 33), [32]), ("c", text(126, 1), [0]), ("d", text(7, 64), [63]), ("e", text(0, 16), [0, 15])],
                    [(who, text(200, 1), [0]) for who in "abcde"]):
        engine.step(entries)
        portions += watched.check(DTYPES[dtype])
    engine.check_status()
    assert portions > 400
    for who in "abcde":
        engine.finish(who)


def model_of(vocab, dtype, **options):
    from pagedserve_b200.config.engine_config import EngineConfig
    from pagedserve_b200.config.gpt2 import named_config
    from pagedserve_b200.engine.engine import Engine

    options = dict(dict(num_blocks=128, max_num_seqs=8, dtype=dtype, kv_cache_dtype="int4", enable_cuda_graphs=False), **options)
    return Engine.random(dataclasses.replace(named_config("tiny-a"), vocab_size=vocab), 3, EngineConfig(**options))


@pytest.mark.parametrize("dtype,top", [("bfloat16", 0), ("bfloat16", 6), ("float32", 6)])
@pytest.mark.parametrize("most", [4096, 128])
def test_scores_read_inside_the_heads_product(dtype, top, most):
    """A vocabulary large enough, steps of rows enough: the numbers and the alternatives of the logits that the same steps return."""
    engine = model_of(9000, dtype)
    ops = engine.ops
    ops.FUSED_HEAD_MOST, calls, plain = most, [], ops._fused_head
    ops._fused_head = lambda x, *rest: (calls.append(x.shape[0]), plain(x, *rest))[1]
    prompts = [[(11 * i * i + 5 * n + 1) % 9000 for i in range(100 + n)] for n in range(5)]
    scored = engine.score(prompts, top=top)
    assert calls == ([] if dtype == "float32" else [505] if most == 4096 else [128, 128, 128, 121]) or sum(calls) == 505
    # the same entries in one step, whose logits are formed
    logits = engine.step([(n, prompt[:-1], list(range(len(prompt) - 1))) for n, prompt in enumerate(prompts)]).cpu().double()
    for n in range(len(prompts)):
        engine.finish(n)
    engine.check_status()
    at = 0
    for prompt, result in zip(prompts, scored):
        rows = logits[at:at + len(prompt) - 1]
        at += len(prompt) - 1
        given, entropy, best, ids = logprobs(rows, torch.tensor(prompt[1:]), top)
        # logits in float32 from the same rows, added in another order: 64 products below 1 in size, 2^-24 each and in sums of 9,000 weights 2^-19
        slack = 64 * 2.0 ** -24 * 4 + 2.0 ** -17
        assert (torch.tensor(result.logprobs).double() - given).abs().max() < slack * (1 + given.abs().max())
        assert (torch.tensor(result.entropies).double() - entropy).abs().max() < 20 * slack
        if top:
            found = torch.tensor([[token for token, _ in place] for place in result.alternatives])
            values = torch.tensor([[value for _, value in place] for place in result.alternatives]).double()
            assert (values - best).abs().max() < slack * (1 + best.abs().max())
            assert (torch.gather(rows, 1, found) - torch.gather(rows, 1, ids.long())).abs().max() < slack      # (the tokens, up to logits as near as that)
            assert all(len(set(place)) == top for place in found.tolist())
