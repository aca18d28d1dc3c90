"""The engine with a cache held in 4 bits, and the scores of given texts, against the plain implementations."""

import pytest
import torch

import plain_gpt2
from plain_packed import held, logprobs

pytestmark = pytest.mark.gpu


def engine_for(name, dtype, cache, **options):
    from pagedserve_b200.main import build_engine

    options = dict(dict(num_blocks=64, max_num_seqs=4, block_size=16), **options)
    return build_engine(name, seed=3, dtype=dtype, kv_cache_dtype=cache, **options)


def plain_logits(engine, tokens, packed):
    """Plain GPT-2 logits of every token, keys and values rounded as the cache rounds them."""
    config = engine.model_config
    weights = {name: tensor.double().cpu() for name, tensor in engine.plain.items()}
    ids = torch.tensor(tokens)
    prefix = "transformer."
    x = weights[prefix + "wte.weight"][ids] + weights[prefix + "wpe.weight"][:len(tokens)]
    width, heads = config.n_embd, config.n_head
    dim = width // heads

    def norm(x, name):
        mean, var = x.mean(-1, keepdim=True), x.var(-1, unbiased=False, keepdim=True)
        return (x - mean) / torch.sqrt(var + config.layer_norm_epsilon) * weights[name + ".weight"] + weights[name + ".bias"]

    for i in range(config.n_layer):
        at = f"{prefix}h.{i}."
        qkv = norm(x, at + "ln_1") @ weights[at + "attn.c_attn.weight"] + weights[at + "attn.c_attn.bias"]
        q, k, v = (part.reshape(len(tokens), heads, dim) for part in qkv.split(width, -1))
        if packed:
            k, v = (torch.from_numpy(held(rows.float().numpy())).double() for rows in (k, v))
        s = torch.einsum("ihd,jhd->hij", q, k) / dim ** 0.5
        s = s.masked_fill(torch.ones(len(tokens), len(tokens)).triu(1).bool(), float("-inf"))
        x = x + torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), v).reshape(len(tokens), width) @ weights[at + "attn.c_proj.weight"] \
            + weights[at + "attn.c_proj.bias"]
        h = norm(x, at + "ln_2") @ weights[at + "mlp.c_fc.weight"] + weights[at + "mlp.c_fc.bias"]
        x = x + torch.nn.functional.gelu(h, approximate="tanh") @ weights[at + "mlp.c_proj.weight"] + weights[at + "mlp.c_proj.bias"]
    return norm(x, prefix + "ln_f") @ weights[prefix + "wte.weight"].T


@pytest.fixture(scope="module")
def tiny():
    """Engines of tiny-a's weights, with the tensors they were made of."""
    from pagedserve_b200.config.gpt2 import named_config
    from pagedserve_b200.weights.random_init import random_tensors

    made = {}

    def make(dtype, cache):
        if (dtype, cache) not in made:
            made[dtype, cache] = engine_for("tiny-a", dtype, cache)
            made[dtype, cache].plain = random_tensors(named_config("tiny-a"), 3)
        return made[dtype, cache]

    return make


TOKENS = [3, 14, 159, 265, 358, 97, 93, 238, 462, 64, 33, 83, 279, 50, 28, 84, 197, 169, 399, 37, 51, 5, 82, 97, 49, 445, 92, 307, 81, 64, 6, 28, 62, 8]


def test_the_plain_layers_are_the_engines(tiny):
    """Without rounding the restatement here is the plain implementation's."""
    import tempfile

    from pagedserve_b200.config.gpt2 import named_config
    from pagedserve_b200.weights.random_init import write_random_model

    with tempfile.TemporaryDirectory() as folder:
        write_random_model(folder, named_config("tiny-a"), seed=3)
        config, weights = plain_gpt2.read_folder(folder, dtype=torch.float64)
        want = plain_gpt2.forward_logits(config, weights, TOKENS)
    assert (plain_logits(tiny("float32", "model"), TOKENS, packed=False) - want).abs().max() < 1e-9


@pytest.mark.parametrize("cut", [[34], [1] * 34, [16, 18], [20, 1, 1, 12], [5, 5, 24]])
def test_logits_with_a_packed_cache(tiny, cut):
    """Prompts as a whole, token by token, in portions: one and the same rounded cache behind them.  (float32 results may fall on the other side of a
    code's border than 64-bit ones: a step of a number that meets small weights.)"""
    engine = tiny("float32", "int4")
    want = plain_logits(engine, TOKENS, packed=True)
    unrounded = plain_logits(engine, TOKENS, packed=False)
    at, rows = 0, []
    for count in cut:
        rows.append(engine.step([("r", TOKENS[at:at + count], list(range(count)))]).cpu().double())
        at += count
    engine.finish("r")
    engine.check_status()
    got = torch.cat(rows)
    assert (got - want).norm() < 0.02 * (unrounded - want).norm() + 1e-5 * want.norm()


def test_mixed_steps_and_generation(tiny):
    """Prompts beside single tokens, decode graphs, a scheduler run: the same tokens whichever way they are batched."""
    from pagedserve_b200.engine.engine import generate

    engine = tiny("float32", "int4")
    prompts = [TOKENS[:7], TOKENS[3:30], TOKENS[10:11], TOKENS]
    alone = [generate(engine, [prompt], max_new_tokens=10)[0] for prompt in prompts]
    assert generate(engine, prompts, max_new_tokens=10) == alone
    assert generate(engine, prompts, max_new_tokens=10, strategy="sarathi", prefill_chunk_size=8) == alone
    assert engine.cache.groups[0].pool.dtype == torch.uint8 and engine.cache.live_requests == 0
    engine.cache.check_invariants()


@pytest.mark.parametrize("name", ["zositar-tiny", "tefopel-tiny", "tiny-b"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_designs_run_with_a_packed_cache(name, dtype):
    """Turned and normed keys, values that are unturned keys, borrowed caches, windows, chunks, sinks and caps: prompts as a whole and token by
    token agree to what the compute type's own cache agrees to, and both are near the unrounded cache."""
    logits = {}
    for cache in ("int4", "model"):
        engine = engine_for(name, dtype, cache)
        tokens = [(7 * i + 3) % engine.vocab_size for i in range(60)]
        whole = engine.step([("a", tokens, list(range(60)))]).float().cpu()
        engine.finish("a")
        single = torch.cat([engine.step([("b", [token], [0])]) for token in tokens]).float().cpu()
        engine.finish("b")
        engine.check_status()
        logits[cache] = whole, single
    spread = logits["model"][0].norm()
    rounding = (logits["int4"][0] - logits["model"][0]).norm() / spread
    assert 1e-4 < rounding < 0.3                                        # 4 bits: something, and not everything
    own = (logits["model"][0] - logits["model"][1]).norm() / spread
    # A number near a border between codes falls to either side, one step apart.  Rows that differ by d of themselves (bfloat16 roundings in front of
    # the cache, about 2^-7 in all; float32 ones 2^-20) put a share d |x| / step of the numbers there, with step about 0.28 of |x|'s spread: 2.2 %.  Their
    # error, a step each, against the rounding's own, step / sqrt(12) for every number: sqrt(12 * 0.022) = 0.51 of it (float32 0.006).
    assert (logits["int4"][0] - logits["int4"][1]).norm() / spread < 4 * own + (0.75 if dtype == "bfloat16" else 0.05) * rounding


def test_caches_of_another_kind_are_refused():
    from pagedserve_b200.config.registry import ConfigError

    for name in ("gozunex-tiny", "vozirax-tiny", "suvunex-tiny"):
        with pytest.raises(ConfigError, match="int4"):
            engine_for(name, "float32", "int4")


def test_pages_cost_less():
    small, large = engine_for("tiny-b", "bfloat16", "int4", block_size=16), engine_for("tiny-b", "bfloat16", "model", block_size=16)
    # head size 48: two groups of 20 bytes a row, 96 in bfloat16
    assert small.bytes_per_block * 96 == large.bytes_per_block * 40 == small.cache.groups[0].bytes_per_page * 96


# ------------------------------------------------------------------------------------------------ scores
@pytest.mark.parametrize("cache", ["model", "int4"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_scores_of_texts(tiny, dtype, cache):
    """Against the log probabilities of the engine's own logits, prompts of one token to many, several at a time, in portions."""
    engine = tiny(dtype, cache)
    prompts = [TOKENS, TOKENS[:1], TOKENS[5:7], TOKENS[::-1], TOKENS[:16], TOKENS[:17]]
    scored = engine.score(prompts, top=4)
    slack = 2e-5 if dtype == "float32" else 0.2
    for prompt, result in zip(prompts, scored):
        assert len(result.logprobs) == len(result.entropies) == len(result.alternatives) == len(prompt) - 1
        if len(prompt) == 1:
            continue
        logits = engine.step([("x", prompt, list(range(len(prompt))))]).cpu().double()
        engine.finish("x")
        given, entropy, best, ids = logprobs(logits[:-1], torch.tensor(prompt[1:]), 4)
        assert (torch.tensor(result.logprobs).double() - given).abs().max() < slack
        assert (torch.tensor(result.entropies).double() - entropy).abs().max() < slack
        assert (torch.tensor([[value for _, value in place] for place in result.alternatives]).double() - best).abs().max() < slack
        assert abs(result.total - sum(result.logprobs)) < 1e-9
    assert engine.cache.live_requests == 0
    engine.cache.check_invariants()


def test_scores_under_a_small_budget_and_few_pages():
    engine = engine_for("tiny-a", "float32", "int4", num_blocks=5, max_num_batched_tokens=20, max_num_seqs=2)
    prompts = [TOKENS, TOKENS[:9], TOKENS[2:], TOKENS[:3]]
    wide = engine_for("tiny-a", "float32", "int4").score(prompts)
    for a, b in zip(engine.score(prompts), wide):
        assert (torch.tensor(a.logprobs) - torch.tensor(b.logprobs)).abs().max() < 0.05
    for bad in ([[]], [[1] * 200], [[-1, 2]], [[512, 1]]):
        with pytest.raises(ValueError):
            engine.score(bad)
    with pytest.raises(ValueError):
        engine.score([[1, 2]], top=33)
    assert engine.cache.live_requests == 0


def test_logprobs_of_a_step(tiny):
    engine = tiny("float32", "int4")
    logits = engine.step([("s", TOKENS[:5], [0, 4])])
    engine.finish("s")
    found = engine.logprobs(logits, [TOKENS[1], -1], top=2)
    given, entropy, best, ids = logprobs(logits.cpu().double(), torch.tensor([TOKENS[1], -1]), 2)
    assert (found.logprob.cpu() - given).abs().max() < 1e-5 and torch.equal(found.top_ids.cpu(), ids)
    with pytest.raises(ValueError):
        engine.logprobs(logits, [1, 2, 3])
    with pytest.raises(ValueError):
        engine.logprobs(logits, [1, 512])


def test_the_command_line(capsys):
    from pagedserve_b200.main import main

    assert main(["--model", "tiny-a", "--seed", "3", "--kv-cache-dtype", "int4", "--num-blocks", "32", "--prompt-ids", "3 14 159", "--score",
                 "--top-logprobs", "2"]) == 0
    lines = capsys.readouterr().out.strip().split("\n")
    assert len(lines) == 3 and lines[0].startswith("prompt 0:") and "top" in lines[1]
    assert main(["--model", "tiny-a", "--seed", "3", "--kv-cache-dtype", "int4", "--num-blocks", "32", "--prompt-ids", "3 14 159"]) == 0
