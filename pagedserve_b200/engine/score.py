"""Scoring given texts: the log probability of every prompt token behind the first.

Prompts run in portions under the engine's token budget, several at a time while pages and slots last, through the step that
generation uses; the head gives the log probabilities without forming the logits as a whole.
"""

from __future__ import annotations

from dataclasses import dataclass, field
from typing import List, Sequence, Tuple

from pagedserve_b200.cache.manager import CacheFull
from pagedserve_b200.engine.batch import StepEntry


@dataclass
class PromptScore:
    """Of one prompt; place i stands for its token i + 1, given tokens 0 .. i."""

    logprobs: List[float] = field(default_factory=list)
    entropies: List[float] = field(default_factory=list)                       # of the distribution at the place, in nats
    alternatives: List[List[Tuple[int, float]]] = field(default_factory=list)  # (token, log probability), most likely first

    @property
    def total(self) -> float:
        return float(sum(self.logprobs))


class _Running:
    """A prompt on its way: a request of its own name, and how many of its tokens have run."""

    def __init__(self, tokens, result):
        self.tokens, self.result, self.done = tokens, result, 0


def score(engine, prompts: Sequence[Sequence[int]], top: int = 0) -> List[PromptScore]:
    from pagedserve_b200.kernels.ops import MOST_ALTERNATIVES

    if not 0 <= top <= min(MOST_ALTERNATIVES, engine.vocab_size):
        raise ValueError(f"top is 0 to {MOST_ALTERNATIVES}, and at most the vocabulary")
    prompts = [[int(token) for token in prompt] for prompt in prompts]
    cache, budget = engine.cache, engine.config.max_num_batched_tokens
    for prompt in prompts:
        if not prompt or len(prompt) > engine.max_model_len:
            raise ValueError(f"a prompt has 1 to {engine.max_model_len} tokens")
        if any(not 0 <= token < engine.vocab_size for token in prompt):
            raise ValueError(f"a prompt's token is outside the vocabulary of {engine.vocab_size}")
        if cache.pages_for_tokens(len(prompt)) > cache.total_pages():
            raise ValueError("a prompt is longer than the cache")
    results = [PromptScore() for _ in prompts]
    # (nothing is known about the first token, so the last one need not run: what comes behind it is not asked)
    waiting = [_Running(prompt, result) for prompt, result in zip(prompts, results) if len(prompt) > 1]
    running: List[_Running] = []
    try:
        while waiting or running:
            promised = sum(cache.pages_for_tokens(len(one.tokens) - 1) - cache.pages_for_tokens(one.done) for one in running)
            while waiting and len(running) < min(budget, cache.free_slots + sum(one in cache for one in running)):
                pages = cache.pages_for_tokens(len(waiting[0].tokens) - 1)
                if cache.free_pages() - promised < pages:
                    break
                promised += pages
                running.append(waiting.pop(0))
            if not running:
                raise CacheFull("no pages or slots are left for a prompt")
            entries, targets, room = [], [], budget
            for one in running:
                count = min(room, len(one.tokens) - 1 - one.done)
                if count > 0:
                    entries.append((one, count))
                    targets += one.tokens[one.done + 1:one.done + 1 + count]
                    room -= count
            found = engine.runner.score([StepEntry(one, one.tokens[one.done:one.done + count], list(range(count))) for one, count in entries],
                                        targets, top)
            logprobs, entropies, values, ids = (tensor.tolist() for tensor in found)
            at = 0
            for one, count in entries:
                one.result.logprobs += logprobs[at:at + count]
                one.result.entropies += entropies[at:at + count]
                one.result.alternatives += [list(zip(ids[place], values[place])) for place in range(at, at + count)]
                one.done += count
                at += count
                if one.done == len(one.tokens) - 1:
                    running.remove(one)
                    engine.finish(one)
        engine.check_status()
    finally:
        for one in running:
            if one in cache:
                engine.finish(one)
    return results
