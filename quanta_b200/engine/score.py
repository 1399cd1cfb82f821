"""Scoring: how probable given texts are, token by token (the reference's teacher-forced perplexity, src/quanta/minimax/model.py:140-149).

The texts go through the engine as prompts do, in portions and several in a step, with the logits of every place; the log probabilities, the
entropies and the most probable tokens are taken from the logits on the device in one launch a step, and only those travel to the host.
"""

from __future__ import annotations

import math
from collections import deque
from dataclasses import dataclass, field

import torch

from .. import kernels
from .step import StepEntry

LOGITS_BYTES = 1 << 30        # float32 logits a step may hold: bounds the tokens of a step


@dataclass
class TextScores:
    """Of a text of n tokens, for its tokens 1 .. n - 1 (each after those before it): ``logprobs`` (natural logarithms), ``entropies`` of the
    distributions they were chosen from, and, where asked for, the most probable tokens ``top_ids`` with their ``top_logprobs``, most probable first."""
    logprobs: list = field(default_factory=list)
    entropies: list = field(default_factory=list)
    top_ids: list = field(default_factory=list)
    top_logprobs: list = field(default_factory=list)

    @property
    def perplexity(self) -> float:
        """exp of the mean of -logprobs (infinite where that is no float); NaN for a text of one token."""
        if not self.logprobs:
            return math.nan
        try:
            return math.exp(-sum(self.logprobs) / len(self.logprobs))
        except OverflowError:
            return math.inf


def score_rows(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0, status: torch.Tensor | None = None):
    """``(logprob [n], entropy [n], ids [n, top], top logprobs [n, top])`` on the device, of rows of logits ``[n, V]`` and a token each (int32)."""
    n = logits.shape[0]
    logprob = torch.empty(n, dtype=torch.float32, device=logits.device)
    entropy = torch.empty(n, dtype=torch.float32, device=logits.device)
    ids = torch.empty((n, top), dtype=torch.int32, device=logits.device)
    best = torch.empty((n, top), dtype=torch.float32, device=logits.device)
    kernels.token_logprobs(logits, tokens, logprob, entropy, ids, best, status)
    return logprob, entropy, ids, best


def score_texts(engine, texts: list, *, top: int = 0, max_tokens: int, max_position: int | None = None) -> list[TextScores]:
    """Score every text (a list of token ids).  Steps hold at most ``max_tokens`` tokens; texts are taken in as pages and state slots allow."""
    texts = [[int(t) for t in text] for text in texts]
    for i, text in enumerate(texts):
        if not text:
            raise ValueError(f"text {i} is empty")
        bad = [t for t in text if not 0 <= t < engine.vocab_size]
        if bad:
            raise ValueError(f"text {i}: token id {bad[0]} outside the vocabulary of {engine.vocab_size}")
        if max_position is not None and len(text) - 1 > max_position:
            raise ValueError(f"text {i} of {len(text)} tokens: the model has {max_position} positions")
    if not 0 <= top <= min(kernels.TOKEN_LOGPROBS_MAX_TOP, engine.vocab_size):
        raise ValueError(f"top {top}: 0 to {min(kernels.TOKEN_LOGPROBS_MAX_TOP, engine.vocab_size)} most probable tokens can be given")
    max_tokens = max(1, min(int(max_tokens), LOGITS_BYTES // (4 * engine.vocab_size)))
    out = [TextScores() for _ in texts]
    # the last token is only predicted: a text of n tokens brings n - 1
    waiting, live = deque(i for i, text in enumerate(texts) if len(text) > 1), {}
    rid = lambda i: ("score", id(out), i)  # noqa: E731
    try:
        while waiting or live:
            budget, entries, taken, end = max_tokens, [], [], []
            while waiting and len(live) < max_tokens:
                i = waiting[0]
                fits = engine.manager.can_reserve({rid(j): len(texts[j]) - 1 for j in (*live, i)})
                if live and not (fits and sum(not engine.manager.has(rid(j)) for j in (*live, i)) <= engine.manager.slots.free_count):
                    break               # it waits for those that are under way; one alone that does not fit is refused by the step
                live[waiting.popleft()] = 0
            for i, done in live.items():
                n = min(budget, len(texts[i]) - 1 - done)
                if n == 0:
                    break
                entries.append(StepEntry(rid(i), texts[i][done: done + n], tuple(range(n))))
                taken.append((i, done, n))
                budget -= n
                if done + n == len(texts[i]) - 1:
                    end.append(rid(i))
            logits = engine.step(entries, end=end)
            next_tokens = [t for i, done, n in taken for t in texts[i][done + 1: done + n + 1]]
            tokens = torch.tensor(next_tokens, dtype=torch.int32).to(engine.device)
            lp, en, ids, best = (t.tolist() for t in score_rows(logits, tokens, top, engine.status))
            at = 0
            for i, done, n in taken:
                s = out[i]
                s.logprobs += lp[at: at + n]
                s.entropies += en[at: at + n]
                if top:
                    s.top_ids += ids[at: at + n]
                    s.top_logprobs += best[at: at + n]
                at += n
                live[i] = done + n
                if live[i] == len(texts[i]) - 1:
                    del live[i]
        engine.check()
    finally:
        for i in range(len(texts)):
            engine.release(rid(i))
    return out
