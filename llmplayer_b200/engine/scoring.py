"""Log probabilities: of tokens that were chosen, and of given continuations of one prompt.

The reference offers neither (its generation returns tokens only: api/LLMEngine.java:743-769); what is added here follows its
per-step order, one row of logits per token. A prompt that many continuations share is run once; its cached pages are shared by
forked slots, and all continuations run in steps of several tokens that attend over the shared pages together.
"""
from __future__ import annotations

from dataclasses import dataclass, field
from typing import List, Optional, Sequence, Tuple

import torch

from ..errors import RequestError
from ..kernels import ops


@dataclass
class TokenLogprob:
    """One token under the distribution that the model gave before it. Natural logarithms; ``entropy`` in nats; ``rank``: its place,
    from 0, in the order of falling logits; ``top``: the first tokens of that order with their log probabilities."""
    token_id: int
    logprob: float
    entropy: float
    rank: int
    top: List[Tuple[int, float]] = field(default_factory=list)


@dataclass
class ScoredTokens:
    """A continuation, token by token."""
    tokens: List[TokenLogprob]

    @property
    def token_ids(self) -> List[int]:
        return [t.token_id for t in self.tokens]

    @property
    def logprob(self) -> float:
        """Of the whole continuation: the sum over its tokens."""
        return float(sum(t.logprob for t in self.tokens))


class LogprobReader:
    """Log probabilities of one token per row of logits, formed on the device and read back in one copy."""

    def __init__(self, device):
        self.device = device
        self._out: Optional[torch.Tensor] = None
        self._host: Optional[torch.Tensor] = None
        self._staging: Optional[torch.Tensor] = None
        self._targets: Optional[torch.Tensor] = None
        self._done = torch.cuda.Event()

    def read(self, logits: torch.Tensor, tokens: Sequence[int], top: int) -> List[TokenLogprob]:
        R, k = logits.shape[0], int(top)
        if len(tokens) != R:
            raise RequestError(f"{len(tokens)} tokens for {R} rows of logits")
        most = min(ops.TOP_LOGPROBS_MOST, logits.shape[1])
        if not 0 <= k <= most:
            raise RequestError(f"the {top} most likely tokens cannot be listed (at most {most})")
        if R == 0:
            return []
        words = R * (3 + 2 * k)
        if self._out is None or self._out.numel() < words:
            self._out = torch.empty(words, dtype=torch.int32, device=self.device)
            self._host = torch.empty(words, dtype=torch.int32).pin_memory()
        if self._targets is None or self._targets.numel() < R:
            self._targets = torch.empty(R, dtype=torch.int32, device=self.device)
            self._staging = torch.empty(R, dtype=torch.int32).pin_memory()
        self._staging[:R].numpy()[:] = tokens                 # the last call's copy out of it has finished: calls end by waiting
        targets = self._targets[:R]
        targets.copy_(self._staging[:R], non_blocking=True)
        out = self._out[:words]
        logprob, entropy, rank = out[:R].view(torch.float32), out[R:2 * R].view(torch.float32), out[2 * R:3 * R]
        ids = out[3 * R:(3 + k) * R].view(R, k) if k else None
        lps = out[(3 + k) * R:].view(torch.float32).view(R, k) if k else None
        with ops.section("logprobs"):
            ops.token_logprobs(logits, targets, logprob, entropy, rank, top_ids=ids, top_logprobs=lps)
        host = self._host[:words]
        host.copy_(out, non_blocking=True)
        self._done.record()
        self._done.synchronize()
        as_float = host.view(torch.float32)
        lp, ent, ranks = as_float[:R].tolist(), as_float[R:2 * R].tolist(), host[2 * R:3 * R].tolist()
        listed = [[] for _ in range(R)]
        if k:
            rows, values = host[3 * R:(3 + k) * R].view(R, k).tolist(), as_float[(3 + k) * R:].view(R, k).tolist()
            listed = [list(zip(a, b)) for a, b in zip(rows, values)]
        return [TokenLogprob(int(t), a, b, c, d) for t, a, b, c, d in zip(tokens, lp, ent, ranks, listed)]


# Logits of one step of scoring: at most so many bytes of float32 rows.
SCORE_LOGITS_BYTES = 1 << 30


def score(engine, prompt: Sequence[int], continuations: Sequence[Sequence[int]], top: int) -> List[ScoredTokens]:
    """See :meth:`Engine.score`."""
    prompt = [int(t) for t in prompt]
    conts = [[int(t) for t in c] for c in continuations]
    if not prompt:
        raise RequestError("score: empty prompt")
    most = min(ops.TOP_LOGPROBS_MOST, engine.vocab_size)
    if not 0 <= int(top) <= most:
        raise RequestError(f"score: the {top} most likely tokens cannot be listed (at most {most})")
    for tokens in [prompt] + conts:
        bad = [t for t in tokens if not 0 <= t < engine.vocab_size]
        if bad:
            raise RequestError(f"score: token id {bad[0]} lies outside the vocabulary of {engine.vocab_size}")
    longest = max((len(c) for c in conts), default=0)
    if len(prompt) - 1 + longest > engine.context_length:
        raise RequestError(f"score: {len(prompt)} prompt and {longest} further tokens exceed the context length of {engine.context_length}")
    results: List[List[TokenLogprob]] = [[] for _ in conts]
    most_rows = max(1, SCORE_LOGITS_BYTES // (4 * engine.vocab_size))
    todo = [i for i, c in enumerate(conts) if c]
    if not todo:
        return [ScoredTokens(r) for r in results]
    # the last prompt token runs with each continuation: its logits are the first token's
    before = prompt[:-1]
    parent = None
    held: List[int] = []
    try:
        if before and len(todo) > 1 and engine.cache.slots.num_free > 1:
            parent = engine.acquire()
            engine.step([(parent, before)], [[]])
        while todo:
            if parent is not None and not engine.forks_fit(parent, [len(conts[todo[0]])]):
                engine.release(parent)             # no room beside it: the prompt is run with each continuation
                parent = None
            batch, rows = [], 0
            for i in todo:
                more = [len(conts[j]) + (0 if parent is not None else len(before)) for j in batch + [i]]
                if batch and (rows + len(conts[i]) > most_rows or not engine.forks_fit(parent, more)):
                    break
                batch.append(i)
                rows += len(conts[i])
            todo = todo[len(batch):]
            if parent is not None:
                held = engine.fork(parent, len(batch))
            else:
                for _ in batch:
                    held.append(engine.acquire())
                if before:
                    engine.step([(slot, before) for slot in held], [[]] * len(held))
            runs = [prompt[-1:] + conts[i][:-1] for i in batch]
            # one step, or several if a single continuation has more tokens than a step may have rows of logits
            for a in range(0, max(len(r) for r in runs), most_rows):
                pieces = [(slot, i, r[a:a + most_rows]) for slot, i, r in zip(held, batch, runs) if a < len(r)]
                logits = engine.step([(slot, piece) for slot, _, piece in pieces], [list(range(len(piece))) for _, _, piece in pieces])
                wanted = [t for _, i, piece in pieces for t in conts[i][a:a + len(piece)]]
                scored = engine.token_logprobs(logits, wanted, top=top)
                at = 0
                for _, i, piece in pieces:
                    results[i] += scored[at:at + len(piece)]
                    at += len(piece)
            while held:
                engine.release(held.pop())
    finally:
        while held:
            engine.release(held.pop())
        if parent is not None:
            engine.release(parent)
    engine.check()
    return [ScoredTokens(r) for r in results]
