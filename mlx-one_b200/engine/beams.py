"""Beam search over the step function: several hypotheses of one prompt, decoded side by side.

Every hypothesis is a request of the cache with pages and slots of its own. A step runs one token of
each; the kernels then choose the best continuations over all of them (``beam_select``), bring the
caches to the hypotheses that continue them (``CacheOrder``) and publish the chosen tokens, which
the next step takes on the device. The host only launches; every few steps it looks whether all
hypotheses have ended.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Any, Sequence

import torch

from ..cache.manager import CacheManager
from .runner import Runner, StepEntry

# steps between two looks at whether every hypothesis has ended (a look waits for the device)
LOOK_EVERY = 8


@dataclass(frozen=True)
class Hypothesis:
    """``tokens``: without the end-of-sequence token. ``score``: the sum of the tokens' logarithms, that
    one's among them. ``ended``: by such a token."""

    tokens: tuple[int, ...]
    score: float
    ended: bool


def search(runner: Runner, cache: CacheManager, prompt: Sequence[int], *, beams: int, max_tokens: int,
           end_tokens: Sequence[int], portion: int, name: Any = "beam") -> list[Hypothesis]:
    """The ``beams`` best hypotheses of up to ``max_tokens`` tokens, best score first. The prompt runs
    in portions of ``portion`` tokens; everything the hypotheses will hold is reserved beforehand
    (``CacheCapacityError`` if it does not fit)."""
    ops, device = runner.model.ops, cache.device
    ids = [(name, b) for b in range(beams)]
    opened: list[Any] = []
    try:
        for request in ids:
            cache.open(request, reserve_tokens=len(prompt) + max_tokens)
            opened.append(request)
        portions = [list(prompt[i:i + portion]) for i in range(0, len(prompt), portion)]
        logits = None
        for tokens in portions:
            want = (len(tokens) - 1,) if tokens is portions[-1] else ()
            logits = runner.step([StepEntry(ids[0], tokens, want)])
        for request in ids[1:]:
            # (the same portions: pages behind a window are given back alike)
            for tokens in portions:
                cache.grow(request, len(tokens))
                cache.advance(request, len(tokens))
        ends = torch.tensor(list(end_tokens), dtype=torch.int32, device=device) if end_tokens else None
        index = torch.tensor([cache.get(request).index for request in ids], dtype=torch.int32, device=device)
        scores = torch.full((1, beams), float("-inf"), dtype=torch.float32, device=device)
        scores[0, 0] = 0.0
        # one hypothesis so far: the other rows, of minus infinity, are not read
        choice = ops.beam_select(logits.expand(beams, -1), scores, end_tokens=ends)
        order, first = cache.order_of(ids), 0
        history = []
        for step in range(max_tokens):
            scores, parents, tokens, ended = choice
            history.append((parents, tokens))
            if step + 1 == max_tokens or (ends is not None and step % LOOK_EVERY == LOOK_EVERY - 1
                                          and bool(ended.all())):
                break
            order.apply(ops, parents, first)
            first = len(prompt)
            ops.publish_tokens(tokens.view(-1), index, runner.published)
            logits = runner.step([StepEntry(request, (0,), (0,), from_device=True) for request in ids])
            choice = ops.beam_select(logits, scores, ended=ended if ends is not None else None,
                                     end_tokens=ends)
        parents = torch.stack([h[0] for h in history]).view(-1, beams).tolist()
        tokens = torch.stack([h[1] for h in history]).view(-1, beams).tolist()
        last, over = scores.view(-1).tolist(), ended.view(-1).tolist()
        check = getattr(ops, "check_errors", None)
        if check is not None:
            check()
    finally:
        for request in opened:
            cache.close(request)
    stops = set(end_tokens)
    found = []
    for b in range(beams):
        if last[b] == float("-inf"):
            continue                     # (fewer continuations than hypotheses)
        path, at = [], b
        for parent, token in zip(reversed(parents), reversed(tokens)):
            path.append(token[at])
            at = parent[at]
        path.reverse()
        if over[b]:
            path = path[:next(i for i, token in enumerate(path) if token in stops)]
        found.append(Hypothesis(tuple(path), last[b], bool(over[b])))
    return found
