"""A beam search by recomputing every hypothesis from its first token, and the plain kernels that the engine's
own needs beside those of plain_ops.py (CPU)."""

import math

import torch

import plain_packed as plain
from plain_ops import PlainOps


class BeamOps(PlainOps):
    def beam_select(self, logits, scores, *, ended=None, end_tokens=None):
        ends = tuple(end_tokens.tolist()) if end_tokens is not None else ()
        rows = plain.choose(logits, scores, ended, ends)
        column = lambda i, kind: torch.tensor([[c[i] for c in row] for row in rows], dtype=kind)
        return (column(0, torch.float32), column(1, torch.int32), column(2, torch.int32), column(3, torch.uint8))

    def reorder_slots(self, state, slots, parents):
        beams = parents.shape[1]
        source = torch.arange(slots.numel()) // beams * beams + parents.view(-1).long()
        state[:, slots.long()] = state[:, slots.long()[source]]

    def reorder_pages(self, storage, block_table, parents, starts, lengths, *, page_size):
        beams, before = parents.shape[1], storage.clone()
        for row in range(block_table.shape[0]):
            r = row // beams
            for block in range(int(starts[r]) // page_size, -(-int(lengths[r]) // page_size)):
                source = int(block_table[r * beams + int(parents[r, row % beams]), block])
                target = int(block_table[row, block])
                if source >= 0 and target >= 0:
                    storage[:, target] = before[:, source]


def beam_search(logits_of, prompt, beams, max_tokens, ends):
    """[(tokens without the end token, score, ended)], best score first; None where two candidates at the
    border are so near that rounding decides."""
    live = [((), 0.0, False)]
    for _ in range(max_tokens):
        found = []
        for tokens, score, over in live:
            if over:
                found.append((tokens, score, True))
                continue
            logs = torch.log_softmax(logits_of(list(prompt) + list(tokens))[-1].double(), -1)
            for v in torch.topk(logs, min(beams + 1, logs.numel())).indices.tolist():
                found.append((tokens + (v,), score + float(logs[v]), v in ends))
        found.sort(key=lambda c: -c[1])
        near = [a[1] - b[1] for a, b in zip(found[:beams], found[1:beams + 1])]
        if near and min(near) < 1e-4:
            return None
        live = found[:beams]
        if all(c[2] for c in live):
            break
    return [(t[:-1] if over else t, score, over) for t, score, over in live]


def same_hypotheses(got, want, length_penalty=1.0, atol=1e-3):
    """Whether an engine's results are these hypotheses, ranked by the penalised score."""
    rank = lambda t, score, over: score / max(len(t) + over, 1) ** length_penalty
    want = sorted(want, key=lambda c: -rank(*c))
    assert len(got) == len(want)
    for result, (tokens, score, over) in zip(got, want):
        assert result.token_ids == tokens and result.finish_reason == ("stop" if over else "length")
        assert result.generation_tokens == len(tokens) and math.isclose(result.score, score, abs_tol=atol)
