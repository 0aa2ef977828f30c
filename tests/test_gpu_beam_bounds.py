"""A beam's choice where its bound counts: large vocabularies and more hypotheses than a few, in clusters (up to eight)
and by the last block; and the vocabularies below which a row is walked value by value."""

import math

import pytest
import torch

from test_gpu_beams import DEVICE, check
from test_gpu_kernels import ops  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("beams", [1, 3, 6, 7, 8, 9, 16, 24, 32])
@pytest.mark.parametrize("vocab", [8192, 8193, 16384, 24577, 33000, 65536, 70001])
def test_random_logits(ops, beams, vocab):
    generator = torch.Generator().manual_seed(100 * beams + vocab)
    logits = 3 * torch.randn(2 * beams, vocab, generator=generator)
    scores = -4 * torch.rand(2, beams, generator=generator)
    check(ops, logits, scores)
    check(ops, logits, scores, ended=torch.rand(2, beams, generator=generator) < 0.3)
    # the first step: one hypothesis there is, whose row all the others share
    scores[:, 1:] = -math.inf
    check(ops, logits[:1].expand(2 * beams, -1), scores)


@pytest.mark.parametrize("beams", [4, 8, 12, 32])
def test_numbers_that_are_none_and_few_that_are_left(ops, beams):
    """NaN and infinities among the best; rows of which a mask leaves fewer threads than hypotheses, or one part."""
    generator = torch.Generator().manual_seed(beams)
    vocab = 66000
    logits = 3 * torch.randn(2 * beams, vocab, generator=generator)
    best = logits.topk(beams, -1).indices
    logits[0, best[0, ::2]] = math.nan
    logits[1, best[1]] = -math.inf
    logits[2, torch.rand(vocab, generator=generator) < 0.9] = math.nan
    kept = logits[3, 65000:65040].clone()
    logits[3] = -math.inf
    logits[3, 65000:65040] = kept                            # ten threads of one part
    logits[beams] = torch.finfo(torch.float32).min
    logits[beams, 8191:8193] = 0.5                           # across two parts
    logits[beams + 1] = math.nan
    logits[beams + 2, 17] = math.inf
    scores = -4 * torch.rand(2, beams, generator=generator)
    check(ops, logits, scores)
    scores[0, 0], scores[1, 3] = math.nan, math.inf
    check(ops, logits, scores, ended=torch.rand(2, beams, generator=generator) < 0.3)


@pytest.mark.parametrize("beams", [5, 8, 17])
def test_equal_logits_at_the_bound(ops, beams):
    """The last that are taken equal others: few of them, and more than the lists hold."""
    generator = torch.Generator().manual_seed(beams)
    logits = torch.randn(beams, 65536, generator=generator)
    scores = torch.zeros(1, beams)
    for count in (beams, 100, 600, 20000):
        x = logits.clone()
        x[:, torch.randperm(65536, generator=generator)[:count]] = 8.0
        x[0, 7], x[beams - 1, 40000] = 9.0, 9.0
        check(ops, x, scores)
        check(ops, x, -torch.arange(float(beams))[None])
