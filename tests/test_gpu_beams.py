"""A beam's choice and the reordering of slots and pages, against plain_packed.py."""

import math

import pytest
import torch

import plain_packed as plain
from test_gpu_kernels import ops  # noqa: F401  (fixture)
from mlx_one_b200.kernels import KernelError

pytestmark = pytest.mark.gpu
DEVICE = "cuda:0"


def check(ops, logits, scores, ended=None, ends=(2, 7)):
    got = ops.beam_select(logits.to(DEVICE), scores.to(DEVICE), ended=None if ended is None else ended.to(DEVICE),
                          end_tokens=torch.tensor(ends, dtype=torch.int32, device=DEVICE) if ends else None)
    want = plain.choose(logits, scores, ended, ends)
    values, parents, tokens, over = (x.cpu() for x in got)
    for r, row in enumerate(want):
        assert parents[r].tolist() == [c[1] for c in row], r
        assert tokens[r].tolist() == [c[2] for c in row], r
        assert over[r].tolist() == [c[3] for c in row], r
        expected = torch.tensor([c[0] for c in row])
        # a logarithm of a sum of exponentials whose arguments, up to 2^5, have 24 bits; the result's rounding
        torch.testing.assert_close(values[r].double(), expected.double(), atol=1e-5, rtol=2.0 ** -22)
    return got


@pytest.mark.parametrize("requests,beams,vocab", [
    (1, 1, 1), (1, 4, 5), (3, 2, 130), (1, 4, 65536), (5, 7, 1023), (2, 16, 4099), (1, 32, 40), (1, 32, 3001),
    (33, 3, 257), (2, 5, 100003)])
def test_choices(ops, requests, beams, vocab):
    generator = torch.Generator().manual_seed(requests * 1000 + vocab)
    logits = 3 * torch.randn(requests * beams, vocab, generator=generator)
    scores = -4 * torch.rand(requests, beams, generator=generator)
    check(ops, logits, scores)
    check(ops, logits, scores, ends=())
    check(ops, logits, scores, ended=torch.rand(requests, beams, generator=generator) < 0.3)
    check(ops, logits, scores, ended=torch.ones(requests, beams, dtype=torch.uint8))


@pytest.mark.parametrize("vocab", [37, 1500, 70000])
def test_ties_go_to_the_lowest_place(ops, vocab):
    generator = torch.Generator().manual_seed(vocab)
    few = torch.randint(0, 3, (8, vocab), generator=generator).float()
    few[0] = few[1]                                           # the same row twice, with the same score
    few[2, :] = -0.0
    few[3, ::2] = 0.0
    few[3, 1::2] = -0.0
    scores = torch.tensor([[-1.0, -1.0, -2.0, -0.5], [0.0, 0.0, 0.0, 0.0]])
    check(ops, few, scores)
    check(ops, torch.zeros(8, vocab), scores)
    # the first step: one hypothesis there is
    check(ops, few, torch.tensor([[-1.0, -math.inf, -math.inf, -math.inf]] * 2))


def test_rows_that_are_not_numbers(ops):
    generator = torch.Generator().manual_seed(0)
    logits = torch.randn(12, 999, generator=generator)
    logits[0, 5] = math.nan
    logits[1] = -math.inf
    logits[1, 17] = 0.5                                       # one token left
    logits[2] = -math.inf
    logits[4] = math.nan
    logits[5, 100] = math.inf
    logits[6] = -3.4028234e38                                 # masks of the type's lowest value
    logits[6, 3:5] = 1.0
    logits[8, 1:] = -math.inf
    scores = -torch.rand(3, 4, generator=generator)
    scores[2, 1], scores[2, 2] = math.nan, math.inf
    check(ops, logits, scores)
    check(ops, logits, scores, ended=torch.tensor([[0, 1, 0, 0], [1, 0, 0, 1], [0, 1, 0, 1]], dtype=torch.uint8))


@pytest.mark.parametrize("beams,vocab", [(3, 37), (4, 9000), (12, 20011)])
def test_masks_of_the_lowest_value(ops, beams, vocab):
    """A row that a mask of the type's lowest value leaves nothing of has that many equal tokens; one that is left
    in a row is certain; beside tokens of minus infinity the masked ones are what there is."""
    lowest = torch.finfo(torch.float32).min
    logits = torch.full((2 * beams, vocab), lowest)
    logits[1, vocab - 2] = 0.25
    logits[2, ::2] = -math.inf
    logits[beams + 1] = torch.randn(vocab, generator=torch.Generator().manual_seed(vocab))
    logits[beams + 2] = -math.inf
    scores = -torch.arange(2.0 * beams).view(2, beams) / 8
    check(ops, logits, scores)
    got, parents, tokens, _ = ops.beam_select(logits[:1].expand(beams, -1).to(DEVICE),
                                              torch.tensor([[0.0] + [-math.inf] * (beams - 1)], device=DEVICE))
    assert tokens.tolist() == [list(range(beams))] and not parents.any()
    torch.testing.assert_close(got, torch.full_like(got, -math.log(vocab)), atol=1e-5, rtol=2.0 ** -22)


def test_rows_of_wider_ones_and_replays(ops):
    """Rows that are slices, at any alignment; a captured choice with other contents."""
    generator = torch.Generator().manual_seed(4)
    wide = torch.randn(8, 2011, generator=generator)
    scores = -torch.rand(2, 4, generator=generator)
    on_device = wide.to(DEVICE)
    for first, last in ((0, 2000), (1, 1777), (4, 2004), (3, 2011)):
        got = ops.beam_select(on_device[:, first:last], scores.to(DEVICE))
        want = ops.beam_select(on_device[:, first:last].contiguous(), scores.to(DEVICE))
        assert all(torch.equal(a, b) for a, b in zip(got[1:], want[1:]))
        torch.testing.assert_close(got[0], want[0], atol=1e-5, rtol=0)
        check(ops, wide[:, first:last].contiguous(), scores)
    rows, held = on_device.clone(), scores.to(DEVICE)
    ops.beam_select(rows, held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = ops.beam_select(rows, held)
    for _ in range(3):
        rows.copy_(torch.randn(rows.shape, generator=generator).to(DEVICE))
        graph.replay()
        again = [x.clone() for x in captured]
        assert all(torch.equal(a, b) for a, b in zip(again, ops.beam_select(rows, held)))


@pytest.mark.parametrize("beams", [7, 8, 9, 12, 31])
def test_ties_numbers_and_replays_of_many_hypotheses(ops, beams):
    """Both ways in which a request's rows hand their candidates over, a cluster's (up to eight) and the last block's."""
    generator = torch.Generator().manual_seed(beams)
    rows, vocab = 3 * beams, 8200
    logits = torch.randint(0, 3, (rows, vocab), generator=generator).float()
    scores = torch.randint(-2, 1, (3, beams), generator=generator).float()
    check(ops, logits, scores)
    logits = 3 * torch.randn(rows, vocab, generator=generator)
    logits[0, 5], logits[1], logits[2, 8195], logits[3, 1:] = math.nan, -math.inf, math.inf, -math.inf
    scores[1, 2], scores[2, 0], scores[2, 1] = math.nan, -math.inf, math.inf
    ended = torch.rand(3, beams, generator=generator) < 0.4
    check(ops, logits, scores)
    check(ops, logits, scores, ended=ended)
    x, held, over = logits.to(DEVICE), scores.to(DEVICE), ended.to(DEVICE)
    ends = torch.tensor([3, 8], dtype=torch.int32, device=DEVICE)
    ops.beam_select(x, held, ended=over, end_tokens=ends)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first = ops.beam_select(x, held, ended=over, end_tokens=ends)
        second = ops.beam_select(x, first[0], ended=first[3], end_tokens=ends)
    for _ in range(3):
        x.copy_(torch.randn(rows, vocab, generator=generator).to(DEVICE))
        graph.replay()
        again = [y.clone() for y in (*first, *second)]
        one = ops.beam_select(x, held, ended=over, end_tokens=ends)
        two = ops.beam_select(x, one[0], ended=one[3], end_tokens=ends)
        assert all(torch.equal(a, b) for a, b in zip(again, (*one, *two)))


@pytest.mark.parametrize("beams", [1, 2, 4, 5, 8, 13, 16, 32])
@pytest.mark.parametrize("shape,dtype", [((3, 40), torch.bfloat16), ((2, 1024), torch.float32), ((7,), torch.uint8),
                                         ((5, 3), torch.float32), ((70000,), torch.uint8)])
def test_slots(ops, beams, shape, dtype):
    """Cycles, several children of one parent, parents without a child; the other slots stay."""
    generator = torch.Generator().manual_seed(beams)
    requests, entries = 3, 2
    state = torch.randint(0, 100, (entries, requests * beams + 4, *shape), generator=generator).to(dtype)
    slots = torch.randperm(requests * beams + 4, generator=generator)[:requests * beams].to(torch.int32)
    parents = torch.stack([torch.randperm(beams, generator=generator), torch.randint(0, beams, (beams,), generator=generator),
                           torch.arange(beams)]).to(torch.int32)
    got = state.to(DEVICE)
    ops.reorder_slots(got, slots.to(DEVICE), parents.to(DEVICE))
    want = state.clone()
    for r in range(requests):
        for b in range(beams):
            want[:, slots[r * beams + b]] = state[:, slots[r * beams + int(parents[r, b])]]
    assert torch.equal(got.cpu(), want)
    ops.check_errors()


@pytest.mark.parametrize("beams", [1, 3, 4, 8, 16, 32])
@pytest.mark.parametrize("page_shape,dtype", [((2, 16, 8), torch.bfloat16), ((3, 1, 2, 576), torch.uint8),
                                              ((5,), torch.uint8), ((1, 3), torch.float32)])
def test_pages(ops, beams, page_shape, dtype):
    """Requests of different lengths, pages given back, whole requests that do not move."""
    generator = torch.Generator().manual_seed(beams + 50)
    requests, width, page_size, outer = 4, 7, 16, 3
    starts, lengths = torch.tensor([0, 20, 48, 40]), torch.tensor([100, 33, 48, 112])
    pages = requests * beams * width + 2
    table = torch.randperm(pages, generator=generator)[:requests * beams * width].view(-1, width).to(torch.int32)
    table[0, 1] = -1
    table[-1, 3] = -1
    parents = torch.randint(0, beams, (requests, beams), generator=generator).to(torch.int32)
    storage = torch.randint(0, 100, (outer, pages, *page_shape), generator=generator).to(dtype)
    got = storage.to(DEVICE)
    on = lambda x: x.to(torch.int32).to(DEVICE)
    ops.reorder_pages(got, on(table), on(parents), on(starts), on(lengths), page_size=page_size)
    want = storage.clone()
    for r in range(requests):
        for b in range(beams):
            for block in range(int(starts[r]) // page_size, -(-int(lengths[r]) // page_size)):
                source, target = int(table[r * beams + int(parents[r, b]), block]), int(table[r * beams + b, block])
                if source >= 0 and target >= 0:
                    want[:, target] = storage[:, source]
    assert torch.equal(got.cpu(), want)
    ops.check_errors()


def test_places_outside_their_range(ops):
    """A parent, slot or page that there is not moves nothing and is told of; the others move."""
    state = torch.arange(6.0, device=DEVICE)[None, :, None].repeat(1, 1, 8)
    slots = torch.arange(6, dtype=torch.int32, device=DEVICE)
    bad = torch.tensor([[1, 0, 3], [-1, 2, 1]], dtype=torch.int32, device=DEVICE)
    ops.reorder_slots(state, slots, bad)
    assert state[0, :, 0].tolist() == [1.0, 0.0, 2.0, 3.0, 5.0, 4.0]
    with pytest.raises(KernelError, match="outside its range"):
        ops.check_errors()
    slots[1] = 6
    good = torch.tensor([[1, 0, 2], [0, 1, 2]], dtype=torch.int32, device=DEVICE)
    before = state.clone()
    ops.reorder_slots(state, slots, good)
    assert torch.equal(state, before)
    with pytest.raises(KernelError, match="outside its range"):
        ops.check_errors()
    table = torch.tensor([[0], [6], [2]], dtype=torch.int32, device=DEVICE)
    one = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=DEVICE)
    ends = torch.tensor([16], dtype=torch.int32, device=DEVICE)
    ops.reorder_pages(state, table, one, ends * 0, ends, page_size=16)
    before[0, 0] = before[0, 2]
    assert torch.equal(state, before)
    with pytest.raises(KernelError, match="outside its range"):
        ops.check_errors()
