"""What attention over packed pages hands to the kernels that read opened pages, without a GPU: a library that
writes down its launches, and a reader that writes down the step that it is given."""

import pytest
import torch

import plain_packed as plain
from mlx_one_b200.kernels.cuda_ops import CudaOps, KernelError
from mlx_one_b200.parts.base import PackedView, PagedKeyValues, PagedView, StepContext, packed_part_bytes


class Library:
    def mlxone_packed_unit_bytes(self, dim):
        return 2 * packed_part_bytes(dim)

    def mlxone_attention_mma_supports(self, dim, code):
        return int(code == 1 and dim % 16 == 0 and dim <= 128)

    def mlxone_open_factors(self, requests, heads, blocks, size):
        return 2 * requests * heads * 200


class Ops(CudaOps):
    """Launches are names and arguments in ``launched``; the readers' calls (queries, arguments) in ``read``."""

    def __init__(self):
        self.device, self.lib, self._sm_count = torch.device("cpu"), Library(), 148
        self.error_flag = torch.zeros(1, dtype=torch.int32)
        self._packed_cluster, self._device_index, self._packed_shapes = 8, 0, {}
        self.open_page, self.open_bytes, self.tensor_core_attention, self.launches = 64, 1 << 29, True, 0
        self.launched, self.read = [], []

    def _launch(self, name, *args):
        self.launched.append((name, args))

    def paged_attention(self, q, *, view, out=None, **how):
        if isinstance(view, PackedView):
            return super().paged_attention(q, view=view, out=out, **how)
        assert isinstance(view, PagedView)
        # (a row tells whose query it is and in which call it was answered)
        rows = q.reshape(how["ctx"].tokens, how["heads"], how["head_dim"])
        self.read.append((rows.clone(), view, how))
        got = (rows[:, :, :1] + 64 * len(self.read)).expand(-1, -1, how["head_dim"]).reshape(how["ctx"].tokens, -1).clone()
        if out is None:
            return got
        out.copy_(got)
        return out


def step(portions, histories, leading):
    as_int = lambda v: torch.tensor(v, dtype=torch.int32)
    starts = [sum(portions[:i]) for i in range(len(portions) + 1)]
    return StepContext(
        tokens=starts[-1], requests=len(portions), token_ids=as_int([0] * starts[-1]),
        positions=as_int([h + i for n, h in zip(portions, histories) for i in range(n)]),
        token_request=as_int([r for r, n in enumerate(portions) for _ in range(n)]), request_start=as_int(starts),
        history=as_int(histories), max_portion=max(portions), max_context=max(n + h for n, h in zip(portions, histories)),
        leading_single=leading)


def attend(ops, ctx, dtype, kv_heads=2, group=2, dim=32, width=8, **how):
    page = 16
    pages = plain.empty_pages(4, kv_heads, page, dim)
    view = PackedView(pages, torch.zeros((ctx.requests, width), dtype=torch.int32), page, PagedKeyValues(kv_heads, dim))
    q = torch.arange(ctx.tokens, dtype=torch.float32)[:, None, None].expand(-1, kv_heads * group, dim).to(dtype).contiguous()
    return ops.paged_attention(q, heads=kv_heads * group, kv_heads=kv_heads, head_dim=dim, scale=1.0, window=None,
                               ctx=ctx, view=view, **how)


@pytest.mark.parametrize("dtype,tensor_cores", [(torch.float32, True), (torch.float32, False), (torch.bfloat16, False)])
@pytest.mark.parametrize("portions,histories,leading", [([1, 1, 5, 3], [40, 7, 9, 0], 2), ([4, 2], [0, 30], 0)])
def test_a_row_goes_with_its_own_position_and_request(dtype, tensor_cores, portions, histories, leading):
    """Kernels that go by token find the rest's positions and requests beside the rest's queries: in 32 bits, and
    in bfloat16 without tensor cores, too."""
    ops, ctx = Ops(), step(portions, histories, leading)
    ops.tensor_core_attention = tensor_cores
    attend(ops, ctx, dtype)
    assert len(ops.read) == 1
    rows, view, how = ops.read[0]
    inner, rest = how["ctx"], len(portions) - leading
    assert inner.tokens == ctx.tokens - leading and inner.requests == rest and view.block_table.shape[0] == rest
    assert len(inner.positions) == len(inner.token_request) == inner.tokens
    assert torch.equal(inner.positions, ctx.positions[leading:])
    assert torch.equal(inner.token_request, ctx.token_request[leading:] - leading)
    assert 0 <= int(inner.token_request.min()) and int(inner.token_request.max()) < view.block_table.shape[0]
    assert rows[:, 0, 0].tolist() == list(range(leading, ctx.tokens))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("room,requests", [(1 << 29, 5), (1, 1), (2.5, 2), (11, 5)])
def test_opened_pages_stay_within_their_room(dtype, room, requests):
    """``open_bytes`` holds for all that is opened at a time, whatever of it is many: ``room`` key heads of one
    request allow ``requests`` requests at once, and as many key heads of these as there is room for. Every row is answered with its own request's keys."""
    portions, histories, leading = [1, 1, 3, 1, 5, 2, 4], [9, 70, 100, 0, 20, 6, 40], 2
    ops, ctx = Ops(), step(portions, histories, leading)
    ops.tensor_core_attention = False
    blocks, each = 2, 2 * 2 * 64 * 32 * torch.empty((), dtype=dtype).element_size()
    ops.open_bytes = int(room * each) if room < 1 << 29 else room
    out = torch.full((ctx.tokens, 8 * 32), -1.0, dtype=dtype)
    attend(ops, ctx, dtype, kv_heads=4, out=out)
    calls = 0
    for first in range(leading, len(portions), requests):
        count = min(requests, len(portions) - first)
        heads = max(min(int(room // count), 4), 1)
        for head in range(0, 4, heads):
            rows, view, how = ops.read[calls]
            inner, calls = how["ctx"], calls + 1
            assert view.kv.shape == (2, count * blocks, heads, 64, 32) and inner.requests == count
            assert view.kv.numel() * view.kv.element_size() <= max(ops.open_bytes, each)
            opening = [args for name, args in ops.launched if name == "mlxone_open_key_values"][calls - 1]
            assert opening[9:13] == (first, count, 4, head)
            mine = (ctx.token_request >= first) & (ctx.token_request < first + count)
            if inner.tokens != ctx.tokens:                   # (all of the rest at once: the rest by itself)
                mine = mine[leading:]
                assert mine.all() and count == len(portions) - leading
            skipped = ctx.tokens - inner.tokens
            assert torch.equal(inner.positions[mine], ctx.positions[skipped:][mine])
            assert torch.equal(inner.token_request[mine], ctx.token_request[skipped:][mine] - first)
            # (no row reads outside the table, and tokens of one request stay neighbours)
            assert 0 <= int(inner.token_request.min()) and int(inner.token_request.max()) < count
            assert (inner.token_request.diff() >= 0).all() and inner.positions.min() >= 0
            assert (inner.positions[~mine] == 0).all()
            if skipped == 0:
                assert torch.equal(inner.history, ctx.history[first:])
                assert torch.equal(inner.request_start, ctx.request_start[first:])
            for t in torch.nonzero(ctx.token_request.ge(first) & ctx.token_request.lt(first + count)).view(-1).tolist():
                got = out[t].view(8, 32)[2 * head:2 * (head + heads)]
                assert (got == t + 64 * calls).all(), (t, calls)
    assert calls == len(ops.read)
    assert (out[:leading] == -1).all()                       # (the single tokens' kernel's)


def test_room_for_the_keys_that_are_opened():
    """A long single token beside short portions: pages for the portions' keys only, where the step says how long they are."""
    portions, histories = [1, 20, 30], [5000, 0, 10]
    for rest, blocks in ((40, 1), (0, 79)):
        ops, ctx = Ops(), step(portions, histories, 1)
        ctx.rest_context = rest
        attend(ops, ctx, torch.float32, width=400)
        (_, view, how), = ops.read
        assert view.block_table.shape == (2, blocks) and how["ctx"].max_context == (rest or 5001)
    # single tokens whose scores are shaped are opened too
    ops, ctx = Ops(), step(portions, histories, 1)
    ctx.rest_context = 40
    attend(ops, ctx, torch.float32, width=400, score_cap=5.0)
    assert ops.read[0][1].block_table.shape == (3, 79)


def test_a_step_says_how_long_its_portions_are(tmp_path):
    """The runner's bound of the requests behind the leading single tokens."""
    from mlx_one_b200.cache import CacheManager
    from mlx_one_b200.engine.loading import load_model
    from mlx_one_b200.engine.runner import Runner, StepEntry
    from plain_ops import PlainOps
    from tiny_models import make_model_dir

    model = load_model(make_model_dir("A", tmp_path, dtype=torch.float32), "float32", "cpu", ops=PlainOps()).model
    cache = CacheManager(model.cache_needs, page_size=4, capacity_tokens=256, max_requests=4, dtype=torch.float32,
                         device="cpu")
    runner = Runner(model, cache)
    steps, forward = [], model.forward
    model.forward = lambda ctx: steps.append(ctx) or forward(ctx)
    for request in "abc":
        cache.open(request)
    runner.step([StepEntry("a", [3] * 40, (39,))])
    runner.step([StepEntry("a", [3], (0,)), StepEntry("b", [3] * 5, (4,)), StepEntry("c", [3] * 7, (6,))])
    runner.step([StepEntry("a", [3], (0,)), StepEntry("b", [3], (0,))])
    assert [(c.leading_single, c.rest_context, c.max_context) for c in steps] == [(0, 40, 40), (1, 7, 41), (2, 0, 42)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("leading", [0, 2])
def test_results_that_are_refused(dtype, leading):
    """A given ``out`` is as large as the result and of its type, over packed pages and over plain ones."""
    ctx = step([1, 1, 3], [4, 0, 9], leading)
    width = 4 * 32
    good = torch.zeros(5, width, dtype=dtype)
    attend(Ops(), ctx, dtype, out=good)
    other = torch.bfloat16 if dtype == torch.float32 else torch.float32
    for bad in (good[:4], good[:, :64].contiguous(), torch.zeros(5, 2 * width, dtype=dtype)[:, ::2], good.to(other),
                torch.zeros(6, width, dtype=dtype), good.view(5, 4, 32), good.view(-1), good.to("meta")):
        ops = Ops()
        with pytest.raises(KernelError, match="out must"):
            attend(ops, ctx, dtype, out=bad)
        plainly = PagedView(torch.zeros(2, 4, 2, 16, 32, dtype=dtype), torch.zeros((3, 8), dtype=torch.int32), 16,
                            PagedKeyValues(2, 32))
        with pytest.raises(KernelError, match="out must"):
            CudaOps.paged_attention(ops, torch.zeros(5, 4, 32, dtype=dtype), heads=4, kv_heads=2, head_dim=32, scale=1.0,
                                    window=None, ctx=ctx, view=plainly, out=bad)
        assert not ops.launched and not ops.read


def test_tables_with_too_few_rows():
    """Writing and reading back look a request's pages up in its row of the block table, as attention does."""
    ops, ctx = Ops(), step([2, 3], [0, 4], 0)
    pages, rows = plain.empty_pages(3, 2, 16, 32), torch.zeros(5, 64)
    for table, good in ((torch.zeros((1, 4), dtype=torch.int32), False), (torch.zeros((2, 4), dtype=torch.int32), True)):
        view = PackedView(pages, table, 16, PagedKeyValues(2, 32))
        for call in (lambda: ops.pack_key_values(rows, rows, ctx=ctx, view=view), lambda: ops.read_key_values(ctx=ctx, view=view)):
            if good:
                call()
            else:
                with pytest.raises(KernelError, match="a row for every request"):
                    call()
    assert len(ops.launched) == 2
