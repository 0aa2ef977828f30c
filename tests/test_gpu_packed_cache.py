"""A cache held in 4 bits: packing, reading back and attention over it, against plain_packed.py in 64 bits."""

import math

import pytest
import torch

import plain_packed as plain
from test_gpu_kernels import make_batch, ops  # noqa: F401  (fixture)
from mlx_one_b200.kernels import KernelError
from mlx_one_b200.parts.base import PackedView, PagedKeyValues

pytestmark = pytest.mark.gpu
DEVICE = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16


def rows_of(tokens, heads, dim, dtype, seed, spread=0.7):
    """Keys or values whose channels differ in size; some rows constant, some with few values (ties)."""
    generator = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, heads, dim, generator=generator) * torch.exp(spread * torch.randn(dim, generator=generator))
    if tokens > 2:
        x[1] = 0.3125                                        # no range at all
        x[2] = torch.randint(-15, 16, (heads, dim), generator=generator) / 4.0    # many quotients are ties
    return x.to(dtype)


def packed_case(heads, dim, page, portions, histories, dtype, seed=0, stale=0xFF):
    """A step, its packed pages filled with an earlier owner's bytes, and the histories packed plainly."""
    ctx, table, pages = make_batch(portions, histories, page, DEVICE, seed=seed)
    kv = plain.empty_pages(pages, heads, page, dim, fill=stale)       # (0xFF: codes of 15, NaN for steps)
    for r, (held, n) in enumerate(zip(histories, portions)):
        if held:
            plain.pack(kv, table.cpu(), page, range(held), [r] * held, rows_of(held, heads, dim, dtype, 10 * r + seed),
                       rows_of(held, heads, dim, dtype, 10 * r + seed + 5))
    return ctx, table, kv, PackedView(kv.to(DEVICE), table, page, PagedKeyValues(heads, dim))


CASES = [([1], [0]), ([1, 1, 1], [0, 15, 16]), ([16], [0]), ([16, 16], [16, 5]), ([40, 1, 7, 33], [3, 31, 0, 16]),
         ([1, 1, 50], [9, 47, 14]), ([2, 1, 1, 1, 17], [15, 8, 0, 63, 31])]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim,heads,page", [(32, 3, 16), (64, 2, 16), (64, 1, 64), (96, 2, 32), (128, 2, 128)])
@pytest.mark.parametrize("portions,histories", CASES)
def test_packing_and_reading(ops, dtype, dim, heads, page, portions, histories):
    """Byte for byte the plain form's, with every other byte as it was, and read back exactly."""
    ctx, table, kv, view = packed_case(heads, dim, page, portions, histories, dtype)
    inner = heads * dim
    wide = torch.zeros(ctx.tokens, 3 * inner + 8, dtype=dtype)
    wide[:, :inner] = rows_of(ctx.tokens, heads, dim, dtype, 71).view(ctx.tokens, -1)
    wide[:, inner + 8:2 * inner + 8] = rows_of(ctx.tokens, heads, dim, dtype, 72).view(ctx.tokens, -1)
    wide = wide.to(DEVICE)
    keys, values = wide[:, :inner], wide[:, inner + 8:2 * inner + 8]
    before = view.kv.clone()
    ops.pack_key_values(keys, values, ctx=ctx, view=view)
    plain.pack(kv, table.cpu(), page, ctx.positions.tolist(), ctx.token_request.tolist(),
               keys.cpu().view(-1, heads, dim), values.cpu().view(-1, heads, dim))
    assert torch.equal(view.kv.cpu(), kv)
    # rows whose addresses allow no wide loads
    shifted = torch.zeros(ctx.tokens, 2 * inner + 3, dtype=dtype, device=DEVICE)
    shifted[:, 1:inner + 1], shifted[:, inner + 1:2 * inner + 1] = keys, values
    again = PackedView(before, table, page, view.need)
    ops.pack_key_values(shifted[:, 1:inner + 1], shifted[:, inner + 1:2 * inner + 1], ctx=ctx, view=again)
    assert torch.equal(again.kv, view.kv)
    for out in (F32, BF16):
        got = ops.read_key_values(ctx=ctx, view=view, dtype=out)
        for which, rows in ((0, keys), (1, values)):
            code, step, low = zip(*(plain.quantized(rows.cpu().view(-1, heads, dim)[:, h]) for h in range(heads)))
            want = torch.stack([plain.values_of(*part) for part in zip(code, step, low)], 1)
            assert torch.equal(got[which].cpu(), want.float().to(out))
            # half a step, a step's own rounding, and the lowest value's
            span = rows.cpu().float().view(-1, heads, plain.groups_of(dim), dim // plain.groups_of(dim))
            bound = torch.stack(step, 1)[..., None] * (0.5 + 16 * 2.0 ** -8) + span.abs().amax(-1, keepdim=True) * 2.0 ** -8
            if out == F32:
                assert ((want.view_as(span) - span).abs() <= bound).all()
    ops.check_errors()


def test_steps_next_to_a_border(ops):
    """Ranges whose fifteenth is another bfloat16 by division than by a product with the inverse: the product's."""
    span = torch.rand(1 << 23, generator=torch.Generator().manual_seed(0)) * 8
    border = span[(span / 15).bfloat16() != (span * torch.tensor(1 / 15)).bfloat16()]
    assert len(border) > 20
    n = len(border)
    ctx, table, kv, view = packed_case(1, 64, 16, [n], [0], F32, stale=0)
    x = torch.rand(n, 1, 64, generator=torch.Generator().manual_seed(1)) * border.view(n, 1, 1)
    x[:, 0, 3], x[:, 0, 60] = 0.0, border
    plain.pack(kv, table.cpu(), 16, range(n), [0] * n, x, x)
    x = x.view(n, 64).to(DEVICE)
    ops.pack_key_values(x, x, ctx=ctx, view=view)
    assert torch.equal(view.kv.cpu(), kv)
    _, steps, _ = plain.quantized(x.cpu())
    assert torch.equal(steps[:, 0].to(DEVICE), (x.amax(-1) / 15).bfloat16().double())
    ops.check_errors()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_values_that_are_not_finite(ops, dtype):
    """A group with NaN, infinity or a range that no number holds reads as NaN; its neighbours do not."""
    ctx, table, kv, view = packed_case(2, 128, 16, [5], [0], dtype, stale=0)
    x = rows_of(5, 2, 128, dtype, 3)
    x[0, 0, 7], x[1, 1, 70], x[2, 0, 127] = math.nan, math.inf, -math.inf
    x[3, 1, 64], x[3, 1, 65] = 3e38, -3e38
    x[4, 0, :64], x[4, 0, 1] = 1e-38, 2e-38                  # a step below the normal numbers
    x = x.to(DEVICE)
    ops.pack_key_values(x.view(5, -1), x.view(5, -1), ctx=ctx, view=view)
    plain.pack(kv, table.cpu(), 16, range(5), [0] * 5, x.cpu(), x.cpu())
    assert torch.equal(view.kv.cpu(), kv)
    keys, values = ops.read_key_values(ctx=ctx, view=view, dtype=F32)
    bad = torch.isnan(keys).view(5, 2, 2, 64)
    want = torch.zeros(5, 2, 2, dtype=torch.bool)
    want[0, 0, 0] = want[1, 1, 1] = want[2, 0, 1] = want[3, 1, 1] = True
    assert torch.equal(bad.all(-1).cpu(), want) and torch.equal(bad.any(-1).cpu(), want)
    assert torch.equal(torch.isnan(values), torch.isnan(keys))


def test_pages_that_are_missing(ops):
    """A token without a page is told of and written nowhere; the others are written."""
    ctx, table, kv, view = packed_case(1, 64, 16, [3, 20], [14, 0], BF16, stale=0)
    table[0, 0], table[1, 1] = -1, view.kv.shape[0]          # none; one behind the last
    before = view.kv.clone()
    x = rows_of(ctx.tokens, 1, 64, BF16, 1).view(ctx.tokens, 64).to(DEVICE)
    ops.pack_key_values(x, x, ctx=ctx, view=view)
    with pytest.raises(KernelError, match="no page"):
        ops.check_errors()
    ops.read_key_values(ctx=ctx, view=view)
    with pytest.raises(KernelError, match="no page"):
        ops.check_errors()
    touched = (view.kv != before).flatten(1).any(1)
    kept = torch.zeros_like(touched)
    kept[table[0, 1].long()] = kept[table[1, 0].long()] = True
    assert not (touched & ~kept).any() and touched[table[1, 0].long()]


# ------------------------------------------------------------------ attention


def bound_of(view_values, q, scale, dim, dtype, keys):
    """How far an output may be off (absolute). k, v: keys and values as they read, float64 [keys, dim]; every
    rounding counted at its largest: scores are sums of dim products of |q| and 128 + code (bfloat16) or
    code - 8 (float32, in parts of their own), each addition off by 2^-23 of the sum where a tensor core cuts; a
    weight is off by twice a score's error, 2^-22 for the exponential, and bfloat16's 2^-8; the values' sums
    are of 128 + code (or code - 8) over keys / 16 additions and the merges; the result is rounded once."""
    k, v = view_values
    step_k, step_v = k.abs().max() / 4, v.abs().max() / 4    # (steps are below: 15 of them span a range)
    q_sum = q.double().abs().sum(-1).max()
    offset = 143.0 if dtype == BF16 else 8.0
    additions = dim / 16 * (1 if dtype == BF16 else 3) + 8
    score = scale * q_sum * (offset * step_k + k.abs().max()) * additions * 2.0 ** -23
    weights = 2 * score + 2.0 ** -22 * 4 + (2.0 ** -8 if dtype == BF16 else 0.0)
    sums = (offset * step_v + v.abs().max()) * (keys / 16 + 40) * 2.0 ** -23
    out = v.abs().max() * (2.0 ** -8 if dtype == BF16 else 2.0 ** -24)
    opened = (2.0 ** -8 * v.abs().max() + 2 * 2.0 ** -8 * scale * q_sum * k.abs().max() * v.abs().max()
              if dtype == BF16 else 0.0)                     # portions read keys and values as bfloat16
    return dict(single=float(weights * 2 * v.abs().max() + sums + out),
                portion=float(weights * 2 * v.abs().max() + sums + out + opened))


def attention_case(ops, dtype, heads, kv_heads, dim, page, portions, histories, window=0, with_sinks=False, seed=0,
                   leading=0, missing=()):
    ctx, table, kv, view = packed_case(kv_heads, dim, page, portions, histories, dtype, seed)
    ctx.leading_single = leading
    generator = torch.Generator().manual_seed(seed + 1)
    q = torch.randn(ctx.tokens, heads, dim, generator=generator).to(dtype)
    keys = rows_of(ctx.tokens, kv_heads, dim, dtype, seed + 2, 0.3)
    values = rows_of(ctx.tokens, kv_heads, dim, dtype, seed + 3, 0.3)
    sinks = torch.randn(heads, generator=generator) if with_sinks else None
    plain.pack(kv, table.cpu(), page, ctx.positions.tolist(), ctx.token_request.tolist(), keys, values)
    ops.pack_key_values(keys.view(ctx.tokens, -1).to(DEVICE), values.view(ctx.tokens, -1).to(DEVICE), ctx=ctx, view=view)
    for r, b in missing:
        table[r, b] = -1
    scale = dim ** -0.5
    got = ops.paged_attention(q.to(DEVICE), heads=heads, kv_heads=kv_heads, head_dim=dim, scale=scale,
                              window=window or None, ctx=ctx, view=view,
                              sinks=None if sinks is None else sinks.to(DEVICE))
    ops.check_errors()
    got = got.view(ctx.tokens, heads, dim).cpu().double()
    want = plain.attend(q, kv, table.cpu(), page, portions, histories, heads, kv_heads, scale, window, sinks)
    t = 0
    for r, (n, held) in enumerate(zip(portions, histories)):
        both = plain.read(kv, table.cpu(), page, r, held + n, dim)
        both = torch.where(torch.isnan(both), 0.0, both)
        bound = bound_of(both, q[t:t + n], scale, dim, dtype, held + n)
        single = r < leading or max(portions) == 1
        off = (got[t:t + n] - want[t:t + n]).abs().max()
        assert off <= bound["single" if single else "portion"], (r, float(off), bound)
        t += n
    return got


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [
    (8, 2, 64, 16), (4, 4, 32, 16), (12, 1, 96, 32), (10, 2, 128, 64), (3, 1, 64, 128), (16, 2, 64, 16)])
@pytest.mark.parametrize("histories", [[0], [14, 15, 16, 31, 32], [300, 0, 5, 127], [1500, 33]])
def test_single_tokens(ops, dtype, heads, kv_heads, dim, page, histories):
    """Lengths around the units' and tiles' edges, one key, more keys than one part; 1 to 12 heads a key head."""
    attention_case(ops, dtype, heads, kv_heads, dim, page, [1] * len(histories), histories)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("window", [1, 15, 16, 33, 100, 5000])
@pytest.mark.parametrize("with_sinks", [False, True])
def test_windows_and_sinks(ops, dtype, window, with_sinks):
    attention_case(ops, dtype, 8, 2, 64, 16, [1] * 5, [0, 31, 64, 200, 333], window=window, with_sinks=with_sinks)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,kv_heads,dim,page,window,with_sinks", [
    (8, 2, 64, 16, 0, False), (6, 2, 32, 32, 0, True), (4, 1, 128, 16, 40, False), (4, 2, 96, 64, 0, False),
    (8, 2, 64, 64, 50, True)])
@pytest.mark.parametrize("portions,histories,leading", [
    ([5], [0], 0), ([1, 1, 37], [40, 9, 0], 2), ([70, 1, 16], [3, 100, 200], 0), ([1, 130], [15, 65], 1)])
def test_portions(ops, dtype, heads, kv_heads, dim, page, window, with_sinks, portions, histories, leading):
    """Portions of prompts alone, and behind single tokens at the head of the step."""
    attention_case(ops, dtype, heads, kv_heads, dim, page, portions, histories, window=window, with_sinks=with_sinks,
                   leading=leading)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_portions_in_parts(ops, dtype):
    """More than the scratch holds: the key heads one after the other, the same numbers."""
    held = ops.open_bytes
    whole = attention_case(ops, dtype, 12, 3, 64, 16, [1, 40, 9], [20, 33, 0], leading=1)
    try:
        for size in (1, 2 * 2 * 2 * 128 * 64 * 4):
            ops.open_bytes = size
            assert torch.equal(attention_case(ops, dtype, 12, 3, 64, 16, [1, 40, 9], [20, 33, 0], leading=1), whole)
    finally:
        ops.open_bytes = held


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_nothing_to_see(ops, dtype):
    """Keys without a page are not seen; a row that sees nothing is zeros, or what its sink leaves: zeros."""
    attention_case(ops, dtype, 8, 2, 64, 16, [1] * 3, [40, 70, 5], missing=[(0, 0), (1, 1), (1, 4)])
    attention_case(ops, dtype, 8, 2, 64, 16, [1] * 3, [40, 70, 5], missing=[(2, 0)], with_sinks=True)
    got = attention_case(ops, dtype, 8, 2, 64, 16, [1] * 3, [40, 70, 5], missing=[(2, 0), (0, 0), (0, 1), (0, 2)])
    assert (got[0] == 0).all() and (got[2] == 0).all()
    # a position ahead of the first key: no key at all
    ctx, table, _, view = packed_case(2, 64, 16, [1, 1], [20, 0], dtype)
    ctx.positions[1] = -1
    q = torch.randn(2, 8, 64, device=DEVICE).to(dtype)
    got = ops.paged_attention(q, heads=8, kv_heads=2, head_dim=64, scale=0.125, window=None, ctx=ctx, view=view)
    assert (got[1] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_what_is_not_a_number_stays_where_it_is(ops, dtype):
    """A key that is NaN spoils the heads that see it and no other; one that nobody sees spoils nothing."""
    ctx, table, kv, view = packed_case(2, 64, 16, [1, 1], [50, 50], dtype, stale=0)
    nan = torch.full((50, 2, 64), math.nan, dtype=dtype)
    plain.pack(kv, table.cpu(), 16, [3], [0], nan[:1, :1].clone(), rows_of(1, 1, 64, dtype, 1))     # head 0 of request 0
    view.kv.copy_(kv)
    x = rows_of(2, 2, 64, dtype, 9).view(2, -1).to(DEVICE)
    ops.pack_key_values(x, x, ctx=ctx, view=view)
    q = torch.randn(2, 8, 64, device=DEVICE).to(dtype)
    call = dict(heads=8, kv_heads=2, head_dim=64, scale=0.125, ctx=ctx, view=view)
    got = torch.isnan(ops.paged_attention(q, window=None, **call)).view(2, 8, 64)
    assert got[0, :4].all() and not got[0, 4:].any() and not got[1].any()
    assert not torch.isnan(ops.paged_attention(q, window=40, **call)).any()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_many_parts_and_large_scores(ops, dtype):
    """More parts than a cluster merges; scores of hundreds, rising and falling along the keys."""
    heads, dim, held = 4, 64, 40000
    ctx, table, pages = make_batch([1], [held], 64, DEVICE)
    assert ops.packed_splits(1, heads, 1, dim, held + 1, 0) > 8
    view = PackedView(torch.zeros(pages, 1, 4, 2, 576, dtype=torch.uint8, device=DEVICE), table, 64, PagedKeyValues(1, dim))
    generator = torch.Generator(DEVICE).manual_seed(1)
    all_, _, _ = make_batch([held + 1], [0], 64, DEVICE)
    along = torch.linspace(-1, 1, held + 1, device=DEVICE)[:, None]
    keys = (torch.randn(held + 1, dim, generator=generator, device=DEVICE) + 8 * along).to(dtype)
    values = torch.randn(held + 1, dim, generator=generator, device=DEVICE).to(dtype)
    ops.pack_key_values(keys, values, ctx=all_, view=view)
    k, v = (x[:, 0].double() for x in ops.read_key_values(ctx=all_, view=view, dtype=F32))
    for sign in (1.0, -1.0, 0.0):
        q = (torch.randn(1, heads, dim, generator=generator, device=DEVICE) + 4 * sign).to(dtype)
        got = ops.paged_attention(q, heads=heads, kv_heads=1, head_dim=dim, scale=0.125, window=None, ctx=ctx, view=view)
        want = torch.softmax(q[0].double() @ k.T * 0.125, -1) @ v
        bound = bound_of((k, v), q[0], 0.125, dim, dtype, held + 1)["single"]
        assert (got.view(heads, dim).double() - want).abs().max() <= bound
    ops.check_errors()


def test_a_cache_beyond_32_bit_offsets(ops):
    """Pages behind the first 2^32 bytes."""
    heads, dim, page = 8, 64, 128
    each = heads * 8 * 1152
    pages = (1 << 32) // each + 40
    kv = torch.zeros(pages, heads, 8, 2, 576, dtype=torch.uint8, device=DEVICE)
    ctx, table, count = make_batch([300], [0], page, DEVICE)
    far = torch.where(table >= 0, table + (pages - count), table)
    x = rows_of(300, heads, dim, BF16, 4).view(300, -1).to(DEVICE)
    one, small = PackedView(kv, far, page, PagedKeyValues(heads, dim)), kv.new_zeros(count, heads, 8, 2, 576)
    other = PackedView(small, table, page, PagedKeyValues(heads, dim))
    q = torch.randn(300, 16, dim, device=DEVICE).bfloat16()
    last, _, _ = make_batch([1], [299], page, DEVICE)
    results = []
    for view in (one, other):
        ops.pack_key_values(x, x, ctx=ctx, view=view)
        call = dict(heads=16, kv_heads=heads, head_dim=dim, scale=0.125, window=None, view=view)
        results.append([*ops.read_key_values(ctx=ctx, view=view), ops.paged_attention(q, ctx=ctx, **call),
                        ops.paged_attention(q[:1], ctx=last, **call)])
    for a, b in zip(*results):
        assert torch.equal(a, b)
    ops.check_errors()


def test_replayed_and_on_another_stream(ops):
    """A captured step with other contents, and a step on a stream of its own, give a plain call's bits."""
    ctx, table, _, view = packed_case(2, 64, 16, [1, 1, 20], [70, 3, 33], BF16, stale=0)
    ctx.leading_single = 2
    generator = torch.Generator(DEVICE).manual_seed(5)
    new = lambda: torch.randn(22, 8 * 64, generator=generator, device=DEVICE).bfloat16()
    q, rows = new(), new()

    def step():
        ops.pack_key_values(rows[:, :128], rows[:, 128:256], ctx=ctx, view=view)
        return ops.paged_attention(q.view(22, 8, 64), heads=8, kv_heads=2, head_dim=64, scale=0.125, window=None,
                                   ctx=ctx, view=view)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(3):
        q.copy_(new())
        rows.copy_(new())
        graph.replay()
        replayed = captured.clone()
        assert torch.equal(step(), replayed)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = step()
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(other, replayed)
    ops.check_errors()


def test_shaped_scores_over_packed_pages(ops):
    """Caps, slopes, chunks and first positions behind a window: the opened pages' kernels."""
    from mlx_one_b200.parts.base import PagedView

    for portions, histories in (([1, 1], [40, 90]), ([30, 1], [50, 7])):
        for dtype in (BF16, F32):
            ctx, table, kv, view = packed_case(2, 64, 16, portions, histories, dtype, stale=0)
            x = rows_of(ctx.tokens, 2, 64, dtype, 9).view(ctx.tokens, -1).to(DEVICE)
            ops.pack_key_values(x, x, ctx=ctx, view=view)
            plainly = torch.zeros(2, view.kv.shape[0], 2, 16, 64, dtype=dtype, device=DEVICE)
            for r, (n, held) in enumerate(zip(portions, histories)):
                both = plain.read(view.kv.cpu(), table.cpu(), 16, r, held + n, 64).to(dtype).to(DEVICE)
                for p in range(held + n):
                    plainly[:, table[r, p // 16].long(), :, p % 16] = both[:, p]
            q = torch.randn(ctx.tokens, 8, 64, device=DEVICE).to(dtype)
            slopes = torch.linspace(0.01, 0.3, 8, device=DEVICE)
            for how in (dict(score_cap=20.0), dict(score_cap=5.0, slopes=slopes, least_slope=0.01), dict(chunk=32),
                        dict(window=24, keep_first=5)):
                call = dict(heads=8, kv_heads=2, head_dim=64, scale=0.125, window=None, ctx=ctx)
                got = ops.paged_attention(q, **{**call, **how}, view=view)
                want = ops.paged_attention(q, **{**call, **how}, view=PagedView(plainly, table, 16, view.need))
                # (both within 2^-8 of a weight and of the result, values below 4.2)
                torch.testing.assert_close(got.float(), want.float(), atol=0.07 if dtype == BF16 else 1e-4, rtol=0)
    ops.check_errors()


@pytest.mark.parametrize("dim,page", [(64, 16), (96, 32), (128, 64), (32, 16)])
@pytest.mark.parametrize("size", [1e-30, 1.0, 2e4, 1e30])
def test_portions_of_values_of_any_size(ops, dim, page, size):
    """Values that half-precision by itself could not hold: opened times a power of two of their request and head."""
    portions, histories = [40, 21], [30, 100]
    ctx, table, kv, view = packed_case(2, dim, page, portions, [0, 0], BF16, stale=0)
    whole, _, _ = make_batch([70, 121], [0, 0], page, DEVICE)
    ctx, table, pages = make_batch(portions, histories, page, DEVICE)
    view = PackedView(torch.full((pages, 2, page // 16, 2, plain.part_bytes(dim)), 0xFF, dtype=torch.uint8, device=DEVICE),
                      table, page, PagedKeyValues(2, dim))
    keys = rows_of(191, 2, dim, BF16, 3, 0.3)
    values = rows_of(191, 2, dim, F32, 4, 0.3)
    values[:, 1] *= 1e3                                       # a head's values are its own matter
    values = (values * size).to(BF16)
    ops.pack_key_values(keys.view(191, -1).to(DEVICE), values.view(191, -1).to(DEVICE), ctx=whole, view=view)
    q = torch.randn(61, 4, dim, generator=torch.Generator().manual_seed(1)).to(BF16)
    got = ops.paged_attention(q.to(DEVICE), heads=4, kv_heads=2, head_dim=dim, scale=dim ** -0.5, window=None, ctx=ctx,
                              view=view).view(61, 4, dim).cpu().double()
    want = plain.attend(q, view.kv.cpu(), table.cpu(), page, portions, histories, 4, 2, dim ** -0.5)
    t = 0
    for r, (n, held) in enumerate(zip(portions, histories)):
        both = plain.read(view.kv.cpu(), table.cpu(), page, r, held + n, dim)
        for h in range(2):
            bound = bound_of(both[:, :, h], q[t:t + n], dim ** -0.5, dim, BF16, held + n)["portion"]
            assert (got[t:t + n, 2 * h:2 * h + 2] - want[t:t + n, 2 * h:2 * h + 2]).abs().max() <= bound, (r, h)
        t += n
    ops.check_errors()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim,window", [(64, 0), (96, 0), (128, 30), (64, 50)])
@pytest.mark.parametrize("of_values", [False, True])
def test_what_is_not_a_number_in_a_portion(ops, dtype, dim, window, of_values):
    """Queries ahead of a key that is none, other heads' and other requests' get their numbers; the ones that see it do not."""
    ctx, table, kv, view = packed_case(2, dim, 16, [60, 20], [0, 0], dtype, stale=0)
    keys, values = rows_of(80, 2, dim, dtype, 1, 0.3), rows_of(80, 2, dim, dtype, 2, 0.3)
    (values if of_values else keys)[17, 1, 5] = math.nan
    ops.pack_key_values(keys.view(80, -1).to(DEVICE), values.view(80, -1).to(DEVICE), ctx=ctx, view=view)
    q = torch.randn(80, 6, dim, device=DEVICE).to(dtype)
    got = ops.paged_attention(q, heads=6, kv_heads=2, head_dim=dim, scale=dim ** -0.5, window=window or None, ctx=ctx,
                              view=view).view(80, 6, dim)
    spoilt = torch.isnan(got).any(-1).cpu()
    sees = torch.zeros(80, 6, dtype=torch.bool)
    sees[17:min(17 + window, 60) if window else 60, 3:] = True
    assert torch.equal(spoilt, sees)
    assert torch.isfinite(got.float()[~sees.to(DEVICE)]).all()
    ops.check_errors()


@pytest.mark.parametrize("dim,page", [(64, 16), (96, 32), (128, 64), (32, 16)])
@pytest.mark.parametrize("of_keys,of_queries", [(1e-30, 1e30), (1e-30, 1e-30), (1.0, 1.0), (1e5, 1e-5), (1e30, 1e-30)])
@pytest.mark.parametrize("window", [0, 24])
def test_portions_of_keys_and_queries_of_any_size(ops, dim, page, of_keys, of_queries, window):
    """Keys and queries beyond half-precision's range: times a power of two of their head's, and of their row's."""
    portions, histories = [40, 21], [30, 100]
    whole, _, _ = make_batch([70, 121], [0, 0], page, DEVICE)
    ctx, table, pages = make_batch(portions, histories, page, DEVICE)
    view = PackedView(torch.full((pages, 2, page // 16, 2, plain.part_bytes(dim)), 0xFF, dtype=torch.uint8, device=DEVICE),
                      table, page, PagedKeyValues(2, dim))
    keys = rows_of(191, 2, dim, F32, 3, 0.3)
    keys[:, 1] *= 1e-3                                        # a head's keys are its own matter
    keys = (keys * of_keys).to(BF16)
    values = rows_of(191, 2, dim, BF16, 4, 0.3)
    ops.pack_key_values(keys.view(191, -1).to(DEVICE), values.view(191, -1).to(DEVICE), ctx=whole, view=view)
    q = (torch.randn(61, 4, dim, generator=torch.Generator().manual_seed(1)) * of_queries)
    q[:, 2:] *= 1e3
    q = q.to(BF16)
    got = ops.paged_attention(q.to(DEVICE), heads=4, kv_heads=2, head_dim=dim, scale=dim ** -0.5, window=window or None,
                              ctx=ctx, view=view).view(61, 4, dim).cpu().double()
    want = plain.attend(q, view.kv.cpu(), table.cpu(), page, portions, histories, 4, 2, dim ** -0.5, window=window)
    t = 0
    for r, (n, held) in enumerate(zip(portions, histories)):
        both = plain.read(view.kv.cpu(), table.cpu(), page, r, held + n, dim)
        for h in range(2):
            bound = bound_of(both[:, :, h], q[t:t + n, 2 * h:2 * h + 2], dim ** -0.5, dim, BF16, held + n)["portion"]
            assert (got[t:t + n, 2 * h:2 * h + 2] - want[t:t + n, 2 * h:2 * h + 2]).abs().max() <= bound, (r, h)
        t += n
    ops.check_errors()


@pytest.mark.parametrize("dim,page", [(64, 16), (96, 32), (128, 64), (32, 16)])
@pytest.mark.parametrize("of_keys,of_queries,of_values", [(1e-30, 1e30, 1e-30), (1e-30, 1e-30, 1e30), (1e5, 1e-5, 2e4),
                                                          (1e30, 1e-30, 1.0)])
@pytest.mark.parametrize("dtype,window", [(BF16, 0), (BF16, 24), (F32, 0)])
def test_single_tokens_of_any_size(ops, dim, page, of_keys, of_queries, of_values, dtype, window):
    """Keys, queries and values beyond half-precision's range, a head's keys and values its own matter."""
    histories = [0, 30, 300]
    lengths = [h + 1 for h in histories]
    whole, _, _ = make_batch(lengths, [0] * 3, page, DEVICE)
    ctx, table, pages = make_batch([1] * 3, histories, page, DEVICE)
    view = PackedView(torch.full((pages, 2, page // 16, 2, plain.part_bytes(dim)), 0xFF, dtype=torch.uint8, device=DEVICE),
                      table, page, PagedKeyValues(2, dim))
    keys, values = rows_of(333, 2, dim, F32, 3, 0.3), rows_of(333, 2, dim, F32, 4, 0.3)
    keys[:, 1] *= 1e-3
    values[:, 1] *= 1e3
    keys, values = (keys * of_keys).to(dtype), (values * of_values).to(dtype)
    ops.pack_key_values(keys.view(333, -1).to(DEVICE), values.view(333, -1).to(DEVICE), ctx=whole, view=view)
    q = torch.randn(3, 4, dim, generator=torch.Generator().manual_seed(1)) * of_queries
    q[:, 2:] *= 1e3
    q = q.to(dtype)
    got = ops.paged_attention(q.to(DEVICE), heads=4, kv_heads=2, head_dim=dim, scale=dim ** -0.5, window=window or None,
                              ctx=ctx, view=view).view(3, 4, dim).cpu().double()
    want = plain.attend(q, view.kv.cpu(), table.cpu(), page, [1] * 3, histories, 4, 2, dim ** -0.5, window=window)
    for r, held in enumerate(lengths):
        both = plain.read(view.kv.cpu(), table.cpu(), page, r, held, dim)
        for h in range(2):
            bound = bound_of(both[:, :, h], q[r, 2 * h:2 * h + 2], dim ** -0.5, dim, dtype, held)["single"]
            assert (got[r, 2 * h:2 * h + 2] - want[r, 2 * h:2 * h + 2]).abs().max() <= bound, (r, h)
    ops.check_errors()
