"""Attention over a cache held in 4 bits within the bounds of the roundings that its kernels have (packed_bounds.py),
each bound a small part of the output that it is about."""

import pytest
import torch

import packed_bounds
import plain_packed as plain
from test_gpu_kernels import make_batch, ops  # noqa: F401  (fixture)
from test_gpu_packed_cache import rows_of
from mlx_one_b200.kernels import KernelError
from mlx_one_b200.parts.base import PackedView, PagedKeyValues

pytestmark = pytest.mark.gpu
DEVICE, F32, BF16 = "cuda:0", torch.float32, torch.bfloat16


def attention_case(ops, heads, kv_heads, dim, page, portions, histories, forms, *, leading=0, seed=0, of_keys=1.0,
                   of_queries=1.0, of_values=1.0, share=None, dtype=BF16, rest_context=0, **how):
    """Keys and values packed plainly; a kernel's output, which is returned, against the exact one. ``share``: see
    packed_bounds.check."""
    ctx, table, pages = make_batch(portions, histories, page, DEVICE, seed=seed)
    ctx.leading_single, ctx.rest_context = leading, rest_context
    lengths = [h + n for h, n in zip(histories, portions)]
    kv = plain.empty_pages(pages, kv_heads, page, dim, fill=0xFF)       # (an earlier owner's NaN)
    for r, n in enumerate(lengths):
        both = [rows_of(n, kv_heads, dim, torch.float32, 10 * r + seed + 5 * which, 0.3) for which in (0, 1)]
        plain.pack(kv, table.cpu(), page, range(n), [r] * n, (both[0] * of_keys).to(dtype), (both[1] * of_values).to(dtype))
    q = (torch.randn(ctx.tokens, heads, dim, generator=torch.Generator().manual_seed(seed + 1)) * of_queries).to(dtype)
    want, bound, variance = packed_bounds.attend(q, kv, table.cpu(), page, portions, histories, heads, kv_heads, dim ** -0.5, forms,
                                                 **how)
    call = dict(how, scale=dim ** -0.5, ctx=ctx, view=PackedView(kv.to(DEVICE), table, page, PagedKeyValues(kv_heads, dim)))
    if "cap" in call:
        call["score_cap"] = call.pop("cap")
    if call.get("slopes") is not None:
        call["least_slope"] = float(call["slopes"].min())
    call = {k: v.to(DEVICE) if isinstance(v, torch.Tensor) else v for k, v in call.items()}
    got = ops.paged_attention(q.to(DEVICE), heads=heads, kv_heads=kv_heads, head_dim=dim,
                              **{"window": None, **call}).view(ctx.tokens, heads, dim).cpu().double()
    ops.check_errors()
    packed_bounds.check(got, want, bound, portions, share or (0.25 if {"bfloat16", "shaped"} & set(forms) else 0.06))
    by_token = [form for n, form in zip(portions, forms) for _ in range(n)]
    for form in {"codes", "half"} & set(forms):
        rows = torch.tensor([f == form for f in by_token])
        packed_bounds.check_mean(got[rows], want[rows], variance[rows], heads // kv_heads)
    return got


@pytest.mark.parametrize("heads,kv_heads,dim,page", [(8, 2, 64, 16), (12, 3, 32, 64), (4, 1, 128, 16), (6, 2, 96, 32)])
@pytest.mark.parametrize("portions,histories,leading", [([1, 1, 37, 5], [40, 9, 0, 130], 2), ([16, 1], [100, 30], 0)])
@pytest.mark.parametrize("cap", [0.0, 5.0])
def test_without_tensor_cores(ops, heads, kv_heads, dim, page, portions, histories, leading, cap):
    """The general kernel, which goes by token, over opened pages: behind single tokens at the head of the step too."""
    held = ops.tensor_core_attention
    forms = ["codes"] * (0 if cap else leading)
    forms += ["bfloat16"] * (len(portions) - len(forms))
    try:
        ops.tensor_core_attention = False
        attention_case(ops, heads, kv_heads, dim, page, portions, histories, forms, leading=leading,
                       **(dict(cap=cap) if cap else {}))
    finally:
        ops.tensor_core_attention = held


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("how,block,told", [
    (dict(), 0, True), (dict(), 2, True), (dict(), 3, False), (dict(window=17), 0, False), (dict(window=18), 0, True),
    (dict(window=17, keep_first=1), 0, True), (dict(window=1, keep_first=16), 1, False), (dict(chunk=32), 1, False),
    (dict(chunk=64), 1, True), (dict(score_cap=5.0), 1, True)])
def test_a_key_of_a_portion_without_a_page_is_told_of(ops, dtype, how, block, told):
    """Opened pages hold zeros there, which their readers would take for a key: an error, unless no token of the
    portion sees it. (Positions 32 to 39 behind 32 keys in pages of 16: the first sees back to 32 - window + 1.)"""
    ctx, table, pages = make_batch([1, 8], [40, 32], 16, DEVICE)
    ctx.leading_single = 1
    view = PackedView(torch.zeros(pages, 2, 1, 2, 576, dtype=torch.uint8, device=DEVICE), table, 16, PagedKeyValues(2, 64))
    q = torch.randn(9, 4, 64, device=DEVICE).to(dtype)
    call = {**dict(heads=4, kv_heads=2, head_dim=64, scale=0.125, window=None, ctx=ctx, view=view), **how}
    ops.paged_attention(q, **call)
    ops.check_errors()                                       # (nothing is missing yet)
    table[1, block] = -1
    ops.paged_attention(q, **call)
    if told:
        with pytest.raises(KernelError, match="no page"):
            ops.check_errors()
    else:
        ops.check_errors()
    # a single token's key is not seen, without a word; nor are the keys of a request that brings no token
    if "window" not in how and "chunk" not in how and "score_cap" not in how:
        table[1, block] = pages - 1
        table[0, 0] = -1
        ctx.request_start[2] = 1
        table[1, 0] = -1
        ops.paged_attention(q, **call)
        ops.check_errors()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_keys_behind_the_bound_are_told_of(ops, dtype):
    """A step whose ``max_context`` is less than what the device's numbers say."""
    ctx, table, pages = make_batch([8], [122], 16, DEVICE)
    view = PackedView(torch.zeros(pages, 2, 1, 2, 576, dtype=torch.uint8, device=DEVICE), table, 16, PagedKeyValues(2, 64))
    q = torch.randn(8, 4, 64, device=DEVICE).to(dtype)
    call = dict(heads=4, kv_heads=2, head_dim=64, scale=0.125, window=None, ctx=ctx, view=view)
    ops.paged_attention(q, **call)
    ops.check_errors()
    ctx.max_context = 128                                    # (two opened pages of 64; position 129 is in the third)
    ops.paged_attention(q, **call)
    with pytest.raises(KernelError, match="no page"):
        ops.check_errors()


SLOPES = torch.linspace(0.01, 0.3, 6)


@pytest.mark.parametrize("dtype,tensor_cores", [(BF16, True), (BF16, False), (F32, True)])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64)])
@pytest.mark.parametrize("how", [dict(), dict(window=24, sinks=torch.linspace(-1, 1, 6)), dict(window=24, keep_first=5),
                                 dict(chunk=32), dict(cap=5.0, slopes=SLOPES)])
@pytest.mark.parametrize("room", [1, 2 * 2 * 2 * 64 * 128 * 4])
def test_some_requests_after_the_others(ops, dtype, tensor_cores, dim, page, how, room):
    """More than the scratch holds with one key head of every request. (``room``: one request's key head at a time, or a few.)"""
    portions, histories, leading = [1, 3, 40, 1, 9], [20, 33, 0, 64, 70], 1
    form = "float32" if dtype == F32 else "bfloat16" if not tensor_cores else "shaped" if "cap" in how else "half"
    forms = [form] * 5
    if dtype == BF16 and "cap" not in how and "keep_first" not in how:
        forms[0] = "codes"
    held = ops.open_bytes, ops.tensor_core_attention
    try:
        ops.open_bytes, ops.tensor_core_attention = room, tensor_cores
        attention_case(ops, 6, 2, dim, page, portions, histories, forms, leading=leading, dtype=dtype, **how)
    finally:
        ops.open_bytes, ops.tensor_core_attention = held


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_some_requests_after_the_others_behind_many_keys(ops, dtype):
    """Few rows over many keys, which are cut into parts with a merge of their own; a captured call's bits."""
    portions, histories = [1, 5, 3, 2], [300, 2900, 1100, 2500]
    held = ops.open_bytes
    forms = ["float32"] * 4 if dtype == F32 else ["codes"] + ["half"] * 3
    try:
        ops.open_bytes = 1
        # (the mean of thousands of values is small beside them, so the bounds are a larger part of it)
        attention_case(ops, 4, 1, 64, 16, portions, histories, forms, leading=1, dtype=dtype, share=0.1)
        ctx, table, pages = make_batch(portions, histories, 16, DEVICE)
        ctx.leading_single = 1
        kv = torch.zeros(pages, 2, 1, 2, 576, dtype=torch.uint8, device=DEVICE)
        whole, _, _ = make_batch([h + n for h, n in zip(histories, portions)], [0] * 4, 16, DEVICE)
        view = PackedView(kv, table, 16, PagedKeyValues(2, 64))
        x = rows_of(whole.tokens, 2, 64, dtype, 1).view(whole.tokens, -1).to(DEVICE)
        ops.pack_key_values(x, x, ctx=whole, view=view)
        q = torch.randn(ctx.tokens, 8, 64, device=DEVICE).to(dtype)
        call = lambda: ops.paged_attention(q, heads=8, kv_heads=2, head_dim=64, scale=0.125, window=None, ctx=ctx, view=view)
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = call()
        for _ in range(2):
            q.copy_(torch.randn(q.shape, device=DEVICE))
            graph.replay()
            replayed = captured.clone()
            assert torch.equal(call(), replayed)
        ops.check_errors()
    finally:
        ops.open_bytes = held


def test_portions_beside_a_long_single_token(ops):
    """With the portions' own bound, and without one."""
    portions, histories, forms = [1, 20, 30], [4000, 0, 10], ["codes", "half", "half"]
    for bound in (0, 40):
        attention_case(ops, 8, 2, 64, 16, portions, histories, forms, leading=1, rest_context=bound, share=0.1)


SHAPES = [(8, 2, 64, 16), (4, 4, 32, 16), (12, 1, 96, 32), (10, 2, 128, 64), (3, 1, 64, 128), (16, 2, 64, 16)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,kv_heads,dim,page", SHAPES)
@pytest.mark.parametrize("histories", [[0], [14, 15, 16, 31, 32], [300, 0, 5, 127], [1500, 33]])
@pytest.mark.parametrize("window,with_sinks", [(0, False), (33, True)])
def test_single_tokens(ops, dtype, heads, kv_heads, dim, page, histories, window, with_sinks):
    """One token a request over codes: weights times steps of 11 bits, everything else in 32."""
    sinks = torch.linspace(-1, 1, heads) if with_sinks else None
    forms = ["float32" if dtype == F32 else "codes"] * len(histories)
    attention_case(ops, heads, kv_heads, dim, page, [1] * len(histories), histories, forms, dtype=dtype, window=window,
                   sinks=sinks, seed=3)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,kv_heads,dim,page", SHAPES)
@pytest.mark.parametrize("portions,histories,leading", [
    ([5], [0], 0), ([1, 1, 37], [40, 9, 0], 2), ([70, 1, 16], [3, 100, 200], 0), ([1, 130], [15, 65], 1), ([300], [700], 0)])
@pytest.mark.parametrize("window,with_sinks", [(0, False), (40, False), (0, True), (50, True)])
def test_portions(ops, dtype, heads, kv_heads, dim, page, portions, histories, leading, window, with_sinks):
    """Opened in half-precision: 11 bits of keys, weights and values."""
    sinks = torch.linspace(-1, 1, heads) if with_sinks else None
    forms = ["float32"] * len(portions) if dtype == F32 else ["codes"] * leading + ["half"] * (len(portions) - leading)
    attention_case(ops, heads, kv_heads, dim, page, portions, histories, forms, leading=leading, dtype=dtype, window=window,
                   sinks=sinks, seed=4)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("portions,histories,leading", [([1, 1], [40, 90], 2), ([30, 1], [50, 7], 0), ([1, 60], [90, 40], 1)])
@pytest.mark.parametrize("how", [dict(cap=20.0), dict(cap=5.0, slopes=SLOPES), dict(slopes=SLOPES), dict(chunk=32),
                                 dict(window=24, keep_first=5)])
def test_shaped_scores(ops, dtype, portions, histories, leading, how):
    """Caps and slopes: opened in bfloat16, single tokens too. First positions: in half-precision. Chunks: as without."""
    form = "float32" if dtype == F32 else "half" if "chunk" in how or "keep_first" in how else "shaped"
    forms = [form] * len(portions)
    if "chunk" in how and dtype == BF16:
        forms[:leading] = ["codes"] * leading
    attention_case(ops, 6, 2, 64, 16, portions, histories, forms, leading=leading, dtype=dtype, seed=5, **how)


@pytest.mark.parametrize("dim,page", [(64, 16), (96, 32), (128, 64), (32, 16)])
@pytest.mark.parametrize("of_keys,of_queries,of_values", [
    (1e-30, 1e30, 1e-30), (1e-30, 1e-30, 1e30), (1e5, 1e-5, 2e4), (1e30, 1e-30, 1.0)])
@pytest.mark.parametrize("window", [0, 24])
def test_any_size(ops, dim, page, of_keys, of_queries, of_values, window):
    """Beyond half-precision's range: everything is times powers of two of its own."""
    attention_case(ops, 8, 2, dim, page, [1, 40, 21], [300, 30, 100], ["codes", "half", "half"], leading=1, window=window,
                   seed=6, of_keys=of_keys, of_queries=of_queries, of_values=of_values)


@pytest.mark.parametrize("heads,kv_heads,dim,page", [(8, 4, 64, 16), (8, 4, 128, 32), (8, 4, 32, 16), (8, 4, 96, 16)])
def test_roundings_in_the_mean(ops, heads, kv_heads, dim, page):
    """Rows enough to tell 8 bits of the keys alone from 11, and over opened pages of the values alone (computed with them
    the ratio is 1.2 to 2.7, with 11 bits 0.93 to 0.97)."""
    attention_case(ops, heads, kv_heads, dim, page, [1] * 16 + [60] * 6, [300] * 16 + [250] * 6, ["codes"] * 16 + ["half"] * 6,
                   leading=16, seed=7)
