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
DEVICE, BF16 = "cuda:0", torch.bfloat16


def attention_case(ops, heads, kv_heads, dim, page, portions, histories, forms, *, leading=0, seed=0, of_keys=1.0,
                   of_queries=1.0, of_values=1.0, share=None, **how):
    """Keys and values packed plainly; a kernel's output against the exact one. ``share``: see packed_bounds.check."""
    ctx, table, pages = make_batch(portions, histories, page, DEVICE, seed=seed)
    ctx.leading_single = leading
    lengths = [h + n for h, n in zip(histories, portions)]
    kv = plain.empty_pages(pages, kv_heads, page, dim, fill=0xFF)       # (an earlier owner's NaN)
    for r, n in enumerate(lengths):
        both = [rows_of(n, kv_heads, dim, torch.float32, 10 * r + seed + 5 * which, 0.3) for which in (0, 1)]
        plain.pack(kv, table.cpu(), page, range(n), [r] * n, (both[0] * of_keys).to(BF16), (both[1] * of_values).to(BF16))
    q = (torch.randn(ctx.tokens, heads, dim, generator=torch.Generator().manual_seed(seed + 1)) * of_queries).to(BF16)
    want, bound = packed_bounds.attend(q, kv, table.cpu(), page, portions, histories, heads, kv_heads, dim ** -0.5, forms,
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
    packed_bounds.check(got, want, bound, portions, share or (0.06 if set(forms) <= {"codes", "half"} else 0.25))


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


@pytest.mark.parametrize("dtype", [torch.float32, BF16])
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


@pytest.mark.parametrize("dtype", [torch.float32, BF16])
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
