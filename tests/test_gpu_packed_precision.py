"""Attention over a cache held in 4 bits within the bounds of the roundings that its kernels have (packed_bounds.py),
each bound a small part of the output that it is about."""

import pytest
import torch

import packed_bounds
import plain_packed as plain
from test_gpu_kernels import make_batch, ops  # noqa: F401  (fixture)
from test_gpu_packed_cache import rows_of
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
