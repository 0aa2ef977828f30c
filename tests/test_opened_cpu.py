"""What attention over packed pages hands to the kernels that read opened pages, without a GPU: a library that
writes down its launches, and a reader that writes down the step that it is given."""

import pytest
import torch

import plain_packed as plain
from mlx_one_b200.kernels.cuda_ops import CudaOps
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
        # (a number that tells whose row it is: the query's own first value)
        rows = q.reshape(how["ctx"].tokens, how["heads"], how["head_dim"])
        self.read.append((rows.clone(), view, how))
        got = rows[:, :, :1].expand(-1, -1, how["head_dim"]).reshape(how["ctx"].tokens, -1).clone()
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
