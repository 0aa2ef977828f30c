"""The format of a cache held in 4 bits, and what its operators refuse, without a GPU."""

import pytest
import torch

import plain_packed as plain
from mlx_one_b200.kernels.cuda_ops import CudaOps, KernelError
from mlx_one_b200.parts.base import PackedView, PagedKeyValues, StepContext, packed_part_bytes


class Library:
    """Answers sizes; any launch is an error of the test."""

    def mlxone_packed_unit_bytes(self, dim):
        return 2 * packed_part_bytes(dim) if dim in (32, 64, 96, 128) else 0

    def __getattr__(self, name):
        raise AssertionError(f"{name} was launched")


@pytest.fixture
def ops():
    ops = CudaOps.__new__(CudaOps)
    ops.device, ops.lib, ops._sm_count = torch.device("cpu"), Library(), 148
    ops.error_flag = torch.zeros(1, dtype=torch.int32)
    ops._packed_cluster, ops._device_index, ops._packed_shapes = 8, 0, {}
    return ops


def step(tokens=4, requests=1):
    as_int = lambda v: torch.tensor(v, dtype=torch.int32)
    return StepContext(tokens=tokens, requests=requests, token_ids=as_int([0] * tokens),
                       positions=as_int(list(range(tokens))), token_request=as_int([0] * tokens),
                       request_start=as_int([0, tokens]), history=as_int([0]), max_portion=tokens, max_context=tokens)


def view(heads=2, dim=64, page=16, pages=3, **changes):
    kv = changes.pop("kv", plain.empty_pages(pages, heads, 16 if page % 16 else page, dim if dim in (32, 64, 96, 128) else 64))
    table = changes.pop("table", torch.zeros((1, 1), dtype=torch.int32))
    return PackedView(kv, table, page, PagedKeyValues(heads, dim, **changes))


@pytest.mark.parametrize("dim", [32, 64, 96, 128])
def test_every_code_has_a_place_of_its_own(dim):
    assert plain.part_bytes(dim) == packed_part_bytes(dim)
    for values in (False, True):
        byte, shift = plain.places(dim, values)
        assert sorted((byte * 2 + shift // 4).view(-1).tolist()) == list(range(16 * dim))
        # a byte belongs to one token
        owner = {}
        for key in range(16):
            for b in byte[key].tolist():
                assert owner.setdefault(b, key) == key
    words = sorted(plain.word_place(dim, k, g) for k in range(16) for g in range(plain.groups_of(dim)))
    assert words == list(range(8 * dim, plain.part_bytes(dim), 4))


def test_other_head_sizes_have_no_format():
    for dim in (16, 48, 80, 256):
        with pytest.raises(ValueError, match="32, 64, 96 or 128"):
            packed_part_bytes(dim)


@pytest.mark.parametrize("bad,message", [
    (dict(page=8), "power of two"), (dict(page=48), "power of two"), (dict(dim=80), "32, 64, 96 or 128"),
    (dict(planes=1), "planes"), (dict(kv=torch.zeros(3, 2, 1, 2, 575, dtype=torch.uint8)), "packed pages"),
    (dict(kv=torch.zeros(3, 2, 1, 2, 576)), "packed pages"), (dict(kv=torch.zeros(3, 1, 1, 2, 576, dtype=torch.uint8)), "packed pages"),
    (dict(kv=plain.empty_pages(3, 4, 16, 64)[:, ::2]), "packed pages"),
    (dict(table=torch.zeros((1, 1), dtype=torch.int64)), "block table")])
def test_views_that_are_refused(ops, bad, message):
    rows = torch.zeros(4, 128)
    with pytest.raises(KernelError, match=message):
        ops.pack_key_values(rows, rows, ctx=step(), view=view(**bad))
    with pytest.raises(KernelError, match=message):
        ops.read_key_values(ctx=step(), view=view(**bad))
    with pytest.raises(KernelError, match=message):
        ops.paged_attention(torch.zeros(4, 4, 64), heads=4, kv_heads=2, head_dim=64, scale=1.0, window=None,
                            ctx=step(), view=view(**bad))


def test_rows_that_are_refused(ops):
    rows = torch.zeros(4, 128)
    for keys, values in ((rows[:, :64], rows), (rows, rows[:3]), (rows, rows.bfloat16()), (rows.t().contiguous().t(), rows),
                         (rows[:3], rows[:3])):
        with pytest.raises(KernelError):
            ops.pack_key_values(keys, values, ctx=step(), view=view())
    with pytest.raises(KernelError, match="float32 and bfloat16"):
        ops.pack_key_values(rows.half(), rows.half(), ctx=step(), view=view())


def test_queries_that_are_refused(ops):
    call = dict(heads=4, kv_heads=2, head_dim=64, scale=1.0, window=None, ctx=step(), view=view())
    for q, change in ((torch.zeros(4, 4, 32), {}), (torch.zeros(4, 3, 64), dict(heads=3)),
                      (torch.zeros(4, 8, 64)[:, ::2], {}), (torch.zeros(4, 4, 64), dict(kv_heads=4)),
                      (torch.zeros(4, 4, 64), dict(sinks=torch.zeros(3))),
                      (torch.zeros(4, 4, 64), dict(window=5, chunk=5)),
                      (torch.zeros(4, 4, 64), dict(view=view(table=torch.zeros((0, 1), dtype=torch.int32))))):
        with pytest.raises(KernelError):
            ops.paged_attention(q, **{**call, **change})


def test_choices_that_are_refused(ops):
    logits, scores = torch.zeros(6, 50), torch.zeros(2, 3)
    ended, ends = torch.zeros(2, 3, dtype=torch.uint8), torch.tensor([2], dtype=torch.int32)
    for args, more in (((logits.bfloat16(), scores), {}), ((logits[:5], scores), {}), ((logits, scores.double()), {}),
                       ((logits, scores.view(-1)), {}), ((logits[:, :2], scores), {}),
                       ((torch.zeros(33, 50), torch.zeros(1, 33)), {}), ((logits, scores), dict(ended=ended)),
                       ((logits, scores), dict(ended=ended.int(), end_tokens=ends)),
                       ((logits, scores), dict(ended=ended[:1], end_tokens=ends)),
                       ((logits, scores), dict(ended=ended, end_tokens=ends.long())),
                       ((logits, scores), dict(ended=ended, end_tokens=ends[:0]))):
        with pytest.raises(KernelError):
            ops.beam_select(*args, **more)


def test_orders_that_are_refused(ops):
    state, slots, parents = torch.zeros(2, 7, 5), torch.arange(6, dtype=torch.int32), torch.zeros(2, 3, dtype=torch.int32)
    for args in ((state[:, :, :3], slots, parents), (state, slots[:5], parents), (state, slots.long(), parents),
                 (state, slots, parents.long()), (state, slots, parents.view(-1)), (torch.zeros(7), slots, parents),
                 (state, slots, torch.zeros(1, 33, dtype=torch.int32))):
        with pytest.raises(KernelError):
            ops.reorder_slots(*args)
    table, ends = torch.zeros(6, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for args, size in (((state, table[:5], parents, ends, ends), 16), ((state, table, parents, ends[:1], ends), 16),
                       ((state, table, parents, ends, ends.long()), 16), ((state[:, ::2], table, parents, ends, ends), 16),
                       ((state[0], table, parents, ends, ends), 16), ((state, table, parents, ends, ends), 0)):
        with pytest.raises(KernelError):
            ops.reorder_pages(*args, page_size=size)
