"""What the operators of decoding over a cache held in 4 bits, and of several hypotheses at a time, are measured on.

pack     keys and values of a step's tokens, written to pages of 4-bit codes and read back
attend   softmax attention of a step's queries over such pages
select   a beam search's choice: the best continuations of a request's hypotheses over the vocabulary
reorder  the caches of the chosen hypotheses, brought to where their new owners look: pages, or slots of fixed size

The format of a page. A page holds ``page`` tokens (a multiple of 16) of every key head: [pages, heads, page / 16, 2,
bytes], units of 16 tokens of one head, the keys' part and behind it the values'. A part is 16 * dim / 2 bytes of codes, then
for every group of a token's values (64 values; 32 where the head size is no multiple of 64) 16 words, the word of
token k at place 2 (k % 8) + k // 8: the step in the low half, the group's lowest value in the high half, both bfloat16.
A value is lowest + step * code. With lowest = bfloat16(min), step = bfloat16(max(max - lowest, 0) / 15 in 32 bits), the
code is (x - lowest) / step to the nearest whole number (ties to even), cut to 0..15; 0 where the step is 0. A group with a
value that is not finite, or whose lowest or step is none, has NaN for both and codes of 0.
The codes lie as 32 lanes of a warp take them for 16 x 16 x 8 matrix instructions. The dimensions are cut into blocks of
64 (the last of 32 where 32 are left) with n = 4 (or 2) runs of 16; a block is 32 lanes x n words. Byte b of lane l's
word s, r = l // 4, c = l % 4, has in the keys' part key r + 8 (b % 2) with the dimensions e and e + 8 of run s, e = 2 c + b
// 2, in its low and high four bits; in the values' part key 2 c + 8 (b % 2) + b // 2 with the dimensions r and r + 8.
"""

import math
import random

import torch

own = False

VOCAB = 65536
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def _pack_case(dtype, requests, tokens, history, kv_heads, dim, page, name=None):
    case = dict(op="pack", dtype=dtype, requests=requests, tokens=tokens, history=history, kv_heads=kv_heads,
                dim=dim, page=page)
    return dict(case, name=name) if name else case


def _attend_case(dtype, singles, portions, portion, context, heads, kv_heads, dim, page, window=0, sinks=False,
                 name=None):
    case = dict(op="attend", dtype=dtype, singles=singles, portions=portions, portion=portion, context=context,
                heads=heads, kv_heads=kv_heads, dim=dim, page=page, window=window, sinks=sinks)
    return dict(case, name=name) if name else case


def _select_case(requests, beams, vocab, name=None):
    case = dict(op="select", requests=requests, beams=beams, vocab=vocab)
    return dict(case, name=name) if name else case


def _pages_case(requests, beams, prompt, length, entries, kv_heads, dim, page, name=None):
    case = dict(op="reorder", what="pages", requests=requests, beams=beams, prompt=prompt, length=length,
                entries=entries, kv_heads=kv_heads, dim=dim, page=page)
    return dict(case, name=name) if name else case


def _slots_case(dtype, requests, beams, entries, values, name=None):
    case = dict(op="reorder", what="slots", dtype=dtype, requests=requests, beams=beams, entries=entries,
                values=values)
    return dict(case, name=name) if name else case


def listed():
    return [
        # a decode step of 16 requests, one token each: the smallest write, bound by its launch
        _pack_case("bfloat16", 16, 1, 700, 8, 64, 16, name="pack_singles"),
        # the largest step of prompt portions that the scheduler makes of two long prompts
        _pack_case("bfloat16", 2, 2048, 4096, 8, 64, 16, name="pack_portions"),
        # the 32-bit engine, ragged prompts, heads of 128 in larger pages
        _pack_case("float32", 5, 333, 77, 4, 128, 32, name="pack_f32_ragged"),
        # one user's chat turn: few keys, launches and latency
        _attend_case("bfloat16", 1, 0, 0, 509, 32, 8, 64, 16, name="attend_chat"),
        # a server: 32 conversations of about 4,096 tokens
        _attend_case("bfloat16", 32, 0, 0, 4096, 32, 8, 64, 16, name="attend_batch32"),
        # four long documents, heads of 128
        _attend_case("bfloat16", 4, 0, 0, 30011, 32, 8, 128, 64, name="attend_long"),
        # a portion of a prompt behind a cached half, beside seven running decodes
        _attend_case("bfloat16", 7, 1, 1024, 4100, 32, 8, 64, 16, name="attend_portion"),
        # the 32-bit engine's decode: scores of a few texts
        _attend_case("float32", 6, 0, 0, 2999, 24, 8, 64, 16, name="attend_f32"),
        # the first request's four hypotheses, the published vocabulary
        _select_case(1, 4, VOCAB, name="select_one"),
        # a batch of translations: 32 requests with eight hypotheses each
        _select_case(32, 8, VOCAB, name="select_batch"),
        # eight requests' hypotheses in 4-bit pages, 300 tokens behind their prompts
        _pages_case(8, 4, 1000, 1300, 6, 8, 64, 16, name="reorder_pages"),
        # matrices of state per head (the delta rule, 8 layers of 16 heads of 128 x 128)
        _slots_case("float32", 2, 4, 8, 16 * 128 * 128, name="reorder_slots"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _cost(case):
    need = work(case)
    return need["bytes"] / 4e12 + need["flops"] / (5e14 if case.get("dtype") != "float32" else 2e13)


def _kind(case):
    return case["op"] + case.get("dtype", "") + case.get("what", "")


def draw(rng):
    most = {}
    for case in listed():
        most[_kind(case)] = max(most.get(_kind(case), 0.0), _cost(case))
    most["reorderbfloat16slots"] = most["reorderfloat32slots"]
    while True:
        op = rng.choice(["pack", "attend", "attend", "select", "reorder"])
        dim, page = rng.choice([32, 64, 64, 96, 128]), rng.choice([16, 16, 32, 64, 128])
        kv_heads = rng.choice([1, 2, 3, 4, 8, 8])
        dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
        if op == "pack":
            case = _pack_case(dtype, _spread(rng, 1, 64), rng.choice([1, _spread(rng, 1, 2048)]),
                              rng.choice([0, _spread(rng, 1, 9000)]), kv_heads, dim, page)
        elif op == "attend":
            single = rng.random() < 0.7
            case = _attend_case(dtype, _spread(rng, 1, 64) if single else rng.choice([0, 1, 5]),
                                0 if single else _spread(rng, 1, 4), 0 if single else _spread(rng, 2, 2048),
                                _spread(rng, 1, 33000), kv_heads * rng.choice([1, 2, 3, 4, 4, 7, 8, 12]), kv_heads,
                                dim, page, rng.choice([0, 0, 0, _spread(rng, 1, 4096)]), rng.random() < 0.25)
        elif op == "select":
            case = _select_case(_spread(rng, 1, 64), _spread(rng, 1, 16), _spread(rng, 40, 200000))
        elif rng.random() < 0.5:
            prompt = _spread(rng, 1, 4000)
            case = _pages_case(_spread(rng, 1, 16), _spread(rng, 1, 16), prompt, prompt + _spread(rng, 1, 1000),
                               _spread(rng, 1, 16), kv_heads, dim, page)
        else:
            case = _slots_case(rng.choice(["float32", "bfloat16"]), _spread(rng, 1, 8), _spread(rng, 1, 16),
                               _spread(rng, 1, 16), _spread(rng, 1, 300000))
        kind = _kind(case)
        if _cost(case) <= most[kind] and _state_bytes(case) < 6e9:
            return case


# ------------------------------------------------------------------ the shape of a pass


def _groups(dim):
    return dim // 64 if dim % 64 == 0 else dim // 32


def _part_bytes(dim):
    return 16 * dim // 2 + 64 * _groups(dim)


def _around(mean, count, what):
    """``count`` lengths between three quarters and five quarters of ``mean``, the same for every seed."""
    if count == 1:
        return [mean]
    rng = random.Random("%s: %d of %d" % (what, count, mean))
    return [max(1, round(mean * rng.uniform(0.75, 1.25))) for _ in range(count)]


def _portions(case):
    """(tokens, tokens held before them) of every request of a pack or attend case."""
    if case["op"] == "pack":
        n = case["requests"]
        tokens = [1] * n if case["tokens"] == 1 else _around(case["tokens"], n, "tokens")
        held = _around(case["history"], n, "history") if case["history"] else [0] * n
        return list(zip(tokens, held))
    singles = [(1, n - 1) for n in _around(case["context"], case["singles"], "singles")] if case["singles"] else []
    tokens = _around(case["portion"], case["portions"], "portion") if case["portions"] else []
    keys = _around(case["context"], case["portions"], "context") if case["portions"] else []
    return singles + [(t, max(k - t, 0)) for t, k in zip(tokens, keys)]


def _seen(case):
    """Pairs of a query and a key that it sees, and keys that some query of their request sees."""
    pairs = keys = 0
    for tokens, held in _portions(case):
        window = case["window"]
        if window:
            for p in range(held, min(held + tokens, window)):
                pairs += p + 1
            pairs += window * max(0, held + tokens - max(held, window))
            keys += held + tokens - max(0, held - window + 1)
        else:
            pairs += tokens * held + tokens * (tokens + 1) // 2
            keys += held + tokens
    return pairs, keys


def work(case):
    if case["op"] == "pack":
        tokens = sum(t for t, _ in _portions(case))
        size = 2 if case["dtype"] == "bfloat16" else 4
        values = 2 * tokens * case["kv_heads"] * case["dim"]
        packed = 2 * tokens * case["kv_heads"] * _part_bytes(case["dim"]) // 16
        return {"bytes": 2 * values * size + 2 * packed, "flops": 8 * values}
    if case["op"] == "attend":
        pairs, keys = _seen(case)
        tokens = sum(t for t, _ in _portions(case))
        size = 2 if case["dtype"] == "bfloat16" else 4
        return {"bytes": 2 * tokens * case["heads"] * case["dim"] * size
                + 2 * keys * case["kv_heads"] * _part_bytes(case["dim"]) // 16,
                "flops": 4 * pairs * case["heads"] * case["dim"]}
    if case["op"] == "select":
        rows = case["requests"] * case["beams"]
        # (about one hypothesis in eight has ended: its row is not needed)
        ended = sum(sum(row) for row in _ended(case))
        values = (rows - ended) * case["vocab"]
        return {"bytes": 4 * values + 26 * rows, "flops": 4 * values}
    moved = sum(p != b for row in _parents(case) for b, p in enumerate(row))
    read = sum(len(set(p for b, p in enumerate(row) if p != b)) for row in _parents(case))
    if case["what"] == "slots":
        one = case["entries"] * case["values"] * (4 if case["dtype"] == "float32" else 2)
        return {"bytes": (moved + read) * one + 8 * case["requests"] * case["beams"], "flops": moved * one // 4 + 1}
    first, last = case["prompt"] // case["page"], -(-case["length"] // case["page"])
    one = (last - first) * case["entries"] * case["kv_heads"] * (case["page"] // 16) * 2 * _part_bytes(case["dim"])
    return {"bytes": (moved + read) * one + 8 * case["requests"] * case["beams"], "flops": moved * one // 4 + 1}


def _state_bytes(case):
    """Roughly what a plain pass holds."""
    if case["op"] == "attend":
        keys = sum(t + h for t, h in _portions(case)) + 128 * len(_portions(case))
        longest = max(t + h for t, h in _portions(case))
        widest = max(t for t, _ in _portions(case))
        return (keys * 2 * case["kv_heads"] * case["dim"] * 16
                + 12 * case["portions"] * widest * case["heads"] * longest
                + 12 * case["singles"] * case["heads"] * longest)
    if case["op"] == "select":
        return 40 * case["requests"] * case["beams"] * case["vocab"]
    return 8 * work(case)["bytes"]


def _parents(case):
    """Whose cache every hypothesis takes over: about half keep their own."""
    rng = random.Random("parents %d %d" % (case["requests"], case["beams"]))
    return [[b if rng.random() < 0.5 else rng.randrange(case["beams"]) for b in range(case["beams"])]
            for _ in range(case["requests"])]


def _ended(case):
    rng = random.Random("ended %d %d" % (case["requests"], case["beams"]))
    return [[rng.random() < 0.125 for _ in range(case["beams"])] for _ in range(case["requests"])]


# ------------------------------------------------------------------ what a caller has in hand


def _generator(seed):
    return torch.Generator("cuda").manual_seed(seed)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _tables(case, seed):
    """Block tables of pages in no order: int32 [requests, width], -1 behind a request's last page, and the pages."""
    blocks = [-(-(t + h) // case["page"]) for t, h in _portions(case)]
    width = max(blocks)
    order = torch.randperm(sum(blocks), generator=torch.Generator().manual_seed(seed)).tolist()
    table, used = [], 0
    for n in blocks:
        table.append(order[used:used + n] + [-1] * (width - n))
        used += n
    return _ints(table), used


def _step_tensors(case):
    portions = _portions(case)
    tokens = [t for t, _ in portions]
    return dict(
        positions=torch.cat([torch.arange(h, h + t, dtype=torch.int32) for t, h in portions]).cuda(),
        token_request=torch.repeat_interleave(torch.arange(len(portions), dtype=torch.int32),
                                              torch.tensor(tokens)).cuda(),
        request_start=_ints([sum(tokens[:i]) for i in range(len(tokens) + 1)]),
        history=_ints([h for _, h in portions]), tokens=sum(tokens), requests=len(portions),
        max_portion=max(tokens), max_context=max(t + h for t, h in portions))


def _used_pages(case, table, pages, generator):
    """Pages of a cache in use: codes of values that are about normal, steps and lowest values to match; rows that no
    token has written yet hold what an earlier owner left, NaN here."""
    dim, groups, part = case["dim"], _groups(case["dim"]), _part_bytes(case["dim"])
    units = case["page"] // 16
    kv = torch.empty((pages, case["kv_heads"], units, 2, part), dtype=torch.uint8, device="cuda")
    shape = (pages, case["kv_heads"], units, 2, 8 * dim)
    low = (torch.randn(shape, generator=generator, device="cuda") * 3 + 7.5).round_().clamp_(0, 15).to(torch.uint8)
    high = (torch.randn(shape, generator=generator, device="cuda") * 3 + 7.5).round_().clamp_(0, 15).to(torch.uint8)
    kv[..., :8 * dim] = low | (high << 4)
    shape = (pages, case["kv_heads"], units, 2, groups, 16)
    step = 0.3 + 0.1 * torch.rand(shape, generator=generator, device="cuda")
    lowest = -7.5 * step + 0.2 * torch.randn(shape, generator=generator, device="cuda")
    words = torch.stack([step, lowest], -1).to(torch.bfloat16)
    # (place 2 (k % 8) + k // 8 of a group's words is token k's)
    token = torch.arange(16, device="cuda") // 2 + 8 * (torch.arange(16, device="cuda") % 2)
    lengths = _ints([t + h for t, h in _portions(case)])
    blocks = torch.arange(table.shape[1], device="cuda")
    written = torch.zeros((pages + 1, units, 16), dtype=torch.bool, device="cuda")
    at = (blocks[:, None, None] * case["page"] + torch.arange(units, device="cuda")[:, None] * 16 + token)
    written[torch.where(table >= 0, table, pages).long()] = at[None] < lengths[:, None, None, None]
    words = torch.where(written[:pages, None, :, None, None, :, None], words, float("nan"))
    kv[..., 8 * dim:] = words.contiguous().view(torch.uint8).reshape(*kv.shape[:-1], 64 * groups)
    return kv


def prepare(case, seed):
    generator = _generator(seed)
    rand = lambda *shape: torch.randn(shape, generator=generator, device="cuda")  # noqa: E731
    state = dict(case=case)
    if case["op"] in ("pack", "attend"):
        dtype = DTYPES[case["dtype"]]
        table, pages = _tables(case, seed)
        state.update(_step_tensors(case), table=table)
        inner = case["kv_heads"] * case["dim"]
        if case["op"] == "pack":
            # keys and values as slices of rows that held queries too; a few channels are much larger than the others
            rows = rand(state["tokens"], 4 * inner) * torch.exp(0.8 * rand(4 * inner))
            state["rows"] = rows.to(dtype)
            state["kv"] = torch.randint(0, 256, (pages, case["kv_heads"], case["page"] // 16, 2,
                                                 _part_bytes(case["dim"])), generator=generator, device="cuda",
                                        dtype=torch.uint8)
        else:
            state["q"] = rand(state["tokens"], case["heads"], case["dim"]).to(dtype)
            state["kv"] = _used_pages(case, table, pages, generator)
            state["sinks"] = rand(case["heads"]) if case["sinks"] else None
        return state
    rows = case["requests"] * case["beams"]
    if case["op"] == "select":
        # (logits of a language model: most of the weight on few tokens; a few tokens are forbidden)
        state["logits"] = 2.5 * rand(rows, case["vocab"])
        state["logits"].masked_fill_(torch.rand(state["logits"].shape, generator=generator, device="cuda") < 0.001,
                                     float("-inf"))
        state["scores"] = -5.0 * torch.rand((case["requests"], case["beams"]), generator=generator, device="cuda")
        state["ended"] = torch.tensor(_ended(case), dtype=torch.uint8, device="cuda")
        state["ends"] = _ints([2, 7])
        return state
    state["parents"] = _ints(_parents(case))
    if case["what"] == "slots":
        order = torch.randperm(rows, generator=torch.Generator().manual_seed(seed))
        state["slots"] = order.to(torch.int32).cuda()
        state["held"] = rand(case["entries"], rows + 1, case["values"]).to(DTYPES[case["dtype"]])
        return state
    blocks = -(-case["length"] // case["page"])
    order = torch.randperm(rows * blocks, generator=torch.Generator().manual_seed(seed))
    state["table"] = order.view(rows, blocks).to(torch.int32).cuda()
    state["starts"] = _ints([case["prompt"]] * case["requests"])
    state["lengths"] = _ints([case["length"]] * case["requests"])
    state["held"] = torch.randint(0, 256, (case["entries"], rows * blocks + 1, case["kv_heads"], case["page"] // 16, 2,
                                           _part_bytes(case["dim"])), generator=generator, device="cuda",
                                  dtype=torch.uint8)
    return state


# ------------------------------------------------------------------ plain forms


def _places(dim, device):
    """Where code (token, dimension) of a unit lies: (byte in the keys' part, byte in the values' part, shift)."""
    k = torch.arange(16, device=device)[:, None]
    d = torch.arange(dim, device=device)[None]
    run, e = d % 64 // 16, d % 16
    runs = torch.clamp((dim - d // 64 * 64) // 16, max=4)
    base = d // 64 * 512
    half, odd = k // 8, e % 2
    keys = base + 4 * ((4 * (k % 8) + e % 8 // 2) * runs + run) + half + 2 * odd
    values = base + 4 * ((4 * (e % 8) + k % 8 // 2) * runs + run) + half + 2 * (k % 2)
    return keys.reshape(-1), values.reshape(-1), (4 * (e // 8)).expand(16, dim).reshape(-1).to(torch.uint8)


def _words_at(device):
    k = torch.arange(16, device=device)
    return 2 * (k % 8) + k // 8


def _read_part(part, dim, place, shift):
    """[..., bytes] -> float32 [..., 16, dim]."""
    groups = _groups(dim)
    codes = (part.index_select(-1, place) >> shift) & 15
    words = part[..., 8 * dim:].contiguous().view(torch.bfloat16).view(*part.shape[:-1], groups, 16, 2)
    words = words.index_select(-2, _words_at(part.device)).float().transpose(-3, -2)
    codes = codes.view(*part.shape[:-1], 16, groups, dim // groups)
    return (words[..., 1:] + words[..., :1] * codes).flatten(-2)


def _coded(x, dim):
    """Rows x [n, heads, dim] -> codes, steps and lowest values of their groups."""
    x = x.float().view(*x.shape[:-1], _groups(dim), dim // _groups(dim))
    lowest = x.amin(-1).to(torch.bfloat16).float()
    step = (torch.clamp(x.amax(-1) - lowest, min=0) / 15).to(torch.bfloat16).float()
    fine = torch.isfinite(x).all(-1) & torch.isfinite(step) & torch.isfinite(lowest)
    step, lowest = torch.where(fine, step, float("nan")), torch.where(fine, lowest, float("nan"))
    # (in 64 bits: values next to a border)
    code = torch.round((x.double() - lowest.double()[..., None]) / step.double()[..., None]).clamp(0, 15)
    code = torch.where(fine[..., None] & (step > 0)[..., None], code, 0.0)
    return code.to(torch.uint8), step, lowest


def _plain_pack(state):
    case, dim, kv = state["case"], state["case"]["dim"], state["kv"]
    inner = case["kv_heads"] * dim
    positions = state["positions"].long()
    page = state["table"][state["token_request"].long(), positions // case["page"]].long()
    unit, k = positions % case["page"] // 16, positions % 16
    keys_at, values_at, _ = _places(dim, kv.device)
    heads = torch.arange(case["kv_heads"], device=kv.device)
    where = (page[:, None], heads[None], unit[:, None])
    outs = []
    for part, place, x in ((0, keys_at, state["rows"][:, 2 * inner:3 * inner]),
                           (1, values_at, state["rows"][:, 3 * inner:])):
        code, step, lowest = _coded(x.reshape(-1, case["kv_heads"], dim), dim)
        code = code.flatten(-2).view(-1, case["kv_heads"], dim // 16, 2, 8)
        both = (code[..., 0, :] | (code[..., 1, :] << 4)).flatten(-2)           # dimensions e and e + 8 share a byte
        at = place.view(16, dim // 16, 2, 8)[:, :, 0].reshape(16, dim // 2)[k]
        kv[where[0][..., None], where[1][..., None], where[2][..., None], part, at[:, None]] = both
        words = torch.stack([step, lowest], -1).to(torch.bfloat16).view(torch.uint8).flatten(-2)
        words = words.view(-1, case["kv_heads"], _groups(dim) * 4)
        at = (8 * dim + 64 * torch.arange(_groups(dim), device=kv.device)[:, None]
              + torch.arange(4, device=kv.device))[None] + 4 * _words_at(kv.device)[k][:, None, None]
        kv[where[0][..., None], where[1][..., None], where[2][..., None], part, at.flatten(1)[:, None]] = words
    return [_plain_read(state, part).to(state["rows"].dtype) for part in (0, 1)]


def _plain_read(state, part):
    """What the step's tokens find at their places: float32 [tokens, heads, dim]."""
    case, dim = state["case"], state["case"]["dim"]
    positions = state["positions"].long()
    page = state["table"][state["token_request"].long(), positions // case["page"]].long()
    rows = state["kv"][page, :, positions % case["page"] // 16, part]           # [tokens, heads, bytes]
    groups, k = _groups(dim), positions % 16
    at = _places(dim, rows.device)[part].view(16, dim)[k]
    shift = _places(dim, rows.device)[2].view(16, dim)[0]
    code = (rows.gather(-1, at[:, None].expand(-1, rows.shape[1], -1)) >> shift) & 15
    words = rows[..., 8 * dim:].contiguous().view(torch.bfloat16).view(*rows.shape[:2], groups, 16, 2).float()
    words = words.gather(-2, _words_at(rows.device)[k][:, None, None, None, None].expand(-1, rows.shape[1], groups, 1, 2))
    step, lowest = words[..., 0, 0], words[..., 0, 1]
    return (lowest[..., None] + step[..., None] * code.view(*code.shape[:2], groups, -1)).flatten(-2)


def _plain_attend(state, first, last, widest, longest):
    """Requests first..last-1, which bring up to ``widest`` tokens and have up to ``longest`` keys."""
    case, dim = state["case"], state["case"]["dim"]
    n, kv_heads = last - first, case["kv_heads"]
    width = -(-longest // case["page"])
    table = state["table"][first:last, :width].long()
    pages = state["kv"][table.clamp(min=0)]                     # [n, width, heads, units, 2, bytes]
    keys_at, values_at, shift = _places(dim, pages.device)
    flat = lambda x: x.permute(0, 2, 1, 3, 4, 5).reshape(n, kv_heads, -1, dim)  # noqa: E731
    keys = flat(_read_part(pages[..., 0, :], dim, keys_at, shift))
    values = flat(_read_part(pages[..., 1, :], dim, values_at, shift))
    start = state["request_start"].long()
    lengths = state["history"].long()[first:last] + start[first + 1:last + 1] - start[first:last]
    key = torch.arange(keys.shape[2], device=keys.device)
    held = (key < lengths[:, None]) & (table >= 0).repeat_interleave(case["page"], 1)
    values = torch.where(held[:, None, :, None], values, 0.0)
    place = torch.arange(widest, device=keys.device)
    token = start[first:last, None] + place
    real = token < start[first + 1:last + 1, None]
    q = state["q"][torch.where(real, token, 0)].float()         # [n, widest, heads, dim]
    q = q.view(n, widest, kv_heads, -1, dim).permute(0, 2, 3, 1, 4).reshape(n, kv_heads, -1, dim)
    scores = (q @ keys.transpose(-1, -2) * dim ** -0.5).view(n, kv_heads, -1, widest, key.numel())
    position = (state["history"].long()[first:last, None] + place)[..., None]
    seen = held[:, None] & (key <= position)
    if case["window"]:
        seen = seen & (key > position - case["window"])
    scores = torch.where(seen[:, None, None], scores, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    if state["sinks"] is not None:
        sinks = state["sinks"].view(1, kv_heads, -1, 1, 1)
        top = torch.maximum(top, sinks)
    top = torch.where(top == float("-inf"), 0.0, top)
    weights = torch.exp(scores - top)
    total = weights.sum(-1, keepdim=True)
    if state["sinks"] is not None:
        total = total + torch.exp(sinks - top)
    out = weights.view(n, kv_heads, -1, key.numel()) @ values
    out = out.view(n, kv_heads, -1, widest, dim) / torch.where(total > 0, total, 1.0)
    out = out.permute(0, 3, 1, 2, 4).reshape(n * widest, -1)    # [n, widest, heads x dim]
    # a row of a request's last, shorter portion goes where nothing is kept
    return out, torch.where(real, token, state["tokens"]).reshape(-1)


def _plain_attention(state):
    case, portions = state["case"], _portions(state["case"])
    out = torch.zeros((state["tokens"] + 1, case["heads"] * case["dim"]), dtype=torch.float32, device="cuda")
    for first, last in ((0, case["singles"]), (case["singles"], len(portions))):      # single tokens, portions
        if first < last:
            here = portions[first:last]
            rows, at = _plain_attend(state, first, last, max(t for t, _ in here), max(t + h for t, h in here))
            out[at] = rows
    return out[:-1].to(state["q"].dtype)


def _plain_select(state):
    case = state["case"]
    requests, beams, vocab = case["requests"], case["beams"], case["vocab"]
    logits = state["logits"].double()                            # (in 64 bits: candidates next to each other)
    top = logits.amax(-1, keepdim=True)
    logs = logits - top - torch.log(torch.exp(logits - top).sum(-1, keepdim=True))
    sums = state["scores"].double()[..., None] + logs.view(requests, beams, vocab)
    ended = state["ended"].bool()[..., None]
    # a hypothesis that has ended stays as it is: one candidate, in the place of the first end token
    kept = torch.arange(vocab, device=sums.device) == state["ends"][0]
    alone = torch.where(kept, state["scores"].double()[..., None], float("nan"))
    sums = torch.where(ended, alone, sums)
    sums = sums.view(requests, beams * vocab)
    exists = ~torch.isnan(sums)
    # the last that is taken, then all above it and the first that equal it; a place that is no candidate is out
    ranked = torch.where(exists, sums, float("-inf"))
    least = ranked.topk(beams, -1).values[:, -1:]
    above, same = exists & (ranked > least), exists & (ranked == least)
    taken = above | (same & (same.cumsum(-1, dtype=torch.int32) <= beams - above.sum(-1, keepdim=True)))
    index = torch.arange(beams * vocab, device=sums.device)
    first = -torch.where(taken, -index, -beams * vocab).topk(beams, -1).values   # in the order of their places
    values, order = ranked.gather(-1, first).sort(dim=-1, descending=True, stable=True)
    first = first.gather(-1, order)
    parents, tokens = first // vocab, first % vocab
    over = state["ended"].gather(-1, parents).bool() | (tokens[..., None] == state["ends"]).any(-1)
    return [values.float(), parents.to(torch.int32), tokens.to(torch.int32), over.to(torch.uint8)]


def _plain_reorder(state):
    case = state["case"]
    requests, beams = case["requests"], case["beams"]
    source = (torch.arange(requests, device="cuda")[:, None] * beams + state["parents"].long()).view(-1)
    if case["what"] == "slots":
        slots = state["slots"].long()
        state["held"][:, slots] = state["held"][:, slots[source]]
        return state["held"]
    blocks = torch.arange(case["prompt"] // case["page"], -(-case["length"] // case["page"]), device="cuda")
    table = state["table"].long()[:, blocks]
    state["held"][:, table.view(-1)] = state["held"][:, table[source].view(-1)]
    return state["held"]


# ------------------------------------------------------------------ one pass


def _step_of(state, view):
    from mlx_one_b200.parts.base import StepContext

    return StepContext(tokens=state["tokens"], requests=state["requests"], token_ids=state["positions"],
                       positions=state["positions"], token_request=state["token_request"],
                       request_start=state["request_start"], history=state["history"],
                       max_portion=state["max_portion"], max_context=state["max_context"],
                       leading_single=state["case"].get("singles", 0))


def _packed_view(state):
    from mlx_one_b200.parts.base import PackedView, PagedKeyValues

    case = state["case"]
    return PackedView(state["kv"], state["table"], case["page"], PagedKeyValues(case["kv_heads"], case["dim"]))


def _run_own(state):
    from mlx_one_b200.kernels import default_ops

    case, ops = state["case"], default_ops("cuda:0")
    if case["op"] == "pack":
        view, inner = _packed_view(state), case["kv_heads"] * case["dim"]
        step = _step_of(state, view)
        ops.pack_key_values(state["rows"][:, 2 * inner:3 * inner], state["rows"][:, 3 * inner:], ctx=step, view=view)
        return list(ops.read_key_values(ctx=step, view=view, dtype=state["rows"].dtype))
    if case["op"] == "attend":
        view = _packed_view(state)
        return ops.paged_attention(state["q"], heads=case["heads"], kv_heads=case["kv_heads"], head_dim=case["dim"],
                                   scale=case["dim"] ** -0.5, window=case["window"] or None,
                                   ctx=_step_of(state, view), view=view, sinks=state["sinks"])
    if case["op"] == "select":
        return list(ops.beam_select(state["logits"], state["scores"], ended=state["ended"], end_tokens=state["ends"]))
    if case["what"] == "slots":
        ops.reorder_slots(state["held"], state["slots"], state["parents"])
    else:
        ops.reorder_pages(state["held"], state["table"], state["parents"], state["starts"], state["lengths"],
                          page_size=case["page"])
    return state["held"]


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op == "pack":
        return _plain_pack(state)
    if op == "attend":
        return _plain_attention(state)
    return _plain_select(state) if op == "select" else _plain_reorder(state)


# ------------------------------------------------------------------ in 64 bits


def _exact_part(part, dim, values):
    """[..., bytes] -> float64 [..., 16, dim], taken apart lane by lane."""
    groups, lead, pieces = _groups(dim), part.shape[:-1], []
    for block in range(0, dim, 64):
        runs = min(4, (dim - block) // 16)
        raw = part[..., 8 * block:8 * block + 128 * runs].reshape(*lead, 8, 4, runs, 2, 2)   # r, c, run, odd, half
        both = torch.stack([raw % 16, raw // 16], -1)                                   # ..., low or high four bits
        n = len(lead)
        r, c, run, odd, half, high = (n + i for i in range(6))
        if values:      # token = half, c, odd; dimension = run, high, r
            both = both.permute(*range(n), half, c, odd, run, high, r)
        else:           # token = half, r; dimension = run, high, c, odd
            both = both.permute(*range(n), half, r, run, high, c, odd)
        pieces.append(both.reshape(*lead, 16, 16 * runs))
    codes = torch.cat(pieces, -1).double()
    words = part[..., 8 * dim:].contiguous().view(torch.bfloat16).double().view(*lead, groups, 8, 2, 2)
    words = words.transpose(-3, -2).reshape(*lead, groups, 16, 2).repeat_interleave(dim // groups, -3)
    return words[..., 1].transpose(-1, -2) + words[..., 0].transpose(-1, -2) * codes


def _exact_pack(state):
    case, dim, outs = state["case"], state["case"]["dim"], []
    inner, size = case["kv_heads"] * dim, dim // _groups(dim)
    for x in (state["rows"][:, 2 * inner:3 * inner], state["rows"][:, 3 * inner:]):
        x = x.double().reshape(-1, size)
        least = x.min(1).values.float().bfloat16()
        # (the difference and the quotient in 32 bits are part of the format)
        span = x.max(1).values.float().sub(least.float()).clamp(min=0)
        step = span.div(15.0).bfloat16().double()[:, None]
        least = least.double()[:, None]
        code = torch.where(step > 0, ((x - least) / step).round(), 0.0).clamp(0, 15)
        outs.append((least + code * step).view(-1, case["kv_heads"], dim))
    return outs


def _exact_attend(state):
    case, dim = state["case"], state["case"]["dim"]
    group, outs = case["heads"] // case["kv_heads"], []
    start = 0
    for r, (tokens, held) in enumerate(_portions(case)):
        q = state["q"][start:start + tokens].double()
        start += tokens
        blocks = -(-(held + tokens) // case["page"])
        pages = state["kv"][state["table"][r, :blocks].long()]
        total = held + tokens
        position = torch.arange(held, total, device="cuda")[:, None]
        key = torch.arange(total, device="cuda")
        hidden = key > position
        if case["window"]:
            hidden |= key <= position - case["window"]
        heads = []
        for h in range(case["kv_heads"]):
            k = _exact_part(pages[:, h, :, 0], dim, False).reshape(-1, dim)[:total]
            v = _exact_part(pages[:, h, :, 1], dim, True).reshape(-1, dim)[:total]
            for g in range(group):
                s = (q[:, h * group + g] @ k.T) / math.sqrt(dim)
                s.masked_fill_(hidden, float("-inf"))
                if state["sinks"] is not None:
                    s = torch.cat([s, state["sinks"][h * group + g].double().expand(tokens, 1)], 1)
                heads.append(torch.softmax(s, -1)[:, :total] @ v)
        outs.append(torch.cat(heads, -1))
    return torch.cat(outs)


def exact(case, seed):
    if case["op"] == "reorder":
        return None
    state = prepare(case, seed)
    if case["op"] == "pack":
        return _exact_pack(state)
    if case["op"] == "attend":
        return _exact_attend(state)
    # the chosen sums of logarithms: only the values are computed numbers
    logs = torch.log_softmax(state["logits"].double(), -1).view(case["requests"], case["beams"], -1)
    sums = logs + state["scores"].double()[..., None]
    ended = state["ended"].bool()
    sums[ended] = float("-inf")
    stay = torch.where(ended, state["scores"].double(), float("-inf"))
    every = torch.cat([sums.flatten(1), stay], 1)
    return [every.sort(-1, descending=True).values[:, :case["beams"]], None, None, None]
