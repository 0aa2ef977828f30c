"""A cache held in 4 bits, attention over it, a beam's choice and the reordering of caches, restated plainly in 64 bits:
loops over tokens, heads and keys, written from the format's description (csrc/packed_cache.cuh)."""

import math

import torch


def groups_of(dim):
    return dim // 64 if dim % 64 == 0 else dim // 32


def part_bytes(dim):
    return 8 * dim + 64 * groups_of(dim)


def code_place(dim, values, key, d):
    """(byte, whether its upper half) of a unit's part for the code of token ``key``, dimension ``d``."""
    block, run, e = d // 64, d % 64 // 16, d % 16
    runs = min(4, (dim - 64 * block) // 16)
    e8, upper = e % 8, e // 8
    if values:
        lane, byte = 4 * e8 + key % 8 // 2, key // 8 + 2 * (key % 2)
    else:
        lane, byte = 4 * (key % 8) + e8 // 2, key // 8 + 2 * (e8 % 2)
    return 512 * block + 4 * (lane * runs + run) + byte, bool(upper)


def word_place(dim, key, group):
    return 8 * dim + 64 * group + 4 * (2 * (key % 8) + key // 8)


def places(dim, values):
    """(byte [16, dim], shift [16, dim])"""
    byte, shift = torch.empty(16, dim, dtype=torch.int64), torch.empty(16, dim, dtype=torch.int64)
    for key in range(16):
        for d in range(dim):
            byte[key, d], upper = code_place(dim, values, key, d)
            shift[key, d] = 4 if upper else 0
    return byte, shift


def quantized(x):
    """Rows x [n, dim] -> (codes int64 [n, dim], steps float64 [n, groups], lowest float64 [n, groups])."""
    n, dim = x.shape
    g = groups_of(dim)
    x = x.float().view(n, g, dim // g)
    low = x.amin(-1).bfloat16()
    # (a 32-bit product with the 32-bit inverse: division may round to the other side)
    step = ((x.amax(-1) - low.float()).clamp(min=0) * torch.tensor(1 / 15)).bfloat16()
    fine = torch.isfinite(x).all(-1) & torch.isfinite(step.float()) & torch.isfinite(low.float())
    low = torch.where(fine, low.double(), math.nan)
    step = torch.where(fine, step.double(), math.nan)
    code = ((x.double() - low[..., None]) / step[..., None]).round().clamp(0, 15)
    code = torch.where(fine[..., None] & (step > 0)[..., None], code, 0.0)
    return code.long().view(n, dim), step, low


def values_of(code, step, low):
    n, dim = code.shape
    g = step.shape[1]
    return (low[..., None] + step[..., None] * code.view(n, g, dim // g).double()).view(n, dim)


def empty_pages(pages, kv_heads, page_size, dim, fill=0):
    return torch.full((pages, kv_heads, page_size // 16, 2, part_bytes(dim)), fill, dtype=torch.uint8)


def put(kv, page, head, inside, which, code, step, low):
    """One token's row into a cache on the CPU."""
    dim = code.numel()
    part, key = kv[page, head, inside // 16, which], inside % 16
    byte, shift = _places(dim, which)
    for half in (0, 4):
        mine = shift[key] == half
        at = byte[key][mine]
        part[at] = (part[at] & (0xF0 if half == 0 else 0x0F)) | (code[mine] << half).to(torch.uint8)
    words = torch.stack([step.bfloat16(), low.bfloat16()], -1)
    words[torch.isnan(words)] = math.nan
    words = words.view(torch.int16)
    words = torch.where(words & 0x7FFF > 0x7F80, torch.tensor(0x7FC0, dtype=torch.int16), words)
    for group in range(step.numel()):
        at = word_place(dim, key, group)
        part[at:at + 4] = words[group].view(torch.uint8)


_CACHE = {}


def _places(dim, which):
    if (dim, which) not in _CACHE:
        _CACHE[dim, which] = places(dim, bool(which))
    return _CACHE[dim, which]


def pack(kv, table, page_size, positions, token_request, keys, values):
    """What the framework writes: ``kv`` changed in place (CPU). keys, values [tokens, heads, dim]."""
    for which, rows in ((0, keys), (1, values)):
        for h in range(rows.shape[1]):
            code, step, low = quantized(rows[:, h])
            for t in range(rows.shape[0]):
                p = int(positions[t])
                page = int(table[int(token_request[t]), p // page_size])
                put(kv, page, h, p % page_size, which, code[t], step[t], low[t])


def read(kv, table, page_size, request, length, dim):
    """float64 [2, length, heads, dim]: what lies at positions 0..length - 1; a position without a page is NaN."""
    heads = kv.shape[1]
    out = torch.full((2, length, heads, dim), math.nan, dtype=torch.float64)
    for block in range(-(-length // page_size)):
        page = int(table[request, block]) if block < table.shape[1] else -1
        if page < 0:
            continue
        for which in (0, 1):
            byte, shift = _places(dim, which)
            for unit in range(page_size // 16):
                first = block * page_size + 16 * unit
                count = min(16, length - first)
                if count <= 0:
                    continue
                part = kv[page, :, unit, which]                              # [heads, bytes]
                code = (part[:, byte].long() >> shift) & 15                  # [heads, 16, dim]
                at = torch.tensor([[word_place(dim, k, g) for g in range(groups_of(dim))] for k in range(16)])
                words = part[:, (at[..., None] + torch.arange(4)).view(-1)].contiguous().view(torch.bfloat16)
                words = words.view(heads, 16, groups_of(dim), 2).double()
                size = dim // groups_of(dim)
                value = (words[..., 1:] + words[..., :1] * code.view(heads, 16, -1, size).double()).view(heads, 16, dim)
                out[which, first:first + count] = value.transpose(0, 1)[:count]
    return out


def attend(q, kv, table, page_size, portions, histories, heads, kv_heads, scale, window=0, sinks=None):
    """float64 [tokens, heads, dim]; keys without a page are not seen."""
    group, dim, out, t = heads // kv_heads, q.shape[-1], [], 0
    for r, (n, held) in enumerate(zip(portions, histories)):
        keys, values = read(kv, table, page_size, r, held + n, dim)
        paged = torch.tensor([int(table[r, p // page_size]) >= 0 for p in range(held + n)], dtype=torch.bool)
        for i in range(n):
            p = held + i
            seen = paged & (torch.arange(held + n) <= p)
            if window:
                seen &= torch.arange(held + n) > p - window
            at = torch.nonzero(seen).view(-1)
            row = q[t + i].double()
            for h in range(heads):
                s = keys[at, h // group] @ row[h] * scale
                if sinks is not None:
                    s = torch.cat([s, sinks[h:h + 1].double()])
                if not s.numel():
                    out.append(torch.zeros(dim, dtype=torch.float64))
                    continue
                w = torch.softmax(s, 0)[:at.numel()]
                out.append(w @ values[at, h // group])
        t += n
    return torch.stack(out).view(t, heads, dim)


def choose(logits, scores, ended=None, end_tokens=()):
    """Lists per request of (score, parent, token, ended): the best candidates, ties to the lowest place."""
    requests, beams = scores.shape
    out = []
    for r in range(requests):
        found = []
        for b in range(beams):
            s = float(scores[r, b])
            if ended is not None and ended[r, b]:
                found.append((-math.inf if math.isnan(s) else s, b, end_tokens[0], 1))
                continue
            x = logits[r * beams + b].double()
            x = torch.where(torch.isnan(x), -math.inf, x)
            whole = float(torch.logsumexp(x, 0))
            if not math.isfinite(s) or not math.isfinite(whole):
                found += [(-math.inf, b, v, int(v in end_tokens)) for v in range(beams)]
                continue
            # (x - maximum - the logarithm: the maximum may be too large for the logarithm to count beside it)
            total = s + torch.log_softmax(x, 0)
            order = torch.sort(x, descending=True, stable=True).indices[:beams].tolist()
            found += [(float(total[v]), b, v, int(v in end_tokens)) for v in order]
        found.sort(key=lambda c: (-c[0], c[1], 0))           # (stable: a hypothesis' own are in order)
        out.append(found[:beams])
    return out
