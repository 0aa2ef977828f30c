"""Attention over a cache held in 4 bits in 64 bits, and how far a kernel's output may be off, element by element,
by the roundings that the kernel has."""

import torch

import plain_packed as plain

# What a kernel rounds, each by at most half a step, relative to the value: the keys, the weights of the values and
# the values. "codes": codes are exact, scores 32-bit, the weight times a value's step has 11 bits, a value's
# lowest comes in 32 bits. "half": pages opened in half-precision. "bfloat16": opened in bfloat16, read by kernels
# that keep weights in 32 bits; "shaped": by tensor cores, whose weights are bfloat16 too. "float32": everything in
# 32 bits, four roundings each, over codes (less 8) as over opened pages.
HALF, BF16, F32 = 2.0 ** -11, 2.0 ** -8, 2.0 ** -22
FORMS = dict(codes=(0.0, HALF, 0.0), half=(HALF, HALF, HALF), bfloat16=(BF16, 0.0, BF16), shaped=(BF16, BF16, BF16),
             float32=(F32, F32, F32))


def parts(kv, table, page, request, length, dim):
    """(keys, values, the values' part above their group's lowest), float64 [length, heads, dim]."""
    keys, values = plain.read(kv, table, page, request, length, dim)
    zero = kv.clone()
    zero[..., :8 * dim] = 0                                  # codes of 0: what is left is the lowest value
    return keys, values, values - plain.read(zero, table, page, request, length, dim)[1]


def attend(q, kv, table, page, portions, histories, heads, kv_heads, scale, forms, *, window=0, chunk=0, keep_first=0,
           sinks=None, cap=0.0, slopes=None):
    """(wanted, bound, variance), float64 [tokens, heads, dim]. ``forms``: a name of FORMS for every request.

    With p the exact weights, o the exact output and e_j how far score j may be off, the weights are off by
    expm1(e_j) of themselves, numerator and denominator alike, which moves o by p_j expm1(e_j) |v_j - o| a key; the
    numerator's own roundings by p_j |v_j| (that of the weight and that of the value). e_j: the keys' rounding times
    scale sum |q_d k_jd|, dim additions that may cut at 2^-23 each, 2^-22 of the largest score for the exponent's
    argument, 2^-21 for the exponential. What is below half-precision's normal numbers (powers of two bring the
    largest to 2^7 or more) is off by 2^-32 of the largest. A value's sum has a sixteenth as many additions as keys
    (in 32 bits as many as keys), and 64 for the merges, of the value and of what is above its group's lowest. The
    result is rounded once.

    The variance is what the same roundings leave in the mean: one of half a step h has h^2 / 3, and h is, relative to a
    value whose leading digits are spread evenly on a logarithmic scale, 3 / (8 ln 2) of its largest squared; the
    result's own is taken as it is."""
    out, bound, spread, group, dim, t = [], [], [], heads // kv_heads, q.shape[-1], 0
    mean = 0.5411 / 3
    for r, (n, held) in enumerate(zip(portions, histories)):
        of_key, of_weight, of_value = FORMS[forms[r]]
        of_result = 2.0 ** -24 if forms[r] == "float32" else BF16
        length = held + n
        keys, values, above = parts(kv, table, page, r, length, dim)
        place = torch.arange(length)[None]
        position = torch.arange(held, length)[:, None]
        seen = place <= position
        if window:
            seen &= (place > position - window) | (place < keep_first)
        if chunk:
            seen &= place >= position - position % chunk
        rows, bounds, variances = [], [], []
        for h in range(heads):
            k, v = keys[:, h // group], values[:, h // group]
            x = q[t:t + n, h].double()
            s, size = scale * x @ k.T, scale * x.abs() @ k.abs().T
            e = size * (of_key + dim * 2.0 ** -23) + scale * dim * x.abs().amax(-1, keepdim=True) * k.abs().max() * 2.0 ** -32
            if cap:
                s = cap * torch.tanh(s / cap)                # (its slope is at most 1; a polynomial, or two approximations)
                e = e + cap * 2.0 ** -16
            if slopes is not None:
                s = s - slopes[h].double() * (position - place)
            s = torch.where(seen, s, -torch.inf)
            top = torch.where(seen, s.abs(), 0.0).amax(-1, keepdim=True)
            all_ = s if sinks is None else torch.cat([s, sinks[h].double().expand(n, 1)], 1)
            p = torch.softmax(all_, -1)[:, :length]
            o = p @ v
            delta = torch.expm1(e + top * 2.0 ** -22 + 2.0 ** -21)
            worst = torch.where(seen, delta, 0.0).amax(-1, keepdim=True)
            off = torch.einsum("nj,njd->nd", p * delta, (v[None] - o[:, None]).abs())
            if sinks is not None:                            # (the sink's own weight, exact but for the exponential)
                off = off + o.abs() * (1 - p.sum(-1, keepdim=True)) * (worst + 2.0 ** -20)
            rounded = above[:, h // group].abs() if forms[r] == "codes" else v.abs()
            sums = (length / (1 if forms[r] == "float32" else 16) + 64) * 2.0 ** -23
            off = off / (1 - worst).clamp(min=1e-9) + (1 + worst) * (
                p @ (rounded * (of_weight + of_value)) + p @ (v.abs() + above[:, h // group].abs()) * sums)
            off = off * (1 + BF16) + length * 2.0 ** -32 * v.abs().max()
            rows.append(o)
            bounds.append(off + of_result * (o.abs() + off))
            of_score = mean * (scale * of_key) ** 2 * (x ** 2 @ (k ** 2).T)
            step = 2.0 ** torch.floor(torch.log2(o.abs().clamp(min=1e-300))) * of_result
            variances.append(torch.einsum("nj,njd->nd", p ** 2 * of_score, (v[None] - o[:, None]) ** 2)
                             + mean * (of_weight ** 2 + of_value ** 2) * (p ** 2 @ rounded ** 2) + step ** 2 / 3)
        out.append(torch.stack(rows, 1))
        bound.append(torch.stack(bounds, 1))
        spread.append(torch.stack(variances, 1))
        t += n
    return torch.cat(out), torch.cat(bound), torch.cat(spread)


def check_mean(got, want, variance, group):
    """The errors' root mean square against what the roundings leave: elements of one dimension and key head count as one
    (``group`` heads that see few keys have the same output), and as many as their variances are worth; the mean
    of n squares of such roundings is off by less than 0.9 / sqrt(n), its root by half of that: 1.1 and six times
    that. (Computed with keys, weights and values in bfloat16 instead of 11 bits the ratio is 1.4 to 2.)"""
    worth = float(variance.sum() ** 2 / (variance ** 2).sum()) / group
    ratio = float(((got - want) ** 2).sum() / variance.sum()) ** 0.5
    assert ratio < 1.1 + 2.7 / worth ** 0.5, (ratio, worth)


def check(got, want, bound, portions, share):
    """Every element within its bound, and every bound a small part of what it bounds: less than ``share`` of the
    largest output of its request and head."""
    t = 0
    for r, n in enumerate(portions):
        most = want[t:t + n].abs().amax((0, 2))
        assert (bound[t:t + n].amax((0, 2)) < share * most).all(), (r, (bound[t:t + n].amax((0, 2)) / most).tolist())
        if got is not None:
            off = (got[t:t + n] - want[t:t + n]).abs()
            assert (off <= bound[t:t + n]).all(), (r, float((off / bound[t:t + n]).max()))
        t += n
