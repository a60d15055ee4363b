"""Plain restatements of the operators around a paged cache, in Python integers
and float64 (fp32 only where the operator's definition rounds to it).  Test
infrastructure, written from the definitions in include/kvq.h."""
from __future__ import annotations

import numpy as np

F32 = np.float32


def pages_of(tokens, size):
    return -(-int(tokens) // size)


def page_map(new_tokens, lengths, table, free_pages, free_count, size, T):
    """One sequence after the other, with the free stack as a list."""
    table = [[int(x) for x in r] for r in table]
    free = [int(x) for x in free_pages]
    num, cap, B = len(free), len(table[0]) * size, len(lengths)
    new_tokens = [int(n) for n in new_tokens]
    F = max(0, min(int(free_count), num))
    stack = free[:F]
    ends, total = [], 0
    for n in new_tokens:
        total += max(n, 0)
        ends.append(total)
    offsets = [0] + [min(e, T) for e in ends]
    old = [max(0, min(cap, int(x))) for x in lengths]
    new = list(old)
    for b, n in enumerate(new_tokens):
        if n < 0:
            new[b] = max(0, old[b] + n)
            stack += [table[b][j] for j in range(pages_of(new[b], size), pages_of(old[b], size))]
    have, asked = len(stack), 0
    for b, n in enumerate(new_tokens):
        if n > 0 and old[b] + n <= cap and ends[b] <= T:
            need = pages_of(old[b] + n, size) - pages_of(old[b], size)
            asked += need
            if need == 0 or asked <= have:
                new[b] = old[b] + n
                for j in range(pages_of(old[b], size), pages_of(new[b], size)):
                    table[b][j] = stack.pop()
    for j in range(F, min(len(stack), num)):
        free[j] = stack[j]
    slot, seq, pos = [-1] * T, [-1] * T, [-1] * T
    for b in range(B):
        for i in range(offsets[b], offsets[b + 1]):
            seq[i], pos[i] = b, min(old[b] + i - offsets[b], 2**31 - 1)
            if new[b] > old[b]:
                page = table[b][pos[i] // size]
                if 0 <= page < num:
                    slot[i] = page * size + pos[i] % size
    return {"block_table": table, "free_pages": free, "new_lengths": new, "new_free_count": [min(len(stack), num)],
            "granted": [y - x for x, y in zip(old, new)], "token_offsets": offsets, "slot_map": slot, "token_seq": seq,
            "token_pos": pos}


def quantise(x):
    """The append rule: int8 codes and fp32 scales of fp32 rows [..., d]."""
    x = np.asarray(x, F32)
    s = (np.abs(x).max(-1) / F32(127.0)).astype(F32)
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.rint((x / s[..., None]).astype(F32)).clip(-127, 127)
    return np.where(s[..., None] > 0, q, 0).astype(np.int8), s


def bounds(k, s):
    """k [n, d] int8, s [n] fp32 -> (bounds [2, d] int8, scale)."""
    S = np.abs(s).max() if not np.isnan(s).any() else F32(np.nan)
    if not np.isfinite(S):
        return np.stack([np.full(k.shape[1], 127), np.full(k.shape[1], -127)]).astype(np.int8), F32(np.inf)
    r = (s / S).astype(F32) if S > 0 else np.zeros_like(s)
    x = k.astype(F32) * r[:, None]  # each product rounds once, in fp32
    return np.stack([np.ceil(x.max(0)), np.floor(x.min(0))]).clip(-127, 127).astype(np.int8), F32(S)


def select(q, bound, scale, pages, keep_first, keep_last, budget):
    """q [G, d] fp32; bound [pages, 2, d], scale [pages] of a sequence's pages in order -> page entries attended."""
    if pages <= budget:
        return list(range(pages))
    code = quantise(q.reshape(1, -1))[0].reshape(q.shape).astype(np.int64)
    lim = bound.astype(np.int64)
    top = np.maximum(code[:, None] * lim[None, :, 0], code[:, None] * lim[None, :, 1]).sum(-1).max(0)
    with np.errstate(invalid="ignore", over="ignore"):
        score = top.astype(F32) * scale.astype(F32)
    score = np.where(np.isnan(score), np.inf, score)
    # NaN above +inf: rank it by a second key.
    nan = np.isnan(top.astype(F32) * scale.astype(F32)) if np.isinf(scale).any() else np.zeros(pages, bool)
    order = sorted(range(keep_first, pages - keep_last), key=lambda i: (not nan[i], -score[i], i))
    return sorted(list(range(keep_first)) + order[:budget - keep_first - keep_last] + list(range(pages - keep_last, pages)))


def attend(q, k, s, v, vs, scale):
    """q [G, d]; k, v [n, d] int8; s, vs [n] -> [G, d] in float64."""
    k = k.astype(np.float64) * s.astype(np.float64)[:, None]
    v = v.astype(np.float64) * vs.astype(np.float64)[:, None]
    x = q.astype(np.float64) @ k.T * scale
    p = np.exp(x - x.max(-1, keepdims=True))
    return (p / p.sum(-1, keepdims=True)) @ v


def attend_tolerance(q, k, s, v, vs, scale):
    """How far an fp32 kernel may be from attend(), for its G rows.

    A score is off by at most e = scale * (2^-22 max|q| + (d + 4) 2^-24 max|q|) * max_t |k_t|_1: q's fixed-point form
    and d + 4 fp32 roundings (products, sums, scalings).  Off scores move each weight by a factor within exp(+-2 e),
    about 1 +- 3 e while e is small; n weights and products then round n + 8 times in fp32, and a weight is kept to
    2^-17 of the largest.  Everything is at most max|v|."""
    d, n = k.shape[1], k.shape[0]
    norm = (np.abs(k.astype(np.float64)).sum(1) * np.abs(s)).max()
    e = scale * np.abs(q).max() * (2.0**-22 + (d + 4) * 2.0**-24) * norm
    top = (np.abs(v.astype(np.float64)).max(1) * np.abs(vs)).max()
    return float((3 * e + (n + 8) * 2.0**-24 + 2.0**-17) * top)
