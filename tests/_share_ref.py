"""Plain restatements of chunk attention and of the operators on shared pages, in
Python integers and float64, written from the definitions in include/kvq.h; and
the batches that their tests use.  Test infrastructure."""
from __future__ import annotations

import numpy as np
import torch

from _paged_ref import pages_of


# ---------------------------------------------------------------------------
# chunk attention
# ---------------------------------------------------------------------------
def attend(q, k, v, scale, keys, bf16):
    """Rows q [n, d] over tokens k, v [L, d] (float64 values), row i over the first keys[i] of them.

    Returns the float64 result and how far a right kernel may be off:
    * a score: products of codes and q are exact or off by q's limbs (2^-23 of each), their fp32 sums round at most d +
      24 times (the generic kernel once an element, matrix cores less) by 2^-24 of the sum of magnitudes, and the scales
      six times;
    * a weight: ln 2 of its score's error, in log2 units, 2^-21 for the exponential, and its rounding to f16 limbs:
      2^-11 for bf16, 2^-22 for fp32, or 2^-36 of the largest where the limb is subnormal;
    * the sums: one rounding of 2^-23 for each 16 keys and a few for the join;
    * the output: half a step of its type."""
    n, L = q.shape[0], k.shape[0]
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    d = q.shape[1]
    if L == 0:
        return out, tol
    t = torch.arange(L, device=q.device)
    there = t < keys[:, None]
    s = torch.where(there, q @ k.T.contiguous() * scale, -torch.inf)
    mag = q.abs() @ k.abs().T.contiguous() * scale
    some = keys > 0
    p = torch.where(some[:, None], s, 0.0).softmax(-1) * there
    eps = mag * ((d + 24) * 2.0**-24 + 2.0**-23 + 6 * 2.0**-24) + 2.0**-21 + (2.0**-11 if bf16 else 2.0**-22)
    size = p @ v.abs()
    err = (p * eps) @ v.abs() + (p * eps).sum(-1, keepdim=True) * size
    err += size * ((L / 16 + 24) * 2.0**-23) + L * 2.0**-36 * (p[..., None] * v.abs() if n * L * d < 1 << 24 else size[:, None]).amax(1)
    out = torch.where(some[:, None], p @ v, 0.0)
    return out, torch.where(some[:, None], err + out.abs() * (2.0**-8 if bf16 else 2.0**-24), 0.0)


def values(codes, scales, table, length):
    """float64 rows [Hkv, length, d] of one sequence of a pool [P, Hkv, page, d]."""
    page = codes.shape[2]
    at = table[:pages_of(length, page)].long()
    x = codes[at].double() * scales[at].double()[..., None]
    return x.transpose(0, 1).flatten(1, 2)[:, :length]


def chunk(i, causal, scale=None):
    """Rows of a batch (tensors as kvq.ChunkAttention takes them): float64 result, tolerance, and which rows are written."""
    q, lengths, offsets = i["q"], i["lengths"].tolist(), i["token_offsets"].tolist()
    granted = i["granted"].tolist() if i.get("granted") is not None else [1] * len(lengths)
    T, Hq, d = q.shape
    Hkv = i["k"].shape[1]
    G = Hq // Hkv
    scale = 1 / np.sqrt(d) if scale is None else scale
    out = torch.zeros((T, Hq, d), dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    written = torch.zeros(T, dtype=torch.bool, device=q.device)
    for b, length in enumerate(lengths):
        r0, r1 = offsets[b], offsets[b + 1]
        n = r1 - r0
        written[r0:r1] = True
        if n == 0 or granted[b] <= 0 or length == 0:
            continue
        k, v = (values(i[c], i[c + "s"], i["block_table"][b], length) for c in "kv")
        at = torch.arange(n, device=q.device)
        keys = (length - n + at + 1).clamp(min=0) if causal else torch.full_like(at, length)
        for h in range(Hkv):
            x = q[r0:r1, h * G:(h + 1) * G].double().flatten(0, 1)
            o, e = attend(x, k[h], v[h], scale, keys.repeat_interleave(G), q.dtype == torch.bfloat16)
            out[r0:r1, h * G:(h + 1) * G], tol[r0:r1, h * G:(h + 1) * G] = o.view(n, G, d), e.view(n, G, d)
    return out, tol, written


def batch(seed, pairs, Hq, Hkv, d, page, dtype, spare=3, fused=False, refused=(), device="cuda"):
    """A batch of (length, new tokens) over a shuffled pool; what no token holds is garbage: NaN scales, wild ids."""
    rng = np.random.default_rng(seed)
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    B = len(pairs)
    lens, new = [x for x, _ in pairs], [n for _, n in pairs]
    used = [pages_of(x, page) for x in lens]
    P = sum(used) + 4
    per = max(max(used), 1) + 2
    ids = rng.permutation(P)
    table = rng.integers(-9, 3 * P, (B, per))
    at = 0
    for b in range(B):
        table[b, :used[b]] = ids[at:at + used[b]]
        at += used[b]
    i = {"block_table": torch.from_numpy(table.astype(np.int32)).to(device)}
    for c in "kv":
        i[c] = torch.randint(-127, 128, (P, Hkv, page, d), generator=g, dtype=torch.int8, device=device)
        s = torch.rand((P, Hkv, page), generator=g, device=device) * 0.02 + 0.005
        held = torch.zeros((P, page), dtype=torch.bool, device=device)
        for b in range(B):
            for j in range(used[b]):
                held[table[b, j], :lens[b] - j * page] = True
        i[c + "s"] = torch.where(held[:, None], s, float("nan"))
    T = sum(new) + spare
    cols = (Hq + 2 * Hkv) * d if fused else Hq * d
    i["q"] = (torch.randn((T, cols), generator=g, device=device) * 1.5).to(dtype)[:, :Hq * d].unflatten(1, (Hq, d))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    i["lengths"], i["token_offsets"] = i32(lens), i32(np.concatenate([[0], np.cumsum(new)]).astype(int).tolist())
    i["granted"] = i32([0 if b in refused else n for b, n in enumerate(new)]) if refused else None
    i["out"] = torch.full((T, Hq, d), float("nan"), dtype=dtype, device=device)
    return i


# ---------------------------------------------------------------------------
# forks and compaction
# ---------------------------------------------------------------------------
def fork(st, size):
    """One row after the other; the free stack as a list, a page's holders counted from the tables and `shares`."""
    table = [list(r) for r in st["block_table"]]
    B, cap, num = len(table), len(table[0]) * size, len(st["free_pages"])
    old = [max(0, min(cap, x)) for x in st["lengths"]]
    parents = [p if 0 <= p < B else -1 for p in st["parents"]]
    keep = st.get("keep")
    new = [0 if p < 0 else old[p] if keep is None else min(old[p], max(0, keep[b])) for b, p in enumerate(parents)]
    rows = [[] if p < 0 else table[p][:pages_of(n, size)] for p, n in zip(parents, new)]
    held = [s + 1 for s in st["shares"]]
    touched = [False] * num
    for b in range(B):
        for page in table[b][:pages_of(old[b], size)]:
            if 0 <= page < num:
                held[page] -= 1
                touched[page] = True
        for page in rows[b]:
            if 0 <= page < num:
                held[page] += 1
    F = max(0, min(num, st["free_count"][0]))
    free = list(st["free_pages"])
    stack = free[:F] + [p for p in range(num) if touched[p] and held[p] <= 0]
    enders = {}
    for b in range(B):
        if new[b] % size and 0 <= rows[b][-1] < num:
            enders.setdefault(rows[b][-1], []).append(b)
    before = list(held)
    src, dst, left = [-1] * B, [-1] * B, len(stack)
    for b in range(B):
        if not new[b] % size or not 0 <= rows[b][-1] < num:
            continue
        page = rows[b][-1]
        if before[page] <= 1 or (before[page] <= len(enders[page]) and enders[page][0] == b):
            continue
        held[page] -= 1
        if left:
            left -= 1
            src[b], dst[b] = page, stack[left]
            rows[b][-1] = stack[left]
        else:
            rows[b].pop()
            new[b] -= new[b] % size
    for i in range(F, left):
        free[i] = stack[i]
    shares = [max(0, h - 1) for h in held]
    for p in dst:
        if p >= 0:
            shares[p] = 0
    return {"new_lengths": new, "rows": rows, "new_shares": shares, "new_free_count": [left], "copy_src": src,
            "copy_dst": dst, "free_pages": free}


def compact(st, size, moves):
    table = [list(r) for r in st["block_table"]]
    num, cap = len(st["free_pages"]), len(table[0]) * size
    F = max(0, min(num, st["free_count"][0]))
    free = set(st["free_pages"][:F])
    used = num - len(free)
    holes = sorted(p for p in free if p < used)
    highs = sorted((p for p in range(used, num) if p not in free), reverse=True)
    n = min(len(holes), moves)
    to = dict(zip(highs[:n], holes[:n]))
    rows = [[to.get(p, p) for p in r[:pages_of(max(0, min(cap, x)), size)]] for r, x in zip(table, st["lengths"])]
    shares = [0] * num
    if st.get("shares") is not None:
        for p in range(num):
            if p not in free:
                shares[to.get(p, p)] = st["shares"][p]
    left = sorted((free - set(holes[:n])) | set(highs[:n]), reverse=True)
    return {"rows": rows, "new_shares": shares, "free_pages": left, "moved": [n],
            "copy_src": highs[:n] + [-1] * (moves - n), "copy_dst": holes[:n] + [-1] * (moves - n)}
