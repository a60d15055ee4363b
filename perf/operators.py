"""The paged cache's operators as a serving program calls them, measured against plain torch.

  map     kvq.PageMapper: block tables, free pages and slot maps from request lengths
  write   kvq.slot_write: a packed batch of K/V rows quantised into the pages its slots name; the
          rows are read back (kvq.slot_read), since what a cache holds is the values its codes stand for
  read    kvq.slot_read: cached tokens as fp32 or bf16 rows, for the dense attention of a prompt
          that continues them
  bounds  kvq.page_bounds: per page and kv head, int8 bounds of its keys
  sparse  kvq.SparseDecoder: one decode step over the pages that the bounds rank highest

Every run leaves its inputs as they were, or writes the same values again, so passes are alike.
"""
import importlib
import math

import numpy as np
import torch

own = False

DEV = "cuda"
CHUNK = 1 << 26  # elements drawn at a time
NONE = -1


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _map(B, page, hi, new):
    """B sequences of up to hi tokens; up to `new` more each (1: a decode step)."""
    return {"op": "map", "B": B, "page": page, "hi": hi, "new": new}


def _write(B, L, Hkv, d, dtype, page, fused):
    """B prompts of up to L tokens; fused: rows are slices of one q/k/v projection."""
    return {"op": "write", "B": B, "L": L, "Hkv": Hkv, "d": d, "dtype": dtype, "page": page, "fused": fused}


def _read(B, L, Hkv, d, dtype, page):
    return {"op": "read", "B": B, "L": L, "Hkv": Hkv, "d": d, "dtype": dtype, "page": page}


def _bounds(B, lo, hi, Hkv, d, page):
    return {"op": "bounds", "B": B, "lo": lo, "hi": hi, "Hkv": Hkv, "d": d, "page": page}


def _sparse(B, Hq, Hkv, d, lo, hi, page, budget, dist):
    return {"op": "sparse", "B": B, "Hq": Hq, "Hkv": Hkv, "d": d, "lo": lo, "hi": hi, "page": page,
            "budget": budget, "dist": dist}


def listed():
    return [
        # Before every decode step of a serving batch: a token more for most
        # sequences, some end and give their pages back.  The call's latency counts.
        dict(_map(256, 16, 4096, 1), name="map_b256_step"),
        # A round of prompts is admitted: tens of thousands of packed rows get slots.
        dict(_map(64, 64, 2048, 2047), name="map_b64_prompts"),
        # One short prompt.
        dict(_write(1, 33, 8, 128, "bf16", 16, False), name="write_b1_l33_bf16_page16"),
        # A round of prompts of unequal lengths, rows still in the projection's output.
        dict(_write(16, 2047, 8, 128, "bf16", 64, True), name="write_b16_l2047_bf16_page64"),
        # A conversation goes on: its cached turns in fp32 for the prompt's dense attention.
        dict(_read(1, 4099, 8, 128, "f32", 16), name="read_b1_l4099_f32_page16"),
        # The cached prefixes of a batch, in bf16.
        dict(_read(16, 8192, 8, 128, "bf16", 64), name="read_b16_l8192_bf16_page64"),
        # Bounds of one prompt that has just been written.
        dict(_bounds(1, 1300, 1300, 8, 128, 16), name="bounds_b1_l1300_page16"),
        # Bounds of a round of long prompts.
        dict(_bounds(16, 1024, 8192, 8, 128, 64), name="bounds_b16_l8192_page64"),
        # One very long context; keys with outlier channels, as trained models have.
        dict(_sparse(1, 32, 8, 128, 131072, 131072, 64, 64, "outlier"), name="sparse_b1_h32_8_l131072"),
        # A batch of long, unequal contexts of a grouped-query model.
        dict(_sparse(16, 32, 8, 128, 4096, 32768, 32, 128, "outlier"), name="sparse_b16_h32_8_l32768"),
        # A multi-head model, a small batch.
        dict(_sparse(8, 32, 32, 128, 4096, 16384, 16, 128, "normal"), name="sparse_b8_h32_l16384_page16"),
        # Three query heads per kv head, a head dim between the powers of two, heavy tails.
        dict(_sparse(4, 24, 8, 96, 500, 9001, 16, 64, "student_t"), name="sparse_b4_h24_8_d96"),
    ]


MAX_BYTES = 3.5e8  # of rows or cache that a drawn case reads and writes


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["map", "map", "write", "write", "read", "bounds", "sparse", "sparse", "sparse", "sparse"])
    page = rng.choice([16, 16, 32, 64, 128])
    if op == "map":
        new = rng.choice([1, 1, 8]) if rng.random() < 0.5 else _log_int(rng, 16, 2047)
        B = _log_int(rng, 1, 1024)
        return _map(max(1, min(B, 131072 // new)), page, _log_int(rng, 64, 4096), new)
    d = rng.choice([64, 80, 96, 112, 128, 128, 128, 192, 256])
    Hkv = rng.choice([1, 2, 4, 8, 8, 8, 16, 32])
    if op in ("write", "read"):
        dtype = rng.choice(["f32", "bf16", "bf16"])
        L, B = _log_int(rng, 1, 8192), _log_int(rng, 1, 64)
        B = max(1, min(B, int(MAX_BYTES / (2 * Hkv * L * d * (5 if dtype == "f32" else 3)))))
        if op == "read":
            return _read(B, L, Hkv, d, dtype, page)
        return _write(B, L, Hkv, d, dtype, page, rng.random() < 0.5)
    B, hi = _log_int(rng, 1, 64), _log_int(rng, 64, 32768)
    lo = max(1, hi // rng.choice([1, 2, 4, 8]))
    if op == "bounds":
        B = max(1, min(B, int(MAX_BYTES / (hi * Hkv * d))))
        return _bounds(B, lo if B > 1 else hi, hi, Hkv, d, page)
    G = rng.choice([1, 2, 3, 4, 4, 5, 6, 7, 8, 8, 16])
    Hkv = rng.choice([8, 16, 32, 40]) if G == 1 else rng.choice([1, 2, 4, 8, 8, 8])
    budget = max(2, _log_int(rng, 128, 4096) // page)
    token = Hkv * (2 * d + 8)
    B = max(1, min(B, int(3 * MAX_BYTES / (hi * token)), int(MAX_BYTES / (min(hi, budget * page) * token))))
    return _sparse(B, G * Hkv, Hkv, d, lo if B > 1 else hi, hi, page, budget, rng.choice(["normal", "outlier", "student_t"]))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _dev(a, dtype=np.int32):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=dtype)).to(DEV)


def _dtype(case):
    return torch.float32 if case["dtype"] == "f32" else torch.bfloat16


def _values(gen, shape, dist):
    x = torch.randn(shape, generator=gen, device=DEV)
    if dist == "student_t":  # 4 degrees of freedom
        chi = torch.randn(shape, generator=gen, device=DEV).square_()
        for _ in range(3):
            chi += torch.randn(shape, generator=gen, device=DEV).square_()
        x = x.div_(chi.div_(4.0).sqrt_())
    return x


def _gain(gen, H, d):
    """One channel in a hundred 20 times the others."""
    g = torch.ones((H, d), device=DEV)
    pick = torch.rand((H, d), generator=gen, device=DEV).argsort(1)[:, :max(1, math.ceil(0.01 * d))]
    return g.scatter_(1, pick, 20.0)


def _pool(gen, X, H, T, d, dist, gain=None):
    """int8 rows [X, H, T, d] and fp32 scales [X, H, T], as a per-token quantiser leaves them."""
    q = torch.empty((X, H, T, d), dtype=torch.int8, device=DEV)
    s = torch.empty((X, H, T), dtype=torch.float32, device=DEV)
    step = max(1, CHUNK // (H * T * d))
    for i in range(0, X, step):
        x = _values(gen, (min(step, X - i), H, T, d), dist)
        if gain is not None:
            x *= gain[:, None, :]
        s[i:i + step] = x.abs().amax(-1) / 127.0
        q[i:i + step] = (x / s[i:i + step, :, :, None]).round_().clamp_(-127.0, 127.0).to(torch.int8)
    return q, s


def _spread(rng, lo, hi, B):
    """B lengths evenly spread over [lo, hi], in an order of the seed (their sum is the case's)."""
    n = np.linspace(lo, hi, B).round().astype(np.int64) if B > 1 else np.array([hi], np.int64)
    return rng.permutation(n)


def _table(rng, B, per):
    """Block table [B, per] over a shuffled pool with a few pages to spare, and the pool's pages."""
    pool = B * per + 7
    return rng.permutation(pool)[:B * per].reshape(B, per), pool


def _map_inputs(case, seed):
    """A pool in use: sequences of unequal lengths, shuffled pages, others on the free stack, the rest in other hands.

    One pool in four has too few free pages for the whole round."""
    rng = np.random.default_rng(seed)
    B, page, hi, new = (case[k] for k in ("B", "page", "hi", "new"))
    per = -(-(hi + new) // page)
    if new == 1:
        lens = rng.integers(1, hi + 1, B)
        add = np.ones(B, np.int64)
    else:  # prompts: most sequences are new ones
        lens = np.where(rng.random(B) < 0.7, 0, rng.integers(1, hi + 1, B))
        add = rng.integers(max(1, new // 2), new + 1, B)
    fate = rng.random(B)
    add = np.where(fate < 0.05, 0, add)                              # waits
    add = np.where((fate >= 0.05) & (fate < 0.12), -lens, add)       # ends
    add = np.where((fate >= 0.12) & (fate < 0.15), -np.minimum(lens, 5), add)  # takes tokens back
    used = -(-lens // page)
    need = np.maximum(-(-(lens + add) // page) - used, 0).sum()
    num = B * per
    ids = rng.permutation(num)
    count = min(num - used.sum(), need + 5 if seed % 4 else need // 2)
    table = np.zeros((B, per), np.int64)
    fill = np.arange(per)[None] < used[:, None]
    table[fill] = ids[:used.sum()]
    free = np.zeros(num, np.int64)
    free[:count] = ids[used.sum():used.sum() + count]
    rows = max(1, B * new)
    e = lambda *s: torch.empty(s, dtype=torch.int32, device=DEV)  # noqa: E731
    return {"new_tokens": _dev(add), "lengths": _dev(lens), "block_table": _dev(table), "free_pages": _dev(free),
            "free_count": _dev([count]), "new_lengths": e(B), "new_free_count": e(1), "granted": e(B),
            "token_offsets": e(B + 1), "slot_map": e(rows), "token_seq": e(rows), "token_pos": e(rows)}


def _slots(rng, case):
    """Slots of B sequences' tokens laid end to end, in shuffled pages; and the pool's pages."""
    page = case["page"]
    lens = _spread(rng, max(1, case["L"] // 2), case["L"], case["B"])
    per = -(-case["L"] // page)
    table, pool = _table(rng, case["B"], per)
    seq = np.repeat(np.arange(case["B"]), lens)
    pos = np.concatenate([np.arange(n) for n in lens])
    return table[seq, pos // page] * page + pos % page, pool


def _write_inputs(case, seed):
    slots, pool = _slots(np.random.default_rng(seed), case)
    gen, T, Hkv, d, page = _gen(seed), len(slots), case["Hkv"], case["d"], case["page"]
    slots[::97] = NONE  # rows that belong to no sequence
    cols = 6 * Hkv * d if case["fused"] else 2 * Hkv * d  # q of four heads per kv head stands before k and v
    x = (torch.randn((T, cols), generator=gen, device=DEV) * 3.0).to(_dtype(case))
    k, v = (c.view(T, Hkv, d) if not case["fused"] else c.unflatten(1, (Hkv, d)) for c in x[:, -2 * Hkv * d:].split(Hkv * d, 1))
    if not case["fused"]:
        k, v = k.contiguous(), v.contiguous()
    i = {"k_new": k, "v_new": v, "slots": _dev(slots)}
    i.update(_empty_pool(pool, Hkv, page, d))
    i["k_out"], i["v_out"] = (torch.empty((T, Hkv, d), dtype=_dtype(case), device=DEV) for _ in "kv")
    return i


def _empty_pool(pool, Hkv, page, d):
    """An empty pool; the row behind its last one, "k_rows"[-1] and so on, belongs to nobody."""
    i = {}
    for c in "kv":
        i[c + "_rows"] = torch.zeros((pool * Hkv * page + 1, d), dtype=torch.int8, device=DEV)
        i[c + "s_rows"] = torch.zeros(pool * Hkv * page + 1, device=DEV)
        i[c], i[c + "s"] = i[c + "_rows"][:-1].view(pool, Hkv, page, d), i[c + "s_rows"][:-1].view(pool, Hkv, page)
    return i


def _read_inputs(case, seed):
    slots, pool = _slots(np.random.default_rng(seed), case)
    gen, T, Hkv, d = _gen(seed), len(slots), case["Hkv"], case["d"]
    slots[::101] = NONE
    i = {"slots": _dev(slots)}
    i["k"], i["ks"] = _pool(gen, pool, Hkv, case["page"], d, "normal")
    i["v"], i["vs"] = _pool(gen, pool, Hkv, case["page"], d, "normal")
    # [Hkv, T, d]: each head's rows together, as dense attention takes them.
    i["k_out"], i["v_out"] = (torch.empty((Hkv, T, d), dtype=_dtype(case), device=DEV).transpose(0, 1) for _ in "kv")
    return i


def _paged_inputs(case, seed):
    rng = np.random.default_rng(seed)
    lens = _spread(rng, case["lo"], case["hi"], case["B"])
    table, pool = _table(rng, case["B"], -(-case["hi"] // case["page"]))
    return {"lens": lens, "lengths": _dev(lens), "block_table": _dev(table)}, pool


def _bounds_inputs(case, seed):
    i, pool = _paged_inputs(case, seed)
    gen, Hkv, d = _gen(seed), case["Hkv"], case["d"]
    i["k"], i["ks"] = _pool(gen, pool, Hkv, case["page"], d, "normal", _gain(gen, Hkv, d))
    # Of the pool's pages and of one behind them that belongs to nobody.
    i["all_bounds"] = torch.zeros((pool + 1, Hkv, 2, d), dtype=torch.int8, device=DEV)
    i["all_scales"] = torch.zeros((pool + 1, Hkv), device=DEV)
    i["bounds"], i["bound_scale"] = i["all_bounds"][:-1], i["all_scales"][:-1]
    return i


def _sparse_inputs(case, seed):
    i, pool = _paged_inputs(case, seed)
    gen, B, Hq, Hkv, d, page = _gen(seed), *(case[k] for k in ("B", "Hq", "Hkv", "d", "page"))
    dist = "normal" if case["dist"] == "outlier" else case["dist"]
    i["q"] = torch.randn((B, Hq, d), generator=gen, device=DEV)
    i["k"], i["ks"] = _pool(gen, pool, Hkv, page, d, dist, _gain(gen, Hkv, d) if case["dist"] == "outlier" else None)
    i["v"], i["vs"] = _pool(gen, pool, Hkv, page, d, dist)
    i["bounds"] = torch.empty((pool, Hkv, 2, d), dtype=torch.int8, device=DEV)
    i["bound_scale"] = torch.empty((pool, Hkv), device=DEV)
    step = max(1, CHUNK // (Hkv * page * d))
    for x in range(0, pool, step):  # of whole pages; the pages that are not whole are attended without a look at them
        i["bounds"][x:x + step], i["bound_scale"][x:x + step] = _page_bounds(i["k"][x:x + step], i["ks"][x:x + step])
    i["out"] = torch.empty_like(i["q"])
    i["selected"] = torch.empty((B, Hkv, case["budget"]), dtype=torch.int32, device=DEV)
    i["selected_lengths"] = torch.empty((B, Hkv), dtype=torch.int32, device=DEV)
    return i


_INPUTS = {"map": _map_inputs, "write": _write_inputs, "read": _read_inputs, "bounds": _bounds_inputs,
           "sparse": _sparse_inputs}


def prepare(case, seed):
    return {"case": case, **_INPUTS[case["op"]](case, seed)}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    return _RUN[state["case"]["op"]](state)


def _kvq():
    return importlib.import_module("cuda-operators_amd").kvq


_MAP_ARGS = ("new_tokens", "lengths", "block_table", "free_pages", "free_count")
_MAP_OUTS = ("new_lengths", "new_free_count", "granted", "token_offsets", "slot_map", "token_seq", "token_pos")


def _run_map(i):
    if own:
        if "handle" not in i:  # a program makes it once
            i["handle"] = _kvq().PageMapper(*(i[n] for n in _MAP_ARGS), page_size=i["case"]["page"],
                                            **{n: i[n] for n in _MAP_OUTS})
        i["handle"]()
        return {n: i[n] for n in ("block_table", "free_pages") + _MAP_OUTS}
    page, table, free = i["case"]["page"], i["block_table"].long(), i["free_pages"].long()
    B, per = table.shape
    num, T = free.numel(), i["slot_map"].numel()
    cap = per * page
    old, n = i["lengths"].long().clamp(0, cap), i["new_tokens"].long()
    pages = lambda x: (x + page - 1) // page  # noqa: E731
    end = n.clamp(min=0).cumsum(0)
    offs = torch.cat([end.new_zeros(1), end]).clamp(max=T)
    want = (old + n).clamp(min=0)
    want = torch.where((n > 0) & ((want > cap) | (end > T)), old, want)
    delta = pages(want) - pages(old)
    need, gone = delta.clamp(min=0), (-delta).clamp(min=0)
    F = i["free_count"].long().clamp(0, num)
    have = F + gone.sum()
    ok = (need == 0) | (need.cumsum(0) <= have)
    new = torch.where(ok, want, old)
    need = torch.where(ok, need, 0)
    col = torch.arange(per, device=DEV)[None]
    # The free stack with the released pages on it (a masked entry goes past its end).
    stack = torch.cat([free, free.new_zeros(B * per + 1)])
    released = (col >= pages(new)[:, None]) & (col < pages(old)[:, None])
    at = F + (gone.cumsum(0) - gone)[:, None] + col - pages(new)[:, None]
    stack[torch.where(released, at, num + B * per)] = table
    added = (col >= pages(old)[:, None]) & (col < pages(new)[:, None])
    at = have - 1 - (need.cumsum(0) - need)[:, None] - col + pages(old)[:, None]
    table = torch.where(added, stack[torch.where(added, at, 0)], table)
    count = have - need.sum()
    j = torch.arange(num, device=DEV)
    free = torch.where((j >= F) & (j < count), stack[:num], free)
    t = torch.arange(T, device=DEV)
    seq = torch.searchsorted(offs[1:], t, right=True).clamp(max=B - 1)
    row = t - offs[seq]
    used = t < offs[B]
    pos = old[seq] + row
    held = used & (row < (new - old)[seq])
    page_of = table[seq, (pos // page).clamp(max=per - 1)]
    i32 = lambda x: x.to(torch.int32)  # noqa: E731
    return {"block_table": i32(table), "free_pages": i32(free), "new_lengths": i32(new), "new_free_count": i32(count),
            "granted": i32(new - old), "token_offsets": i32(offs),
            "slot_map": i32(torch.where(held, page_of * page + pos % page, NONE)),
            "token_seq": i32(torch.where(used, seq, NONE)), "token_pos": i32(torch.where(used, pos, NONE))}


def _over_127(x):
    """x / 127 with the division itself (a plain number's reciprocal would be multiplied in)."""
    return x / torch.full_like(x, 127.0)


def _quantise(x):
    """Codes (as fp32) and scales of rows [..., d]."""
    x = x.float()
    s = _over_127(x.abs().amax(-1))
    return torch.where(s[..., None] > 0, (x / s[..., None]).round().clamp(-127.0, 127.0), 0.0), s


def _plain_read(i, dtype):
    """Values [T, Hkv, d] of K and V at the slots."""
    page = i["case"]["page"]
    at = i["slots"].long().clamp(min=0)
    p, o, there = at // page, at % page, (i["slots"] >= 0)[:, None, None]
    return [torch.where(there, i[c][p, :, o].float() * i[s][p, :, o][..., None], 0.0).to(dtype) for c, s in (("k", "ks"), ("v", "vs"))]


def _run_write(i):
    if own:
        kvq = _kvq()
        kvq.slot_write(i["k_new"], i["v_new"], i["slots"], i["k"], i["v"], i["ks"], i["vs"])
        kvq.slot_read(i["slots"], i["k"], i["v"], i["ks"], i["vs"], i["k_out"], i["v_out"])
        return {"k": i["k_out"], "v": i["v_out"], "k_scale": i["ks"], "v_scale": i["vs"]}
    page, slots = i["case"]["page"], i["slots"].long()
    P, Hkv = i["k"].shape[:2]
    row = ((slots // page)[:, None] * Hkv + torch.arange(Hkv, device=DEV)) * page + (slots % page)[:, None]
    row = torch.where((slots >= 0)[:, None], row, P * Hkv * page)  # without a slot: behind the pool
    for c in "kv":
        code, scale = _quantise(i[c + "_new"])
        i[c + "_rows"][row], i[c + "s_rows"][row] = code.to(torch.int8), scale
    k, v = _plain_read(i, _dtype(i["case"]))
    return {"k": k, "v": v, "k_scale": i["ks"], "v_scale": i["vs"]}


def _run_read(i):
    if own:
        _kvq().slot_read(i["slots"], i["k"], i["v"], i["ks"], i["vs"], i["k_out"], i["v_out"])
        return {"k": i["k_out"], "v": i["v_out"]}
    k, v = _plain_read(i, _dtype(i["case"]))
    return {"k": k, "v": v}


def _page_bounds(k, ks, there=None):
    """k [..., page, d] int8, ks [..., page] -> bounds [..., 2, d] int8 and scales [...]; there: which rows count."""
    if there is not None:
        ks = torch.where(there, ks, 0.0)
    s = ks.abs().amax(-1)
    x = k.float() * torch.where(s[..., None] > 0, ks / s[..., None], 0.0)[..., None]
    hi, lo = x, x
    if there is not None:
        hi, lo = torch.where(there[..., None], x, -math.inf), torch.where(there[..., None], x, math.inf)
    return torch.stack([hi.amax(-2).ceil(), lo.amin(-2).floor()], -2).clamp(-127.0, 127.0).to(torch.int8), s


def _run_bounds(i):
    if own:
        _kvq().page_bounds(i["k"], i["ks"], i["block_table"], i["lengths"], i["bounds"], i["bound_scale"],
                           max_seq_len=i["case"]["hi"])
    else:
        page, table = i["case"]["page"], i["block_table"]
        per = table.shape[1]
        tokens = (i["lengths"][:, None] - torch.arange(per, device=DEV) * page).flatten()  # of each table entry
        ids = table.flatten().long()
        there = (torch.arange(page, device=DEV) < tokens[:, None, None]).expand(-1, i["k"].shape[1], -1)
        to = torch.where(tokens > 0, ids, i["k"].shape[0])  # an unused entry: behind the pool
        i["all_bounds"][to], i["all_scales"][to] = _page_bounds(i["k"][ids], i["ks"][ids], there)
    return {"values": i["bounds"] * i["bound_scale"][..., None, None], "scale": i["bound_scale"]}


def _run_sparse(i):
    c = i["case"]
    if own:
        if "handle" not in i:  # a program makes it once
            i["handle"] = _kvq().SparseDecoder(i["q"], i["k"], i["v"], i["ks"], i["vs"], i["block_table"], i["lengths"],
                                               i["bounds"], i["bound_scale"], i["out"], i["selected"],
                                               i["selected_lengths"], max_seq_len=c["hi"], keep_first=1, keep_last=1)
        i["handle"]()
        return {n: i[n] for n in ("out", "selected", "selected_lengths")}
    B, Hq, Hkv, d, page, budget = (c[k] for k in ("B", "Hq", "Hkv", "d", "page", "budget"))
    G, table, per = Hq // Hkv, i["block_table"].long(), i["block_table"].shape[1]
    n = i["lengths"].long()
    pages = (n + page - 1) // page
    # Scores: whole numbers below 2^24, which fp32 sums hold; one rounding by the page's scale.
    q = i["q"].view(B, Hkv, G * d)
    code = _quantise(q)[0].view(B, Hkv, G, d)
    both = torch.cat([code.clamp(min=0), code.clamp(max=0)], -1)
    lim = i["bounds"][table].transpose(1, 2).flatten(3).float()  # [B, Hkv, per, 2 d]
    top = torch.matmul(lim, both.transpose(2, 3).contiguous()).amax(-1)
    score = top * i["bound_scale"][table].transpose(1, 2)
    # The first and the last page first of all, what is not there last.
    j = torch.arange(per, device=DEV)
    kept = (j == 0) | (j == pages[:, None] - 1)
    score = torch.where(kept[:, None], math.inf, score)
    score = torch.where((j < pages[:, None])[:, None], score, -math.inf)
    width = min(budget, per)
    pick = score.sort(dim=-1, descending=True, stable=True)[1][..., :width]
    took = torch.minimum(pages, torch.full_like(pages, budget))
    pick = torch.where((torch.arange(width, device=DEV) < took[:, None])[:, None], pick, per).sort(-1)[0]
    real = pick < per
    ids = torch.gather(table, 1, pick.clamp(max=per - 1).flatten(1)).view(pick.shape)
    h = torch.arange(Hkv, device=DEV)[:, None]
    rows = ids * Hkv + h
    selected = torch.full((B, Hkv, budget), NONE, dtype=torch.int32, device=DEV)
    selected[..., :width] = torch.where(real, rows, NONE).to(torch.int32)
    count = ((took - 1) * page + (n - 1) % page + 1)[:, None].expand(B, Hkv)
    # Attention over the selected pages.
    pool = lambda x: x.flatten(0, 1)[rows].flatten(2, 3)  # noqa: E731
    pos = (pick[..., None] * page + torch.arange(page, device=DEV)).flatten(2)
    there = (pos < n[:, None, None]) & real.repeat_interleave(page, -1)
    k = pool(i["k"]).float() * pool(i["ks"])[..., None]
    s = torch.matmul(i["q"].view(B, Hkv, G, d), k.transpose(2, 3).contiguous()) / math.sqrt(d)
    s = torch.where(there[:, :, None], s, -math.inf)
    p = (s - s.amax(-1, keepdim=True)).exp()
    v = pool(i["v"]).float() * pool(i["vs"])[..., None]
    out = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    return {"out": out.view(B, Hq, d), "selected": selected, "selected_lengths": count.to(torch.int32)}


_RUN = {"map": _run_map, "write": _run_write, "read": _run_read, "bounds": _run_bounds, "sparse": _run_sparse}


# ---------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------
def _ieee_codes(x):
    """The quantiser's codes and scales, rounded in fp32 as its rule says (on the CPU), as 64-bit values."""
    x = x.float().cpu()
    s = x.abs().amax(-1) / 127.0
    code = (x / s[..., None]).round().clamp(-127.0, 127.0)
    code[s == 0] = 0.0
    return code.double(), s.double()


def _exact_write(case, seed):
    i = _write_inputs(case, seed)
    slots = i["slots"].cpu().long()
    got = {}
    for c, x in (("k", i["k_new"]), ("v", i["v_new"])):
        code, s = _ieee_codes(x)
        value = code * s[..., None]
        value[slots < 0] = 0.0
        got[c] = value
        scales = torch.zeros(i[c + "s"].shape, dtype=torch.float64)
        at = slots[slots >= 0]
        scales[at // case["page"], :, at % case["page"]] = s[slots >= 0]
        got[c + "_scale"] = scales
    return got


def _exact_read(case, seed):
    i = _read_inputs(case, seed)
    got = {}
    for c in ("k", "v"):
        rows = i[c].transpose(1, 2).flatten(0, 1)  # [slot, Hkv, d]
        scales = i[c + "s"].transpose(1, 2).flatten(0, 1)
        at = i["slots"].long()
        value = rows[at].double() * scales[at].double()[..., None]  # slot -1: the last one, taken out again
        value[at < 0] = 0.0
        got[c] = value
    return got


def _bounds_of(k, s):
    """Bounds [2, d] (whole numbers) and scale of one page's keys [n, d] and scales [n]: the ratio and the product are
    fp32 roundings by definition, the rest is exact."""
    top = s.abs().max()
    x = (k.float() * (s / top)[:, None]).double() if float(top) > 0 else torch.zeros(k.shape, dtype=torch.float64)
    return torch.stack([x.max(0)[0].ceil(), x.min(0)[0].floor()]), top.double()


def _exact_bounds(case, seed):
    i = _bounds_inputs(case, seed)
    page, Hkv = case["page"], case["Hkv"]
    if int((-(-i["lens"] // page)).sum()) * Hkv > 60000:  # one at a time on the CPU: minutes
        return None
    k, s, table = i["k"].cpu(), i["ks"].cpu(), i["block_table"].cpu()
    values = torch.zeros(i["bounds"].shape, dtype=torch.float64)
    scale = torch.zeros(i["bound_scale"].shape, dtype=torch.float64)
    for b, n in enumerate(int(x) for x in i["lens"]):
        for j in range(-(-n // page)):
            x, m = int(table[b, j]), min(page, n - j * page)
            for h in range(Hkv):
                lim, top = _bounds_of(k[x, h, :m], s[x, h, :m])
                values[x, h], scale[x, h] = lim * top, top
    return {"values": values, "scale": scale}


def _exact_sparse(case, seed):
    i = _sparse_inputs(case, seed)
    B, Hq, Hkv, d, page, budget = (case[k] for k in ("B", "Hq", "Hkv", "d", "page", "budget"))
    G = Hq // Hkv
    codes = _ieee_codes(i["q"].view(B, Hkv, G * d))[0].view(B, Hkv, G, d).numpy().astype(np.int64)
    table = i["block_table"].cpu().numpy()
    out = torch.empty((B, Hkv, G, d), dtype=torch.float64, device=DEV)
    for b, n in enumerate(int(x) for x in i["lens"]):
        pages = -(-n // page)
        ids = table[b, :pages]
        lim = i["bounds"][_dev(ids, np.int64)].cpu().numpy().astype(np.int64)
        scale = i["bound_scale"][_dev(ids, np.int64)].cpu().numpy()
        for h in range(Hkv):
            if pages > budget:
                best = np.maximum(codes[b, h, :, None] * lim[None, :, h, 0], codes[b, h, :, None] * lim[None, :, h, 1]).sum(-1).max(0)
                score = best.astype(np.float32) * scale[:, h]
                order = 1 + np.argsort(-score[1:pages - 1], kind="stable")[:budget - 2]
                chosen = np.sort(np.concatenate([[0], order, [pages - 1]]))
            else:
                chosen = np.arange(pages)
            at = _dev(ids[chosen], np.int64)
            m = (len(chosen) - 1) * page + (n - 1) % page + 1
            k, v = (i[c][at, h].reshape(-1, d)[:m].double() * i[s][at, h].reshape(-1)[:m].double()[:, None] for c, s in (("k", "ks"), ("v", "vs")))
            s = i["q"][b].view(Hkv, G, d)[h].double() @ k.T.contiguous() / math.sqrt(d)
            out[b, h] = s.softmax(-1) @ v
    return {"out": out.view(B, Hq, d), "selected": None, "selected_lengths": None}


def exact(case, seed):
    if case["op"] == "map":  # whole numbers alone
        return None
    return {"write": _exact_write, "read": _exact_read, "bounds": _exact_bounds, "sparse": _exact_sparse}[case["op"]](case, seed)


# ---------------------------------------------------------------------------
# work
# ---------------------------------------------------------------------------
def work(case):
    rng = np.random.default_rng(0)
    if case["op"] == "map":
        B, rows = case["B"], case["B"] * case["new"]
        pages = max(B // case["page"], rows // case["page"])  # moved between the table and the stack, either way
        return {"bytes": 4 * (2 * B + 1) + 4 * (3 * B + 2) + 12 * rows + 8 * pages, "flops": 0}
    page, Hkv, d = case["page"], case["Hkv"], case["d"]
    if case["op"] in ("write", "read"):
        tokens = int(_spread(rng, max(1, case["L"] // 2), case["L"], case["B"]).sum())
        e = 4 if case["dtype"] == "f32" else 2
        once = d * e + d + 4  # a row in the model's type and in the cache's
        if case["op"] == "write":  # and read back
            once += d * e + d + 4
        return {"bytes": 2 * tokens * Hkv * once + 4 * tokens, "flops": 2 * tokens * Hkv * d}
    lens = _spread(rng, case["lo"], case["hi"], case["B"])
    pages = -(-lens // page)
    if case["op"] == "bounds":
        n = int(lens.sum()) * Hkv * (d + 4) + int(pages.sum()) * (Hkv * (2 * d + 4) + 4)
        # The values that the bounds stand for are formed from them.
        return {"bytes": n + int(pages.sum()) * Hkv * (10 * d + 4), "flops": 3 * int(lens.sum()) * Hkv * d}
    took = np.minimum(pages, case["budget"])
    tokens = int(((took - 1) * page + (lens - 1) % page + 1).sum())
    ranked = int(pages[pages > case["budget"]].sum())
    n = ranked * (Hkv * (2 * d + 4) + 4) + tokens * Hkv * (2 * d + 8) + 8 * case["B"] * case["Hq"] * d
    n += 4 * case["B"] * Hkv * (case["budget"] + 1)
    return {"bytes": n, "flops": 4 * ranked * case["Hq"] * d + 4 * tokens * case["Hq"] * d}
