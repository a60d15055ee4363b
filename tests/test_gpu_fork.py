"""kvq_page_fork_launch, kvq_page_copy_launch and kvq_page_compact_launch against
sequential restatements: every integer and every copied byte is equal, entries
without a meaning are left as they were."""
import numpy as np
import pytest
import torch

import _share_ref as ref
from _gpu import kvq, up
from _paged_ref import pages_of

pytestmark = pytest.mark.gpu

GARBAGE = -77


def pool(rng, B, size, hi, groups, spare):
    """Rows in groups that share whole pages, each with a tail of its own; spare: free pages."""
    group = rng.integers(0, groups, B)
    prompt = rng.integers(0, hi // size + 1, groups)
    lens = prompt[group] * size + rng.integers(0, 3 * size, B) * (rng.random(B) < 0.8)
    used = [pages_of(x, size) for x in lens]
    per = max(max(used), 1) + 1
    num = int(sum(prompt)) + sum(used) + spare + 3
    ids = iter(rng.permutation(num).tolist())
    shared = [[next(ids) for _ in range(n)] for n in prompt]
    table = rng.integers(-9, num + 9, (B, per)).tolist()
    for b in range(B):
        mine = shared[group[b]]
        table[b][:used[b]] = mine + [next(ids) for _ in range(used[b] - len(mine))]
    held = np.zeros(num, int)
    for b in range(B):
        for p in table[b][:used[b]]:
            held[p] += 1
    left = [p for p in ids]
    for g in range(groups):  # groups without a row: their prompt is the caller's own
        for p in shared[g]:
            held[p] += (group != g).all()
    free = left[:spare] + rng.integers(-9, 9, num - min(spare, len(left))).tolist()
    return {"lengths": lens.tolist(), "block_table": table, "shares": np.maximum(held - 1, 0).tolist(), "free_pages": free,
            "free_count": [min(spare, len(left))]}


def fork_state(rng, B, size, hi, groups, spare):
    st = pool(rng, B, size, hi, groups, spare)
    parents = rng.integers(0, B, B)
    parents = np.where(rng.random(B) < 0.3, np.arange(B), parents)
    parents = np.where(rng.random(B) < 0.1, rng.choice([-1, -5, B, 1 << 30], B), parents)
    st["parents"] = parents.tolist()
    st["keep"] = np.where(rng.random(B) < 0.4, rng.integers(-3, hi + 3 * size, B), 1 << 30).tolist()
    return st


def device(st):
    return {k: up(np.asarray(v, np.int32)) for k, v in st.items() if v is not None}


def forker(g, size, in_place=False, **kw):
    B, per, num = *g["block_table"].shape, g["free_pages"].shape[0]
    fill = lambda *n: torch.full(n, GARBAGE, dtype=torch.int32, device="cuda")  # noqa: E731
    if not in_place:
        kw |= dict(new_lengths=fill(B), new_block_table=fill(B, per), new_shares=fill(num), new_free_count=fill(1))
    return kvq.PageForker(g["parents"], g["lengths"], g["block_table"], g["shares"], g["free_pages"], g["free_count"], size,
                          keep=g.get("keep"), **kw)


def check_fork(f, st, size, table=None):
    torch.cuda.synchronize()
    want = ref.fork(st, size)
    for n in ("new_lengths", "new_shares", "new_free_count", "copy_src", "copy_dst", "free_pages"):
        assert getattr(f, n).tolist() == want[n], n
    got = f.new_block_table.tolist()
    for b, row in enumerate(want["rows"]):
        assert got[b][:len(row)] == row, b
        assert got[b][len(row):] == (table[b][len(row):] if table else [GARBAGE] * (len(got[b]) - len(row))), b
    if f.ws is not None:
        assert not f.ws.any()
    return want


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("B,size,hi,groups,spare", [(1, 16, 40, 1, 3), (2, 4, 30, 1, 0), (5, 16, 100, 2, 2), (16, 64, 900, 4, 16),
                                                    (64, 1, 90, 9, 40), (33, 7, 200, 5, 4), (300, 16, 900, 40, 100),
                                                    (1500, 16, 300, 200, 700), (4096, 32, 100, 900, 1000), (3, 16, 40000, 2, 2)])
def test_fork(B, size, hi, groups, spare, in_place):
    rng = np.random.default_rng(B + size)
    for _ in range(3):
        st = fork_state(rng, B, size, hi, groups, spare)
        g = device(st)
        f = forker(g, size, in_place)
        f()
        check_fork(f, st, size, st["block_table"] if in_place else None)
        if not in_place:
            for n in ("parents", "keep", "lengths", "block_table", "shares", "free_count"):
                assert g[n].tolist() == st[n], n


def test_fork_without_keep_and_again():
    """All of the parents' tokens; the same handle launched on its own result, many times over."""
    rng = np.random.default_rng(0)
    st = fork_state(rng, 24, 8, 100, 3, 200)
    st["keep"] = None
    g = device(st)
    f = forker(g, 8, True)
    for _ in range(12):
        f()
        torch.cuda.synchronize()
        table = st["block_table"]
        want = check_fork(f, st, 8, table)
        rows = [r + t[len(r):] for r, t in zip(want["rows"], table)]
        st = {"lengths": want["new_lengths"], "block_table": rows, "shares": want["new_shares"], "keep": None,
              "free_pages": want["free_pages"], "free_count": want["new_free_count"],
              "parents": rng.integers(-1, 24, 24).tolist()}
        g["parents"].copy_(up(np.asarray(st["parents"], np.int32)))


def test_fork_keeps_pages_that_others_hold():
    """A page held outside the tables (one more in shares) survives its rows, and is copied before one writes into it."""
    st = {"lengths": [20, 5], "block_table": [[3, 4], [6, 0]], "shares": [0, 0, 0, 1, 1, 0, 0, 0], "free_pages": [7, 5] + [0] * 6,
          "free_count": [2], "parents": [0, -1], "keep": [1 << 30, 0]}
    f = forker(device(st), 16)
    f()
    check_fork(f, st, 16)
    assert f.copy_src.tolist() == [4, -1] and f.copy_dst.tolist() == [6, -1]  # 6 has just become free
    assert f.new_shares.tolist() == [0, 0, 0, 1, 0, 0, 0, 0] and f.new_free_count.tolist() == [2]
    st["parents"] = [-1, -1]
    f = forker(device(st), 16)
    f()
    check_fork(f, st, 16)
    assert f.new_free_count.tolist() == [3] and f.new_shares.tolist() == [0] * 8


def test_fork_wants_pages_it_does_not_get():
    """Rows in excess of the free pages keep their whole pages."""
    st = {"lengths": [40, 0, 0, 0], "block_table": [[1, 2, 3]] * 4, "shares": [0] * 6, "free_pages": [5] + [0] * 5, "free_count": [1],
          "parents": [0, 0, 0, 0], "keep": [40, 39, 35, 33]}
    f = forker(device(st), 16)
    f()
    check_fork(f, st, 16)
    assert f.new_lengths.tolist() == [40, 39, 32, 32] and f.copy_dst.tolist() == [-1, 5, -1, -1]


def test_fork_in_a_graph():
    rng = np.random.default_rng(4)
    st = fork_state(rng, 40, 16, 400, 6, 30)
    g = device(st)
    f = forker(g, 16)
    f()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        f()
    for _ in range(4):
        st["parents"] = rng.integers(-1, 40, 40).tolist()
        g["parents"].copy_(up(np.asarray(st["parents"], np.int32)))
        g["free_pages"].copy_(up(np.asarray(st["free_pages"], np.int32)))
        f.new_block_table.fill_(GARBAGE)
        graph.replay()
        check_fork(f, st, 16)


def test_one_workspace_for_all_forks():
    rng = np.random.default_rng(5)
    ws = torch.zeros(8 << 20, dtype=torch.uint8, device="cuda")
    for B, size, hi in ((5, 16, 100), (300, 16, 900), (16, 64, 900), (64, 1, 90), (5, 16, 100)):
        st = fork_state(rng, B, size, hi, 3, 20)
        f = forker(device(st), size, workspace=lambda n: ws)
        assert f.ws_bytes <= ws.numel()
        f()
        check_fork(f, st, size)


# ---- copies ----------------------------------------------------------------------
@pytest.mark.parametrize("layers,Hkv,size,d,n", [(1, 1, 1, 1, 1), (1, 8, 16, 128, 4), (3, 2, 5, 20, 9), (2, 8, 64, 128, 70),
                                                 (4, 3, 16, 80, 33), (1, 2, 7, 33, 5), (40, 1, 4, 64, 3), (1, 4, 128, 256, 150)])
@pytest.mark.parametrize("bounds", [False, True])
@pytest.mark.parametrize("flat", [False, True])
def test_copy(layers, Hkv, size, d, n, bounds, flat):
    if flat:  # a 4-d pool
        layers = 1
    rng = np.random.default_rng(n)
    P = 2 * n + 5
    g = torch.Generator(device="cuda")
    g.manual_seed(n)
    lead = (P,) if flat else (layers, P)
    code = lambda *s: torch.randint(-128, 128, lead + s, generator=g, dtype=torch.int8, device="cuda")  # noqa: E731
    word = lambda *s: torch.randint(-2**31, 2**31 - 1, lead + s, generator=g, dtype=torch.int32, device="cuda").view(torch.float32)  # noqa: E731
    names = ["k", "v", "ks", "vs"] + (["bounds", "scale"] if bounds else [])
    x = dict(zip(names, [code(Hkv, size, d), code(Hkv, size, d), word(Hkv, size), word(Hkv, size)]
                 + ([code(Hkv, 2, d), word(Hkv)] if bounds else [])))
    ids = rng.permutation(P)
    src, dst = ids[rng.integers(0, n, n)], ids[n:2 * n].copy()
    none = rng.random(n) < 0.2
    src, dst = np.where(none & (rng.random(n) < 0.5), -1, src), np.where(none, rng.choice([-1, P, 1 << 30], n), dst)
    want = {k: t.clone().view(torch.int32 if t.dtype == torch.float32 else torch.int8) for k, t in x.items()}
    for a, b in zip(src.tolist(), dst.tolist()):
        if 0 <= a < P and 0 <= b < P:
            for t in want.values():
                if flat:
                    t[b] = t[a]
                else:
                    t[:, b] = t[:, a]
    kvq.page_copy(up(src.astype(np.int32)), up(dst.astype(np.int32)), *x.values())
    torch.cuda.synchronize()
    for k, t in want.items():
        assert torch.equal(x[k].view(t.dtype), t), k


def test_copy_past_4_gb():
    Hkv, size, d = 8, 64, 128
    P = (1 << 32) // (Hkv * size * d) + 20
    k, v = (torch.empty((P, Hkv, size, d), dtype=torch.int8, device="cuda") for _ in "kv")
    ks, vs = (torch.empty((P, Hkv, size), device="cuda") for _ in "kv")
    for t in (k, v, ks, vs):
        t[-3] = 7
        t[0] = 1
        t[-1] = 2
    kvq.page_copy(up(np.array([P - 3], np.int32)), up(np.array([P - 1], np.int32)), k, v, ks, vs)
    for t in (k, v, ks, vs):
        assert (t[-1] == 7).all() and (t[0] == 1).all()


def test_copy_of_nothing():
    k = torch.zeros((4, 1, 2, 8), dtype=torch.int8, device="cuda")
    s = torch.zeros((4, 1, 2), device="cuda")
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    kvq.page_copy(none, none, k, k.clone(), s, s.clone())


# ---- compaction --------------------------------------------------------------------
def check_compact(c, st, size, moves, table=None):
    torch.cuda.synchronize()
    want = ref.compact(st, size, moves)
    assert c.moved.tolist() == want["moved"]
    assert c.copy_src.tolist() == want["copy_src"] and c.copy_dst.tolist() == want["copy_dst"]
    if st["shares"] is not None:
        assert c.new_shares.tolist() == want["new_shares"]
    got, F = c.new_free_pages.tolist(), len(want["free_pages"])
    assert got[:F] == want["free_pages"]
    assert got[F:] == (st["free_pages"][F:] if table else [GARBAGE] * (len(got) - F))
    got = c.new_block_table.tolist()
    for b, row in enumerate(want["rows"]):
        assert got[b][:len(row)] == row, b
        assert got[b][len(row):] == (table[b][len(row):] if table else [GARBAGE] * (len(got[b]) - len(row))), b


@pytest.mark.parametrize("shares", [True, False])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("B,size,hi,groups,spare,moves", [(1, 16, 40, 1, 3, 1), (2, 4, 30, 1, 0, 5), (5, 16, 100, 2, 9, 2),
                                                          (64, 1, 90, 9, 400, 10000), (33, 7, 200, 5, 90, 30),
                                                          (300, 16, 900, 40, 3000, 900), (4096, 32, 100, 900, 1000, 300),
                                                          (2, 16, 300000, 2, 60000, 30000), (3, 1, 200000, 2, 90000, 50000)])
def test_compact(B, size, hi, groups, spare, moves, in_place, shares):
    rng = np.random.default_rng(B + size)
    st = pool(rng, B, size, hi, groups, spare)
    rng.shuffle(mine := st["free_pages"][:st["free_count"][0]])
    st["free_pages"][:len(mine)] = mine
    if not shares:
        st["shares"] = None
    g = device(st)
    per, num = g["block_table"].shape[1], len(st["free_pages"])
    fill = lambda *n: torch.full(n, GARBAGE, dtype=torch.int32, device="cuda")  # noqa: E731
    more = {} if in_place else dict(new_block_table=fill(B, per), new_free_pages=fill(num))
    if shares and not in_place:
        more["new_shares"] = fill(num)
    c = kvq.PageCompactor(g["lengths"], g["block_table"], g.get("shares"), g["free_pages"], g["free_count"], size, moves, **more)
    c()
    check_compact(c, st, size, moves, st["block_table"] if in_place else None)
    if in_place and c.moved.item() < moves:  # all moved: a second call has nothing to do
        c()
        torch.cuda.synchronize()
        assert c.moved.item() == 0 and (c.copy_src == -1).all()


@pytest.mark.parametrize("free", [[], list(range(9)), [8, 7, 6], [0, 1, 2]])
def test_compact_of_whole_and_empty_pools(free):
    used = [p for p in range(9) if p not in free]
    st = {"lengths": [len(used) * 4], "block_table": [used + [0] * (9 - len(used))], "shares": [0] * 9,
          "free_pages": free + [0] * (9 - len(free)), "free_count": [len(free)]}
    g = device(st)
    c = kvq.PageCompactor(g["lengths"], g["block_table"], g["shares"], g["free_pages"], g["free_count"], 4)
    c()
    check_compact(c, st, 4, 9, st["block_table"])


def test_compact_in_a_graph():
    rng = np.random.default_rng(6)
    st = pool(rng, 40, 16, 400, 6, 200)
    g = device(st)
    fill = lambda *n: torch.full(n, GARBAGE, dtype=torch.int32, device="cuda")  # noqa: E731
    num = len(st["free_pages"])
    c = kvq.PageCompactor(g["lengths"], g["block_table"], g["shares"], g["free_pages"], g["free_count"], 16, 60,
                          new_block_table=fill(*g["block_table"].shape), new_shares=fill(num), new_free_pages=fill(num))
    c()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c()
    for count in (st["free_count"][0], 50, 0, 10):
        st["free_count"] = [count]
        g["free_count"].fill_(count)
        c.new_block_table.fill_(GARBAGE)
        c.new_free_pages.fill_(GARBAGE)
        graph.replay()
        check_compact(c, st, 16, 60)
