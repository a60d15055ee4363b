"""kvq_sparse_decode_launch: the pages selected are equal to the definition's,
the output is attention over them."""
import numpy as np
import pytest
import torch

import _paged_ref as ref
from _gpu import down, kvq, poisoned, up

pytestmark = pytest.mark.gpu


class Problem:
    """A paged batch in numpy, with the bounds of every whole page."""

    def __init__(self, rng, lens, G, Hkv, d, size, dist="outlier", spare=3, per=None):
        self.lens, self.G, self.Hkv, self.d, self.size = [int(n) for n in lens], G, Hkv, d, size
        B = len(lens)
        per = per or max(1, max(ref.pages_of(n, size) for n in lens))
        pages = B * per + spare
        self.table = rng.permutation(pages)[:B * per].reshape(B, per).astype(np.int32)
        x = rng.standard_normal((2, pages, Hkv, size, d)).astype(np.float32)
        if dist == "outlier":
            x[0, ..., rng.integers(0, d, 2)] *= 20
        elif dist == "student":
            x = rng.standard_t(4, x.shape).astype(np.float32)
        self.k, self.ks = ref.quantise(x[0])
        self.v, self.vs = ref.quantise(x[1])
        self.q = rng.standard_normal((B, Hkv * G, d)).astype(np.float32)
        self.bounds = rng.integers(-127, 128, (pages, Hkv, 2, d)).astype(np.int8)  # of pages that are not whole: anything
        self.scale = rng.random((pages, Hkv)).astype(np.float32)
        self.set_bounds()

    def set_bounds(self, upto=None):
        for b, n in enumerate(self.lens):
            for j in range(n // self.size):
                p = self.table[b, j]
                for h in range(self.Hkv):
                    self.bounds[p, h], self.scale[p, h] = ref.bounds(self.k[p, h], self.ks[p, h])

    def chosen(self, b, h, budget, first, last):
        n = self.lens[b]
        ids = self.table[b, :ref.pages_of(n, self.size)]
        q = self.q[b].reshape(self.Hkv, self.G, self.d)[h]
        return ref.select(q, self.bounds[ids, h], self.scale[ids, h], len(ids), first, last, budget)

    def rows(self, b, h, entries):
        ids = self.table[b, entries]
        n = (len(entries) - 1) * self.size + (self.lens[b] - 1) % self.size + 1
        flat = lambda x: x[ids, h].reshape((-1,) + x.shape[3:])[:n]  # noqa: E731
        return flat(self.k), flat(self.ks), flat(self.v), flat(self.vs)

    def gpu(self):
        names = ("q", "k", "v", "ks", "vs", "table", "bounds", "scale")
        g = {n: up(getattr(self, n)) for n in names}
        g["lengths"] = up(np.array(self.lens, np.int32))
        return g


def decoder(p, g, budget, first=1, last=1, lengths=True, **kw):
    B = len(p.lens)
    out = poisoned(p.q.shape)
    sel = torch.full((B, p.Hkv, budget), -77, dtype=torch.int32, device="cuda")
    n = torch.full((B, p.Hkv), -77, dtype=torch.int32, device="cuda")
    dec = kvq.SparseDecoder(g["q"], g["k"], g["v"], g["ks"], g["vs"], g["table"], g["lengths"] if lengths else None,
                            g["bounds"], g["scale"], out, sel, n, keep_first=first, keep_last=last,
                            max_seq_len=kw.pop("max_seq_len", 0 if lengths else p.lens[0]), **kw)
    return dec, out, sel, n


def verify(p, out, sel, n, budget, first, last, softmax_scale=None, choose=None):
    out, sel, n = down(out).reshape(len(p.lens), p.Hkv, p.G, p.d), down(sel), down(n)
    scale = softmax_scale or 1 / np.sqrt(p.d)
    for b, length in enumerate(p.lens):
        for h in range(p.Hkv):
            if length == 0:
                assert n[b, h] == 0 and (sel[b, h] == -1).all() and (out[b, h] == 0).all()
                continue
            entries = (choose or p.chosen)(b, h, budget, first, last)
            want = np.full(budget, -1)
            want[:len(entries)] = p.table[b, entries] * p.Hkv + h
            assert np.array_equal(sel[b, h], want), (b, h)
            rows = p.rows(b, h, entries)
            assert n[b, h] == len(rows[0])
            q = p.q[b].reshape(p.Hkv, p.G, p.d)[h]
            exact = ref.attend(q, *rows, scale)
            err = np.abs(out[b, h] - exact).max()
            assert err <= ref.attend_tolerance(q, *rows, scale), (b, h, err)


def check(p, budget, first=1, last=1, **kw):
    g = p.gpu()
    dec, out, sel, n = decoder(p, g, budget, first, last, **kw)
    dec()
    torch.cuda.synchronize()
    verify(p, out, sel, n, budget, first, last, kw.get("softmax_scale"))
    dec()  # the workspace is left ready
    again = torch.empty_like(out).copy_(out)
    dec()
    assert torch.equal(again, out)
    return g


@pytest.mark.parametrize("G,Hkv", [(1, 4), (4, 2), (3, 2), (8, 1), (16, 1), (17, 1), (40, 1)])
@pytest.mark.parametrize("d", [128, 64, 96])
def test_groups_and_dims(d, G, Hkv):
    rng = np.random.default_rng(d + G)
    check(Problem(rng, [700, 333, 64, 1, 0, 129], G, Hkv, d, 16), 9)


@pytest.mark.parametrize("size", [16, 32, 64, 128, 1, 5, 24])
@pytest.mark.parametrize("d", [128, 32, 48, 80, 112, 144, 192, 256, 20, 272])
def test_page_sizes_and_dims(d, size):
    rng = np.random.default_rng(d * 3 + size)
    n = 21 * size
    check(Problem(rng, [n, n - 1, n + 1, 4 * size, 2], 2, 2, d, size), 6)


@pytest.mark.parametrize("first,last,budget", [(0, 1, 1), (0, 1, 2), (1, 1, 2), (3, 4, 7), (3, 4, 12), (0, 8, 9), (2, 1, 40), (1, 1, 63)])
def test_kept_pages(first, last, budget):
    rng = np.random.default_rng(budget)
    check(Problem(rng, [1000, 16 * 40, 16 * 12, 112, 16 * 8 + 1, 5], 4, 2, 64, 16), budget, first, last)


@pytest.mark.parametrize("dist", ["normal", "student", "outlier"])
@pytest.mark.parametrize("n,size,budget", [(4097, 16, 64), (40000, 64, 100), (70001, 16, 128), (16 * 1025, 16, 30)])
def test_long_contexts(n, size, budget, dist):
    """One sequence, whose pages are scored by several workgroups; keys past 2^16 pages among them."""
    rng = np.random.default_rng(n)
    check(Problem(rng, [n], 4, 2, 64, size, dist), budget)


def test_many_pages():
    """More pages than fit LDS as ranks."""
    rng = np.random.default_rng(1)
    check(Problem(rng, [16 * 20000 + 3, 500], 1, 1, 32, 16), 40)


@pytest.mark.parametrize("B", [5, 33, 70, 300])
def test_batches(B):
    rng = np.random.default_rng(B)
    lens = rng.integers(0, 600, B)
    lens[0] = 600
    check(Problem(rng, lens, 4, 2, 64, 16), 8)


def test_equal_scores_take_the_lower_pages():
    rng = np.random.default_rng(3)
    p = Problem(rng, [16 * 50], 4, 2, 64, 16)
    p.k[:], p.ks[:] = p.k[:1, :, :1], p.ks[:1, :, :1]  # every page alike
    p.set_bounds()
    check(p, 11)
    p.q[:] = 0  # every score 0, of one sign or the other
    check(p, 11)
    half = p.table[0, ::2]
    p.ks[half] *= 2  # two scores, each many times
    p.set_bounds()
    p.q[:] = np.random.default_rng(4).standard_normal(p.q.shape)
    check(p, 30)


def test_scales_that_are_not_finite_rank_first():
    rng = np.random.default_rng(5)
    p = Problem(rng, [16 * 60], 2, 2, 64, 16)
    p.ks[p.table[0, 17], 0, 4] = np.inf
    p.ks[p.table[0, 33], 1, 2] = np.nan
    p.set_bounds()
    g = p.gpu()
    dec, out, sel, n = decoder(p, g, 5)
    dec()
    torch.cuda.synchronize()
    for h, entry in ((0, 17), (1, 33)):
        assert int(p.table[0, entry]) * 2 + h in sel[0, h].tolist()
        assert sorted(sel[0, h].tolist()) == sorted(int(p.table[0, e]) * 2 + h for e in p.chosen(0, h, 5, 1, 1))


def test_uniform_lengths_scale_and_splits():
    rng = np.random.default_rng(6)
    p = Problem(rng, [900, 900, 900], 4, 2, 128, 32)
    check(p, 10, lengths=False)
    check(p, 10, softmax_scale=0.3)
    for splits in (1, 2, 7, 100):
        check(p, 10, num_splits=splits)


def test_lengths_beyond_the_bound_are_clamped():
    rng = np.random.default_rng(7)
    p = Problem(rng, [640, 640], 4, 2, 64, 16)
    g = p.gpu()
    g["lengths"] = up(np.array([10**9, -5], np.int32))
    p.lens = [512, 0]
    dec, out, sel, n = decoder(p, g, 6, max_seq_len=512)
    dec()
    verify(p, out, sel, n, 6, 1, 1)


@pytest.mark.parametrize("d,size,G", [(128, 16, 4), (128, 64, 1), (96, 32, 3), (256, 16, 2), (20, 5, 2), (64, 1, 4)])
def test_steps_with_append_keep_bounds_current(d, size, G):
    """Decode steps with the fused append: the token is stored as kvq_paged_append_launch stores it, and the bounds of a
    page are written when the next one opens."""
    rng = np.random.default_rng(d + size)
    Hkv, steps = 2, 2 * size + 3 if size < 32 else size + 3
    base = [10 * size - 2, 7 * size, 3, 0]
    p = Problem(rng, [n + steps for n in base], G, Hkv, d, size)
    full_k, full_ks = p.k.copy(), p.ks.copy()
    p.lens = list(base)
    for b, n in enumerate(base):  # what later steps bring is not there yet
        for t in range(n, p.table.shape[1] * size):
            for c, fill in ((p.k, 99), (p.v, 99), (p.ks, np.nan), (p.vs, np.nan)):
                c[p.table[b, t // size], :, t % size] = fill
    p.bounds[:], p.scale[:] = 55, 3e9
    p.set_bounds()
    g = p.gpu()
    lengths = g["lengths"]
    kn, vn = (torch.empty((len(base), Hkv, d), device="cuda") for _ in "kv")
    budget = 5
    dec, out, sel, n = decoder(p, g, budget, k_new=kn, v_new=vn)
    for step in range(steps):
        x = rng.standard_normal((2, len(base), Hkv, d)).astype(np.float32)
        kn.copy_(torch.from_numpy(x[0])), vn.copy_(torch.from_numpy(x[1]))
        lengths += 1
        dec()
        torch.cuda.synchronize()
        p.lens = [m + 1 for m in p.lens]
        for b, m in enumerate(p.lens):
            page, o = p.table[b, (m - 1) // size], (m - 1) % size
            p.k[page, :, o], p.ks[page, :, o] = ref.quantise(x[0, b])
            p.v[page, :, o], p.vs[page, :, o] = ref.quantise(x[1, b])
            if (m - 1) % size == 0 and m > 1:
                before = p.table[b, (m - 1) // size - 1]
                for h in range(Hkv):
                    p.bounds[before, h], p.scale[before, h] = ref.bounds(p.k[before, h], p.ks[before, h])
        verify(p, out, sel, n, budget, 1, 1)
    assert np.array_equal(down(g["bounds"]), p.bounds) and np.array_equal(down(g["scale"]), p.scale)
    for name in ("k", "v", "ks", "vs"):
        assert np.array_equal(down(g[name]), getattr(p, name), equal_nan=name.endswith("s")), name


def test_short_sequences_equal_the_dense_step_in_value():
    rng = np.random.default_rng(9)
    p = Problem(rng, [300, 128, 16, 1, 77], 4, 2, 128, 16)
    g = p.gpu()
    dec, out, sel, n = decoder(p, g, 19)
    dec()
    verify(p, out, sel, n, 19, 1, 1)
    dense = poisoned(p.q.shape)
    kvq.PagedDecoder(g["q"], g["k"], g["v"], g["ks"], g["vs"], g["table"], g["lengths"], dense)()
    for b in range(len(p.lens)):
        rows = [p.rows(b, h, list(range(ref.pages_of(p.lens[b], 16)))) for h in range(2)]
        tol = max(ref.attend_tolerance(p.q[b], *r, 1 / np.sqrt(128)) for r in rows)
        assert float((dense[b] - out[b]).abs().max()) <= 2 * tol


def test_graph_replays_with_other_queries_and_lengths():
    rng = np.random.default_rng(10)
    p = Problem(rng, [1500, 900, 1300], 4, 2, 128, 16)
    g = p.gpu()
    dec, out, sel, n = decoder(p, g, 12)
    dec()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dec()
    for step in range(4):
        p.q = rng.standard_normal(p.q.shape).astype(np.float32)
        lens = [1500 - 16 * step, 900 - 7 * step, 1300 - 300 * step]
        p.lens = lens
        g["q"].copy_(up(p.q)), g["lengths"].copy_(up(np.array(lens, np.int32)))
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        verify(p, out, sel, n, 12, 1, 1)
        dec()  # eager work between the replays
        torch.cuda.synchronize()
        verify(p, out, sel, n, 12, 1, 1)


def test_two_streams_with_their_own_workspaces():
    rng = np.random.default_rng(12)
    p = Problem(rng, [4000, 2500], 4, 4, 128, 16)
    g = p.gpu()
    decs = []
    for _ in range(2):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        decs.append((decoder(p, g, 20, stream=s), s))
    for _ in range(5):
        for (dec, *_), s in decs:
            dec(s)
    torch.cuda.synchronize()
    for (_, out, sel, n), _ in decs:
        verify(p, out, sel, n, 20, 1, 1)


def test_pool_past_4_gib():
    """Pages whose K bytes lie past 2^32, and bounds of all of them."""
    Hkv, d, size, G = 8, 128, 64, 4
    pages = (5 << 30) // (Hkv * d * size)
    k = torch.zeros((pages, Hkv, size, d), dtype=torch.int8, device="cuda")
    v = torch.zeros((pages, Hkv, size, d), dtype=torch.int8, device="cuda")
    ks, vs = (torch.zeros((pages, Hkv, size), device="cuda") for _ in "kv")
    rng = np.random.default_rng(13)
    p = Problem(rng, [size * 30 + 9], G, Hkv, d, size)
    ids = pages - 1 - np.arange(p.k.shape[0]) * 700
    at = torch.from_numpy(ids).cuda()
    k[at], v[at], ks[at], vs[at] = up(p.k), up(p.v), up(p.ks), up(p.vs)
    bounds, scale = kvq.new_bounds(k)
    table = up(ids[p.table].astype(np.int32))
    lengths = up(np.array(p.lens, np.int32))
    kvq.page_bounds(k, ks, table, lengths, bounds, scale)
    g = {"q": up(p.q), "k": k, "v": v, "ks": ks, "vs": vs, "table": table, "lengths": lengths, "bounds": bounds, "scale": scale}
    dec, out, sel, n = decoder(p, g, 7)
    dec()
    torch.cuda.synchronize()
    want = [[sorted(int(ids[p.table[0, e]]) * Hkv + h for e in p.chosen(0, h, 7, 1, 1)) for h in range(Hkv)]]
    assert [sorted(x) for x in sel[0].tolist()] == want[0]
    for h in range(Hkv):
        rows = p.rows(0, h, p.chosen(0, h, 7, 1, 1))
        q = p.q[0].reshape(Hkv, G, d)[h]
        err = np.abs(down(out)[0].reshape(Hkv, G, d)[h] - ref.attend(q, *rows, 1 / np.sqrt(d))).max()
        assert err <= ref.attend_tolerance(q, *rows, 1 / np.sqrt(d))
