"""Decode steps after a page map that refuses a sequence or leaves one waiting:
what those sequences hold stays as it was, byte for byte, whether the step's
rows go through the slot map or through the step's fused append (with length 0
for the sequences that were granted nothing)."""
import numpy as np
import pytest
import torch

import _paged_ref as ref
from _gpu import down, kvq, up

pytestmark = pytest.mark.gpu

# Lengths before the step, and the tokens asked for: one that grows within its
# page, a waiting one, one whose last page is full (no page is free: refused),
# one behind a prefix page that it shares with the refused one, an empty one
# that is refused, and one that grows to the end of its page.
LENS, ASKS = lambda n: [n + 4, 2 * n + 5, 2 * n, n + 3, 0, 2 * n - 1], [1, 0, 1, 1, 1, 1]
GRANTED = [1, 0, 0, 1, 0, 1]


class Batch:
    def __init__(self, G, d, size, seed):
        rng = np.random.default_rng(seed)
        self.G, self.d, self.size, self.Hkv, self.per = G, d, size, 2, 4
        self.lens = LENS(size)
        B = len(self.lens)
        self.table = rng.integers(0, 8, (B, self.per)).astype(np.int32)  # entries without meaning
        self.num = 0
        for b, n in enumerate(self.lens):
            for j in range(ref.pages_of(n, size)):
                self.table[b, j] = self.num
                self.num += 1
        self.table[3, 0] = self.table[2, 1]  # the refused sequence's last page is a prefix of another
        x = rng.standard_normal((2, self.num, self.Hkv, size, d), dtype=np.float32)
        (self.k, self.ks), (self.v, self.vs) = ref.quantise(x[0]), ref.quantise(x[1])
        self.q = rng.standard_normal((B, self.Hkv * G, d), dtype=np.float32)
        self.new = rng.standard_normal((2, B, self.Hkv, d), dtype=np.float32)  # a row for every sequence, granted or not
        self.gpu = {n: up(getattr(self, n)) for n in ("k", "v", "ks", "vs", "table", "q")}
        self.gpu["lengths"] = up(np.array(self.lens, np.int32))
        self.free, self.count = torch.zeros(self.num, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
        self.bounds, self.scale = kvq.new_bounds(self.gpu["k"])
        g = self.gpu
        kvq.page_bounds(g["k"], g["ks"], g["table"], g["lengths"], self.bounds, self.scale)

    def expected(self):
        """The pool after the step: only granted rows are written."""
        pool = [self.k.copy(), self.v.copy(), self.ks.copy(), self.vs.copy()]
        for b, n in enumerate(self.lens):
            if GRANTED[b]:
                page, at = self.table[b, n // self.size], n % self.size
                for i in range(2):
                    pool[i][page, :, at], pool[2 + i][page, :, at] = ref.quantise(self.new[i, b])
        return pool

    def check(self, pool, out, attended):
        want = self.expected()
        for got, w, name in zip(pool, want, ("k", "v", "ks", "vs")):
            assert np.array_equal(down(got).view(np.uint8), w.view(np.uint8)), name
        o = down(out).reshape(len(self.lens), self.Hkv, self.G, self.d)
        for b, n in enumerate(self.lens):
            n += GRANTED[b]
            if not attended[b] or n == 0:
                assert (o[b] == 0).all()
                continue
            t = np.arange(n)
            rows = self.table[b, t // self.size], t % self.size
            for h in range(self.Hkv):
                args = (self.q[b].reshape(self.Hkv, self.G, self.d)[h], *(x[rows[0], h, rows[1]] for x in
                        (want[0], want[2], want[1], want[3])), 1 / np.sqrt(self.d))
                assert np.abs(o[b, h] - ref.attend(*args)).max() <= ref.attend_tolerance(*args), (b, h)


def steps(batch, form, sparse):
    """(what a step calls, its output, the sequences attended)"""
    g = batch.gpu
    asks = up(np.array(ASKS, np.int32))
    B = len(ASKS)
    slots = torch.empty(B, dtype=torch.int32, device="cuda")
    mapper = kvq.PageMapper(asks, g["lengths"], g["table"], batch.free, batch.count, batch.size, slot_map=slots)
    out = torch.full((B, batch.Hkv * batch.G, batch.d), float("nan"), device="cuda")
    rows = up(batch.new)
    attended = torch.empty_like(g["lengths"])  # lengths of the sequences that the step attends
    pool = (g["k"], g["v"], g["ks"], g["vs"])
    new = dict(k_new=rows[0], v_new=rows[1]) if form == "append" else {}
    lens = attended if form == "append" else g["lengths"]
    if sparse:
        sel = torch.empty((B, batch.Hkv, batch.per), dtype=torch.int32, device="cuda")
        n = torch.empty((B, batch.Hkv), dtype=torch.int32, device="cuda")
        step = kvq.SparseDecoder(g["q"], *pool, g["table"], lens, batch.bounds, batch.scale, out, sel, n, **new)
    else:
        step = kvq.PagedDecoder(g["q"], *pool, g["table"], lens, out, **new)
    # Packed rows follow the sequences that asked.
    packed = torch.cat([rows[:, b:b + 1] for b in range(B) if ASKS[b]] + [rows[:, :1]] * ASKS.count(0), 1).contiguous()

    def run():
        mapper()
        if form == "append":
            torch.mul(g["lengths"], mapper.granted > 0, out=attended)
        else:
            kvq.slot_write(packed[0], packed[1], slots, *pool)
        step()

    return run, mapper, out, [bool(x) for x in GRANTED] if form == "append" else [True] * B


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("sparse", [False, True])
@pytest.mark.parametrize("form", ["slots", "append"])
@pytest.mark.parametrize("G,d,size", [(4, 128, 16), (1, 128, 64), (6, 96, 16), (2, 20, 5)])
def test_refused_and_waiting_sequences_keep_their_tokens(G, d, size, form, sparse, captured):
    batch = Batch(G, d, size, G * d + size)
    run, mapper, out, attended = steps(batch, form, sparse)
    g = batch.gpu
    if captured:
        before = {n: g[n].clone() for n in ("k", "v", "ks", "vs", "lengths")}
        run()  # loads the kernels
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
        for _ in range(3):
            for n, x in before.items():
                g[n].copy_(x)
            graph.replay()
            torch.cuda.synchronize()
            assert mapper.granted.tolist() == GRANTED
            batch.check((g["k"], g["v"], g["ks"], g["vs"]), out, attended)
    else:
        run()
        torch.cuda.synchronize()
        assert mapper.granted.tolist() == GRANTED
        assert g["lengths"].tolist() == [n + a for n, a in zip(batch.lens, GRANTED)]
        batch.check((g["k"], g["v"], g["ks"], g["vs"]), out, attended)
