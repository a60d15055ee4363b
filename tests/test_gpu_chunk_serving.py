"""Chunk attention, forks, copies and compaction together, as a serving loop runs
them around the paged cache's other operators: prompts in chunks, beams that go on
from each other, cuts, ends, a pool that is compacted; and the same through
torch.ops.kvq.  A host model of the cache (token rows per sequence) is the reference."""
import importlib

import numpy as np
import pytest
import torch

import _paged_ref as pref
import _share_ref as ref
from _gpu import kvq, up

pytestmark = pytest.mark.gpu

I32 = torch.int32


class Server:
    """Two layers' pools, tables and counts on the GPU; what each row holds on the host."""

    def __init__(self, size, d, B=6, Hkv=2, G=2, per=20, num=70, layers=2):
        self.size, self.d, self.B, self.Hkv, self.G, self.layers = size, d, B, Hkv, G, layers
        self.k, self.v = (torch.zeros((layers, num, Hkv, size, d), dtype=torch.int8, device="cuda") for _ in "kv")
        self.ks, self.vs = (torch.full((layers, num, Hkv, size), float("nan"), device="cuda") for _ in "kv")
        self.bounds = torch.zeros((layers, num, Hkv, 2, d), dtype=torch.int8, device="cuda")
        self.scale = torch.zeros((layers, num, Hkv), device="cuda")
        self.lengths = torch.zeros(B, dtype=I32, device="cuda")
        self.table = torch.zeros((B, per), dtype=I32, device="cuda")
        self.shares = torch.zeros(num, dtype=I32, device="cuda")
        self.free = torch.randperm(num, device="cuda").to(I32)
        self.count = torch.tensor([num], dtype=I32, device="cuda")
        self.held = [np.zeros((layers, 2, 0, Hkv, d), np.float32) for _ in range(B)]

    def pool(self, layer):
        return self.k[layer], self.v[layer], self.ks[layer], self.vs[layer]

    def add(self, rng, add, dtype):
        """New tokens: pages, rows in every layer, and their attention against the host's."""
        T = int(add.sum()) + 2
        slots = torch.empty(T, dtype=I32, device="cuda")
        m = kvq.page_map(up(add.astype(np.int32)), self.lengths, self.table, self.free, self.count, self.size, slot_map=slots)
        granted, offsets = m.granted.tolist(), m.token_offsets.tolist()
        rows = torch.from_numpy(rng.standard_normal((self.layers, 2, T, self.Hkv, self.d)).astype(np.float32)).to(dtype)
        q = torch.from_numpy(rng.standard_normal((T, self.Hkv * self.G, self.d)).astype(np.float32)).to(dtype).cuda()
        for b in range(self.B):
            if granted[b] > 0:
                self.held[b] = np.concatenate([self.held[b], rows.float().numpy()[:, :, offsets[b]:offsets[b + 1]]], 2)
        for layer in range(self.layers):
            kvq.slot_write(rows[layer, 0].cuda(), rows[layer, 1].cuda(), slots, *self.pool(layer))
            kvq.page_bounds(self.k[layer], self.ks[layer], self.table, self.lengths, self.bounds[layer], self.scale[layer])
            out = torch.full_like(q, float("nan"))
            kvq.chunk_attention(q, *self.pool(layer), self.table, self.lengths, m.token_offsets, out, granted=m.granted)
            for b in range(self.B):
                o = out[offsets[b]:offsets[b + 1]]
                if granted[b] <= 0:
                    assert (o == 0).all()
                    continue
                self.check(layer, b, q[offsets[b]:offsets[b + 1]], o)
            assert torch.isnan(out[offsets[-1]:]).all()
        return granted

    def check(self, layer, b, q, out):
        n, L = q.shape[0], self.held[b].shape[2]
        keys = torch.arange(n, device="cuda") + L - n + 1
        for h in range(self.Hkv):
            k, v = (torch.from_numpy(c.astype(np.float64) * s[:, None]).cuda()
                    for c, s in (pref.quantise(self.held[b][layer, i, :, h]) for i in range(2)))
            x = q[:, h * self.G:(h + 1) * self.G]
            want, tol = ref.attend(x.double().flatten(0, 1), k, v, self.d**-0.5, keys.repeat_interleave(self.G), q.dtype == torch.bfloat16)
            got = out[:, h * self.G:(h + 1) * self.G].double().flatten(0, 1)
            assert ((got - want).abs() <= tol).all(), (layer, b, h)

    def consistent(self):
        """Every page is free, or held by as many rows as shares says."""
        lens = self.lengths.tolist()
        assert lens == [x.shape[2] for x in self.held]
        holders = np.zeros(len(self.free), int)
        for b, row in enumerate(self.table.tolist()):
            for p in row[:pref.pages_of(lens[b], self.size)]:
                holders[p] += 1
        free = self.free.tolist()[:int(self.count)]
        assert sorted(free) == np.flatnonzero(holders == 0).tolist()
        assert (np.maximum(holders - 1, 0) == np.array(self.shares.tolist())).all()

    def copy(self, src, dst):
        kvq.page_copy(src, dst, self.k, self.v, self.ks, self.vs, self.bounds, self.scale)

    def fork(self, parents, keep):
        f = kvq.page_fork(up(parents.astype(np.int32)), self.lengths, self.table, self.shares, self.free, self.count, self.size,
                          keep=up(keep.astype(np.int32)))
        self.copy(f.copy_src, f.copy_dst)
        lens = self.lengths.tolist()
        old = self.held
        self.held = [old[p][:, :, :n] if 0 <= p < self.B else old[0][:, :, :0] for p, n in zip(parents.tolist(), lens)]
        asked = [min(max(k, 0), old[p].shape[2]) if 0 <= p < self.B else 0 for p, k in zip(parents.tolist(), keep.tolist())]
        assert all(n == a or (n == a - a % self.size and self.count.item() == 0) for n, a in zip(lens, asked))

    def compact(self, moves):
        c = kvq.page_compact(self.lengths, self.table, self.shares, self.free, self.count, self.size, max_moves=moves)
        self.copy(c.copy_src, c.copy_dst)
        if c.moved.item() < moves:
            used = len(self.free) - int(self.count)
            assert sorted(self.free.tolist()[:int(self.count)]) == list(range(used, len(self.free)))

    def read_back(self):
        """Every row's tokens, in every layer, are those of the host."""
        table, lens = self.table.tolist(), self.lengths.tolist()
        for layer in range(self.layers):
            for b in range(self.B):
                at = np.array([table[b][t // self.size] * self.size + t % self.size for t in range(lens[b])], np.int32)
                k, v = (torch.empty((len(at), self.Hkv, self.d), device="cuda") for _ in "kv")
                kvq.slot_read(up(at), *self.pool(layer), k, v)
                for i, x in enumerate((k, v)):
                    codes, s = pref.quantise(self.held[b][layer, i])
                    assert np.array_equal(x.cpu().numpy(), codes.astype(np.float32) * s[..., None]), (layer, b)


@pytest.mark.parametrize("size,d,dtype", [(16, 64, torch.bfloat16), (16, 128, torch.float32), (5, 20, torch.float32)])
def test_serving_loop(size, d, dtype):
    rng = np.random.default_rng(size + d)
    s = Server(size, d)
    short = 0
    for step in range(14):
        add = rng.integers(0, 3 * size, s.B) if step % 4 == 0 else np.ones(s.B, np.int64)
        add = np.where([x.shape[2] == 0 for x in s.held], np.maximum(add, 1), add)
        granted = s.add(rng, add, dtype)
        short += sum(a > 0 and g == 0 for a, g in zip(add, granted))
        s.consistent()
        if step % 3 == 1:  # a beam step: rows go on from others; some end, some are cut
            parents = rng.integers(0, s.B, s.B)
            parents[rng.random(s.B) < 0.1] = -1
            keep = np.where(rng.random(s.B) < 0.3, rng.integers(0, 4 * size, s.B), 1 << 30)
            s.fork(parents, keep)
            s.consistent()
        if step % 5 == 4:
            s.compact(int(rng.integers(1, 40)))
            s.consistent()
        s.read_back()


def test_torch_ops():
    ops = importlib.import_module("cuda-operators_amd.torch_ops") and torch.ops.kvq
    i = ref.batch(3, [(100, 20), (70, 1), (300, 9)], 8, 2, 64, 16, torch.bfloat16, refused=(1,))
    args = [i[n] for n in ("q", "k", "v", "ks", "vs", "block_table", "lengths", "token_offsets", "granted")]
    out = ops.chunk_attention(*args, True, 0, 0.0)
    want, tol, written = ref.chunk(i, True)
    assert ((out.double() - want).abs() <= tol)[written].all() and (out[~written] == 0).all()
    st = {"lengths": [20, 5, 0], "block_table": [[3, 4], [6, 0], [0, 0]], "shares": [0] * 8, "free_pages": [7, 5, 2, 1, 0] + [0] * 3,
          "free_count": [5], "parents": [0, 0, 1], "keep": [1 << 30, 18, 1 << 30]}
    g = {n: up(np.asarray(x, np.int32)) for n, x in st.items()}
    want = ref.fork(st, 16)
    src, dst = ops.page_fork(g["parents"], g["keep"], g["lengths"], g["block_table"], g["shares"], g["free_pages"], g["free_count"], 16)
    assert src.tolist() == want["copy_src"] and dst.tolist() == want["copy_dst"]
    assert g["lengths"].tolist() == want["new_lengths"] and g["shares"].tolist() == want["new_shares"]
    k = torch.arange(8, dtype=torch.int8, device="cuda")[:, None, None, None].expand(8, 1, 16, 32).contiguous()
    ks = k[..., 0].float().contiguous()
    ops.page_copy(src, dst, k, k.clone(), ks, ks.clone(), None, None)
    for a, b in zip(src.tolist(), dst.tolist()):
        assert a < 0 or ((k[b] == a).all() and (ks[b] == a).all())
    after = {n: g[n].tolist() for n in ("lengths", "block_table", "shares", "free_pages", "free_count")}
    want = ref.compact(after, 16, 4)
    src, dst, moved = ops.page_compact(g["lengths"], g["block_table"], g["shares"], g["free_pages"], g["free_count"], 16, 4)
    assert [src.tolist(), dst.tolist(), moved.tolist()] == [want["copy_src"], want["copy_dst"], want["moved"]]
    assert g["shares"].tolist() == want["new_shares"]
    for op, a in ((ops.chunk_attention, (*args, True, 0, 0.0)),):
        torch.library.opcheck(op, a, test_utils=("test_schema", "test_faketensor"))


def test_a_step_in_one_graph():
    """Page map, write, attention, fork and copies captured together and replayed over growing sequences."""
    size, d, B, Hkv, num = 16, 64, 4, 2, 60
    rng = np.random.default_rng(9)
    k, v = (torch.zeros((num, Hkv, size, d), dtype=torch.int8, device="cuda") for _ in "kv")
    ks, vs = (torch.zeros((num, Hkv, size), device="cuda") for _ in "kv")
    lengths, table = torch.zeros(B, dtype=I32, device="cuda"), torch.zeros((B, 12), dtype=I32, device="cuda")
    free, count = torch.arange(num, dtype=I32, device="cuda"), torch.tensor([num], dtype=I32, device="cuda")
    shares, parents = torch.zeros(num, dtype=I32, device="cuda"), torch.arange(B, dtype=I32, device="cuda")
    new = torch.tensor([9, 3, 5, 1], dtype=I32, device="cuda")
    T = 20
    slots = torch.empty(T, dtype=I32, device="cuda")
    rows = torch.zeros((2, T, Hkv, d), device="cuda")
    q, out = torch.zeros((T, 2 * Hkv, d), device="cuda"), torch.zeros((T, 2 * Hkv, d), device="cuda")
    fork = kvq.PageForker(parents, lengths, table, shares, free, count, size)
    mapper = kvq.PageMapper(new, lengths, table, free, count, size, slot_map=slots)
    att = kvq.ChunkAttention(q, k, v, ks, vs, table, lengths, mapper.token_offsets, out, granted=mapper.granted)

    def step():
        fork()
        kvq.page_copy(fork.copy_src, fork.copy_dst, k, v, ks, vs)
        mapper()
        kvq.slot_write(rows[0], rows[1], slots, k, v, ks, vs)
        att()

    state = [lengths, table, free, count, shares, k, v, ks, vs]
    begin = [x.clone() for x in state]
    step()
    torch.cuda.synchronize()
    for x, y in zip(state, begin):
        x.copy_(y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for x, y in zip(state, begin):
        x.copy_(y)
    held = [np.zeros((2, 0, Hkv, d), np.float32) for _ in range(B)]
    for _ in range(6):
        p = rng.integers(0, B, B)
        parents.copy_(up(p.astype(np.int32)))
        held = [held[i] for i in p]
        x = rng.standard_normal((2, T, Hkv, d)).astype(np.float32)
        rows.copy_(torch.from_numpy(x))
        q.copy_(torch.from_numpy(rng.standard_normal(q.shape).astype(np.float32)))
        graph.replay()
        torch.cuda.synchronize()
        at = 0
        for b, n in enumerate(new.tolist()):
            held[b] = np.concatenate([held[b], x[:, at:at + n]], 1)
            L = held[b].shape[1]
            keys = (torch.arange(n, device="cuda") + L - n + 1).repeat_interleave(2)
            for h in range(Hkv):
                kk, vv = (torch.from_numpy(c.astype(np.float64) * s[:, None]).cuda() for c, s in (pref.quantise(held[b][i][:, h]) for i in range(2)))
                want, tol = ref.attend(q[at:at + n, 2 * h:2 * h + 2].double().flatten(0, 1), kk, vv, d**-0.5, keys, False)
                assert ((out[at:at + n, 2 * h:2 * h + 2].double().flatten(0, 1) - want).abs() <= tol).all(), (b, h)
            at += n
