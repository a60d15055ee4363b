"""The operators around a paged cache together, as a serving loop runs them:
prompts and decode steps of changing batches, every length, page and slot on
the GPU; prompts read their cached prefix back; pages of ended sequences are
used again.  A host model of the cache (token rows per sequence) is the
reference."""
import numpy as np
import pytest
import torch

import _paged_ref as ref
from _gpu import down, kvq, up

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size,d,dtype", [(16, 128, torch.bfloat16), (64, 96, torch.float32), (5, 20, torch.float32)])
def test_serving_loop(size, d, dtype):
    rng = np.random.default_rng(size)
    B, Hkv, G, per, num, budget = 6, 2, 3, 24, 36, 7
    k, v = (torch.zeros((num, Hkv, size, d), dtype=torch.int8, device="cuda") for _ in "kv")
    ks, vs = (torch.full((num, Hkv, size), float("nan"), device="cuda") for _ in "kv")  # what is not written is never read
    bounds, scale = kvq.new_bounds(k)
    lengths = torch.zeros(B, dtype=torch.int32, device="cuda")
    table = torch.zeros((B, per), dtype=torch.int32, device="cuda")
    free = up(rng.permutation(num).astype(np.int32))
    count = torch.tensor([num], dtype=torch.int32, device="cuda")
    held = [np.zeros((2, 0, Hkv, d), np.float32) for _ in range(B)]  # rows as given, per sequence
    refused = 0
    for step in range(24):
        add = np.ones(B, np.int64)
        if step % 5 == 0:
            add = rng.integers(1, 9 * size, B)  # a round of prompts
        add[rng.random(B) < 0.15] = 0
        for b in np.flatnonzero(rng.random(B) < 0.12):
            add[b] = -held[b].shape[1]  # ends
        if step % 7 == 3:
            add[0] = -3  # taken back
        T = int(np.maximum(add, 0).sum()) + 4
        slots = torch.empty(T, dtype=torch.int32, device="cuda")
        start = lengths.clone()
        m = kvq.page_map(up(add.astype(np.int32)), lengths, table, free, count, size, slot_map=slots)
        rows = torch.from_numpy(rng.standard_normal((2, T, Hkv, d)).astype(np.float32)).to(dtype)
        kvq.slot_write(rows[0].cuda(), rows[1].cuda(), slots, k, v, ks, vs)
        start = torch.minimum(start, lengths)
        kvq.page_bounds(k, ks, table, lengths, bounds, scale, start=start)
        # The host's model.
        granted, offsets = m.granted.tolist(), m.token_offsets.tolist()
        x = rows.float().numpy()
        for b in range(B):
            if granted[b] > 0:
                held[b] = np.concatenate([held[b], x[:, offsets[b]:offsets[b] + granted[b]]], 1)
            else:
                held[b] = held[b][:, :held[b].shape[1] + granted[b]]
            refused += add[b] > 0 and granted[b] == 0
        lens = [h.shape[1] for h in held]
        assert lengths.tolist() == lens
        used = [ref.pages_of(n, size) for n in lens]
        tb = table.tolist()
        pages = [p for b in range(B) for p in tb[b][:used[b]]] + free[:int(count)].tolist()
        assert sorted(pages) == list(range(num))  # every page is held once
        # The cached tokens read back, whole sequences laid end to end.
        at = np.concatenate([[tb[b][t // size] * size + t % size for t in range(lens[b])] for b in range(B)] + [[]]).astype(np.int32)
        out = [torch.empty((len(at), Hkv, d), device="cuda") for _ in "kv"]
        kvq.slot_read(up(at), k, v, ks, vs, *out)
        codes = [[ref.quantise(h[i]) for h in held] for i in range(2)]
        for i in range(2):
            want = np.concatenate([c.astype(np.float32) * s[..., None] for c, s in codes[i]])
            assert np.array_equal(down(out[i]), want)
        # A decode query over what is there.
        q = rng.standard_normal((B, Hkv * G, d)).astype(np.float32)
        o = torch.full((B, Hkv * G, d), float("nan"), device="cuda")
        sel = torch.empty((B, Hkv, budget), dtype=torch.int32, device="cuda")
        n = torch.empty((B, Hkv), dtype=torch.int32, device="cuda")
        kvq.SparseDecoder(up(q), k, v, ks, vs, table, lengths, bounds, scale, o, sel, n)()
        o = down(o).reshape(B, Hkv, G, d)
        for b in range(B):
            for h in range(Hkv):
                if lens[b] == 0:
                    assert (o[b, h] == 0).all()
                    continue
                (kc, kss), (vc, vss) = codes[0][b], codes[1][b]
                lim = [ref.bounds(kc[j * size:(j + 1) * size, h], kss[j * size:(j + 1) * size, h]) for j in range(used[b])]
                qq = q[b].reshape(Hkv, G, d)[h]
                pick = ref.select(qq, np.stack([x[0] for x in lim]), np.array([x[1] for x in lim]), used[b], 1, 1, budget)
                t = np.concatenate([np.arange(j * size, min((j + 1) * size, lens[b])) for j in pick])
                assert sel[b, h].tolist() == [tb[b][j] * Hkv + h for j in pick] + [-1] * (budget - len(pick)), (step, b, h)
                args = (qq, kc[t, h], kss[t, h], vc[t, h], vss[t, h], 1 / np.sqrt(d))
                assert np.abs(o[b, h] - ref.attend(*args)).max() <= ref.attend_tolerance(*args)
    assert refused > 0  # the pool ran out at least once
