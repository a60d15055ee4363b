"""Page bounds and sparse steps of as many sequences as one grid holds."""
import numpy as np
import pytest
import torch

import _paged_ref as ref
from _gpu import down, kvq, up

pytestmark = pytest.mark.gpu


def test_page_bounds_of_the_most_sequences():
    B, size, d = (1 << 24) - 1, 2, 16
    rng = np.random.default_rng(0)
    k, ks = ref.quantise(rng.standard_normal((4, 1, size, d), dtype=np.float32))
    # All but the last sequence share page 3; that one alone has page 1.
    table = torch.full((B, 1), 3, dtype=torch.int32, device="cuda")
    table[-1] = 1
    lengths = torch.full((B,), size, dtype=torch.int32, device="cuda")
    gk, gks = up(k), up(ks)
    bounds, scale = kvq.new_bounds(gk)
    kvq.page_bounds(gk, gks, table, lengths, bounds, scale)
    for page in range(4):
        want, s = ref.bounds(k[page, 0], ks[page, 0]) if page in (1, 3) else (np.zeros((2, d), np.int8), 0)
        assert np.array_equal(down(bounds[page, 0]), want) and float(scale[page, 0]) == s


def test_sparse_steps_of_the_most_sequences():
    B, d = (1 << 23) - 1, 16
    rng = np.random.default_rng(1)
    x = rng.standard_normal((2, 5, 1, 1, d), dtype=np.float32)
    (k, ks), (v, vs) = ref.quantise(x[0]), ref.quantise(x[1])
    pool = [up(a) for a in (k, v, ks, vs)]
    bounds, scale = kvq.new_bounds(pool[0])
    lengths = torch.full((B,), 3, dtype=torch.int32, device="cuda")
    row = torch.tensor([4, 0, 2], dtype=torch.int32, device="cuda")
    table = row.repeat(B, 1)
    kvq.page_bounds(pool[0], pool[2], table[:1].contiguous(), lengths[:1], bounds, scale)
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn((B, 1, d), generator=g, device="cuda")
    out = torch.full_like(q, float("nan"))
    sel = torch.empty((B, 1, 2), dtype=torch.int32, device="cuda")
    n = torch.empty((B, 1), dtype=torch.int32, device="cuda")
    kvq.SparseDecoder(q, *pool, table, lengths, bounds, scale, out, sel, n)()  # the first and the last page
    assert torch.equal(sel, torch.tensor([4, 2], dtype=torch.int32, device="cuda").expand(B, 1, 2)) and (n == 2).all()
    rows = [a.reshape(5, -1)[[4, 2]] for a in (k, ks, v, vs)]
    kk, vv = (torch.from_numpy(rows[i].astype(np.float64) * rows[i + 1].astype(np.float64)).cuda() for i in (0, 2))
    p = torch.softmax((q[:, 0, None].double() * kk).sum(-1) / np.sqrt(d), 1)
    want = (p[:, :, None] * vv).sum(1)
    top = float(q.abs().max())
    tol = ref.attend_tolerance(np.full((1, d), top), rows[0], rows[1][:, 0], rows[2], rows[3][:, 0], 1 / np.sqrt(d))
    assert float((out[:, 0] - want).abs().max()) <= tol
