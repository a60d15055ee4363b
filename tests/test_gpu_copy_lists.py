"""kvq_page_copy_launch with the lists that forks and compactions of large pools
write: long ones, mostly empty, more pairs than a launch has workgroups."""
import numpy as np
import pytest
import torch

from _gpu import kvq, up

pytestmark = pytest.mark.gpu


def pools(layers, P, Hkv, size, d):
    """A pool whose every page holds its own number (and its layer's)."""
    n = torch.arange(P, device="cuda")[None] * 7 + torch.arange(layers, device="cuda")[:, None] * 3
    k = (n % 251 - 125).to(torch.int8)[:, :, None, None, None].expand(layers, P, Hkv, size, d).contiguous()
    v = (n % 241 - 120).to(torch.int8)[:, :, None, None, None].expand(layers, P, Hkv, size, d).contiguous()
    ks = n.float()[:, :, None, None].expand(layers, P, Hkv, size).contiguous()
    return k, v, ks, -ks


def check(pool, src, dst):
    """Pages are the sources' where they were copied to, and their own elsewhere."""
    layers, P = pool[0].shape[:2]
    want = torch.arange(P, device="cuda")
    live = (src >= 0) & (src < P) & (dst >= 0) & (dst < P)
    want[dst[live].long()] = src[live].long()
    n = want[None] * 7 + torch.arange(layers, device="cuda")[:, None] * 3
    for x, y in zip(pool, ((n % 251 - 125), (n % 241 - 120), n.float(), -n.float())):
        assert torch.equal(x.flatten(2), y.to(x.dtype)[:, :, None].expand_as(x.flatten(2)))


def test_a_compaction_of_a_large_pool_in_all_layers():
    """524,288 pages in 32 layers: as many pairs as the pool has pages, nearly all of them -1."""
    layers, P, per = 32, 1 << 19, 300
    pool = pools(layers, P, 1, 1, 8)
    rng = np.random.default_rng(1)
    ids = rng.permutation(P)
    table = up(ids[:2 * per].reshape(2, per).astype(np.int32))
    lengths, count = up(np.full(2, per, np.int32)), up(np.array([P - 2 * per], np.int32))
    free = up(np.concatenate([ids[2 * per:], np.zeros(2 * per)]).astype(np.int32))
    c = kvq.page_compact(lengths, table, None, free, count, 1)
    assert c.copy_src.numel() == P
    kvq.page_copy(c.copy_src, c.copy_dst, *pool)
    assert c.moved.item() > 590 and table.max().item() == 2 * per - 1
    check(pool, c.copy_src, c.copy_dst)


@pytest.mark.parametrize("layers,P,n,live", [(1, 200_000, 100_000, 1.0), (3, 70_000, 70_000, 0.3), (40, 3000, 1400, 0.02),
                                             (1, 40_000, 32_768, 0.0), (2, 50_000, 32_769, 0.5), (64, 1500, 513, 1.0)])
def test_lists_of_any_length(layers, P, n, live):
    """Live pairs among others (-1, pages outside the pool), at random places."""
    rng = np.random.default_rng(n)
    pool = pools(layers, P, 2, 3, 4)
    ids = rng.permutation(P)
    half = min(n, P // 2)
    src = np.concatenate([ids[rng.integers(0, half, half)], np.full(n - half, -1)])
    dst = np.concatenate([ids[half:2 * half], np.full(n - half, P)])
    dead = rng.random(n) >= live
    src = np.where(dead & (rng.random(n) < 0.5), -1, src)
    dst = np.where(dead, rng.choice([-1, -9, P, 1 << 30], n), dst)
    at = rng.permutation(n)
    src, dst = up(src[at].astype(np.int32)), up(dst[at].astype(np.int32))
    kvq.page_copy(src, dst, *pool)
    torch.cuda.synchronize()
    check(pool, src, dst)


def test_large_pages():
    """Pages of more pieces than one workgroup's, few and many pairs."""
    for layers, P, n in ((1, 9, 4), (2, 300, 150)):
        pool = pools(layers, P, 8, 128, 64)
        src, dst = up(np.arange(n, dtype=np.int32)), up(np.arange(n, 2 * n, dtype=np.int32))
        kvq.page_copy(src, dst, *pool)
        check(pool, src, dst)
