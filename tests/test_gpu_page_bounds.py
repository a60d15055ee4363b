"""kvq_page_bounds_launch: codes and scales are equal to the definition's, pages
outside the range keep what they held."""
import numpy as np
import pytest
import torch

import _paged_ref as ref
from _gpu import kvq, up

pytestmark = pytest.mark.gpu


def paged(rng, lens, Hkv, size, d, spare=3):
    per = max(1, max(ref.pages_of(n, size) for n in lens))
    pages = len(lens) * per + spare
    table = rng.permutation(pages)[:len(lens) * per].reshape(len(lens), per).astype(np.int32)
    x = rng.standard_normal((pages, Hkv, size, d)).astype(np.float32)
    x[..., 0] *= 20
    k, ks = ref.quantise(x)
    return k, ks, table


def want_bounds(k, ks, table, lens, start, size, bounds, scale):
    for b, n in enumerate(lens):
        first = max(int(start[b]), 0) if start is not None else 0
        for j in range(first // size, ref.pages_of(n, size) if first < n else 0):
            m = min(size, n - j * size)
            for h in range(k.shape[1]):
                bounds[table[b, j], h], scale[table[b, j], h] = ref.bounds(k[table[b, j], h, :m], ks[table[b, j], h, :m])


def check(rng, lens, Hkv, size, d, start=None, k=None, ks=None, table=None, lengths_given=True):
    if k is None:
        k, ks, table = paged(rng, lens, Hkv, size, d)
    bounds = rng.integers(-127, 128, (k.shape[0], Hkv, 2, d)).astype(np.int8)
    scale = rng.random((k.shape[0], Hkv)).astype(np.float32)
    gb, gs = up(bounds), up(scale)
    kvq.page_bounds(up(k), up(ks), up(table), up(np.array(lens, np.int32)) if lengths_given else None, gb, gs,
                    start=None if start is None else up(np.array(start, np.int32)),
                    max_seq_len=0 if lengths_given else lens[0])
    torch.cuda.synchronize()
    with np.errstate(invalid="ignore"):
        want_bounds(k, ks, table, [min(max(n, 0), table.shape[1] * size) for n in lens], start, size, bounds, scale)
    assert np.array_equal(gs.cpu().numpy(), scale)
    assert np.array_equal(gb.cpu().numpy(), bounds)
    return gb, gs


@pytest.mark.parametrize("size", [16, 32, 64, 128, 256, 1, 5, 24, 100])
@pytest.mark.parametrize("d", [128, 64, 16, 48, 80, 96, 160, 256, 20, 272])
def test_matches_definition(d, size):
    rng = np.random.default_rng(d * 7 + size)
    check(rng, [0, 1, size, size + 1, 2 * size - 1, 3 * size + 2], 3, size, d)


@pytest.mark.parametrize("Hkv", [1, 8, 32])
def test_start_and_uniform_lengths(Hkv):
    rng = np.random.default_rng(Hkv)
    check(rng, [100, 77, 64, 64, 1, 90], Hkv, 16, 128, start=[0, 77, 63, 64, -5, 33])
    check(rng, [90, 90, 90], Hkv, 32, 64, lengths_given=False)


def test_lengths_outside_the_table_are_clamped():
    rng = np.random.default_rng(4)
    k, ks, table = paged(rng, [64, 64], 2, 16, 64)
    check(rng, [2**31 - 1, -2**31], 2, 16, 64, k=k, ks=ks, table=table)


def test_scales_of_every_kind():
    """Zero, negative, subnormal, huge, infinite and NaN scales."""
    rng = np.random.default_rng(5)
    k, ks, table = paged(rng, [16 * 9], 2, 16, 64)
    p = table[0]
    ks[p[0]] = 0
    ks[p[1]] *= -1
    ks[p[2], :, ::2] = 0
    ks[p[3]] = np.float32(1e-42)
    ks[p[4]] = np.float32(3e38)
    ks[p[5], 0, 3] = np.inf
    ks[p[6], 1, 9] = np.nan
    ks[p[7], :, 5] = np.float32(1e-30)
    check(rng, [16 * 9], 2, 16, 64, k=k, ks=ks, table=table)


def test_rows_behind_the_end_do_not_count():
    """What stands behind a sequence's last token in its last page changes nothing."""
    rng = np.random.default_rng(6)
    k, ks, table = paged(rng, [16 * 3 + 5], 2, 16, 128)
    ks[table[0, 3], :, 5:] = np.nan
    k[table[0, 3], :, 5:] = 127
    check(rng, [16 * 3 + 5], 2, 16, 128, k=k, ks=ks, table=table)


def test_bounds_hold_the_keys():
    rng = np.random.default_rng(7)
    k, ks, table = paged(rng, [640], 4, 64, 128)
    gb, gs = check(rng, [640], 4, 64, 128, k=k, ks=ks, table=table)
    lim = gb.cpu().numpy().astype(np.float64) * gs.cpu().numpy()[..., None, None]
    for j in table[0]:
        x = k[j].astype(np.float64) * ks[j][..., None]
        # The ratio and the product round to fp32: 2^-24 each, of at most 127 S.
        slack = 127 * gs.cpu().numpy()[j][:, None, None] * 2.0**-23
        assert (x <= lim[j, :, 0][:, None] + slack).all() and (x >= lim[j, :, 1][:, None] - slack).all()


def test_page_ids_outside_the_pool_are_clamped():
    rng = np.random.default_rng(8)
    k, ks, table = paged(rng, [64], 2, 16, 64)
    bad = table.copy()
    bad[0, 1], bad[0, 2] = -7, 2**31 - 1
    clamped = np.clip(bad, 0, k.shape[0] - 1)
    b, s = kvq.new_bounds(up(k))
    kvq.page_bounds(up(k), up(ks), up(bad), up(np.array([64], np.int32)), b, s)
    wb, ws = np.zeros(b.shape, np.int8), np.zeros(s.shape, np.float32)
    want_bounds(k, ks, clamped, [64], None, 16, wb, ws)
    assert np.array_equal(b.cpu().numpy(), wb) and np.array_equal(s.cpu().numpy(), ws)
