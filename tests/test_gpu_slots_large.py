"""Packed writes and reads of so many rows that their workgroups do not fit one
dimension of a grid: rows at both sides of every border, and everything else
left as it was."""
import numpy as np
import pytest
import torch

import _paged_ref as ref
from _gpu import down, kvq, up

pytestmark = pytest.mark.gpu


def pool(pages, Hkv, size, d):
    return [torch.full((pages, Hkv, size, d), 85, dtype=torch.int8, device="cuda") for _ in "kv"] + \
           [torch.full((pages, Hkv, size), float("nan"), device="cuda") for _ in "kv"]


# One more workgroup than fits the first row of the grid, and two whole rows.
@pytest.mark.parametrize("Hkv", [(1 << 22) + 3, 1 << 23])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_token_of_many_heads(Hkv, dtype):
    d = 8
    g = torch.Generator(device="cuda").manual_seed(Hkv)
    rows = torch.randn((2, 1, Hkv, d), generator=g, device="cuda").to(dtype)
    gpu = pool(1, Hkv, 1, d)
    slot = torch.zeros(1, dtype=torch.int32, device="cuda")
    kvq.slot_write(rows[0], rows[1], slot, *gpu)
    out = [torch.full((1, Hkv, d), float("nan"), dtype=dtype, device="cuda") for _ in "kv"]
    kvq.slot_read(slot, *gpu, *out)
    for i in range(2):
        codes, scales = ref.quantise(down(rows[i, 0].float()))
        assert np.array_equal(down(gpu[i]).reshape(Hkv, d), codes)
        assert np.array_equal(down(gpu[2 + i]).reshape(Hkv), scales)
        want = torch.from_numpy(codes.astype(np.float32) * scales[:, None]).to(dtype)
        assert torch.equal(out[i].cpu()[0], want)


def test_heads_past_the_threads_of_a_dimension():
    """2^26 heads of one token, a wave each: 2^32 threads for K."""
    Hkv, d = 1 << 26, 4
    g = torch.Generator(device="cuda").manual_seed(3)
    k = torch.randn((1, Hkv, d), generator=g, device="cuda")
    v = torch.randn((1, Hkv, d), generator=g, device="cuda")
    gpu = pool(1, Hkv, 1, d)
    slot = torch.zeros(1, dtype=torch.int32, device="cuda")
    kvq.slot_write(k, v, slot, *gpu)
    out = [torch.full((1, Hkv, d), float("nan"), device="cuda") for _ in "kv"]
    kvq.slot_read(slot, *gpu, *out)
    for i, x in enumerate((k, v)):
        codes, scales = gpu[i].view(Hkv, d), gpu[2 + i].view(Hkv)
        assert torch.equal(scales, x[0].abs().amax(1) / torch.full((1,), 127.0, device="cuda"))  # every row was written
        assert torch.equal(out[i][0], codes.float() * scales[:, None])
        at = torch.cat([torch.arange(s - 70, s + 70) for s in range(1 << 22, Hkv, 1 << 22)] + [torch.arange(70), Hkv - 70 + torch.arange(70)])
        want = ref.quantise(down(x[0, at.cuda()]))[0]
        assert np.array_equal(down(codes[at.cuda()]), want)


def test_rows_past_the_threads_of_a_dimension():
    """2^30 short rows, four threads each; few of them have a slot."""
    T, Hkv, d, size, pages = 1 << 24, 64, 4, 16, 80
    at = np.unique(np.concatenate([np.arange(max(0, s - 20), min(T, s + 20)) for s in range(0, T + 1, 1 << 20)]))
    rng = np.random.default_rng(4)
    rows = torch.zeros((T, Hkv, d), device="cuda")
    x = rng.standard_normal((len(at), Hkv, d), dtype=np.float32)
    rows[up(at)] = up(x)
    place = rng.permutation(size * pages)[:len(at)].astype(np.int32)
    slots = torch.full((T,), -1, dtype=torch.int32, device="cuda")
    slots[up(at)] = up(place)
    gpu = pool(pages, Hkv, size, d)
    kvq.slot_write(rows, rows, slots, *gpu)
    codes, scales = ref.quantise(x)
    want = np.full((pages, Hkv, size, d), 85, np.int8), np.full((pages, Hkv, size), np.nan, np.float32)
    want[0][place // size, :, place % size] = codes
    want[1][place // size, :, place % size] = scales
    for i in range(2):
        assert np.array_equal(down(gpu[i]), want[0])
        assert np.array_equal(down(gpu[2 + i]), want[1], equal_nan=True)
