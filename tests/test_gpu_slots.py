"""kvq_slot_write_launch and kvq_slot_read_launch: codes and scales bit for bit,
values to the rounding of their type, everything else untouched."""
import numpy as np
import pytest
import torch

import _paged_ref as ref
from _gpu import kvq, up

pytestmark = pytest.mark.gpu

DIMS = [64, 128, 1, 20, 32, 48, 80, 96, 100, 112, 192, 256, 272]


def problem(rng, T, Hkv, d, size, pages, dtype):
    x = rng.standard_normal((2, T, Hkv, d)).astype(np.float32) * 3
    x[:, ::5] *= 1e-20
    if T > 3:
        x[0, 3] = 0
    rows = torch.from_numpy(x).to(dtype)
    slots = rng.permutation(pages * size)[:T].astype(np.int32)
    return rows, slots


def pool(rng, pages, Hkv, size, d):
    return [rng.integers(-127, 128, (pages, Hkv, size, d)).astype(np.int8) for _ in "kv"] + \
           [rng.random((pages, Hkv, size)).astype(np.float32) for _ in "kv"]


def rows_at(slots, size):
    return slots // size, slots % size


def layout(rows, how):
    """The packed rows [2, T, Hkv, d] as K and V tensors on the GPU."""
    _, T, Hkv, d = rows.shape
    if how == "packed":
        return rows[0].cuda(), rows[1].cuda()
    pad = {"fused": 5 * Hkv * d, "odd": 3}[how]
    x = torch.full((T, 2 * Hkv * d + pad), float("nan"), dtype=rows.dtype)
    x[:, pad:pad + Hkv * d] = rows[0].reshape(T, -1)
    x[:, pad + Hkv * d:] = rows[1].reshape(T, -1)
    x = x.cuda()
    return x[:, pad:pad + Hkv * d].unflatten(1, (Hkv, d)), x[:, pad + Hkv * d:].unflatten(1, (Hkv, d))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", DIMS)
def test_write_bits(d, dtype):
    rng = np.random.default_rng(d)
    for T, Hkv, size, how in [(1, 1, 16, "packed"), (37, 8, 16, "packed"), (70, 3, 5, "fused"), (130, 2, 64, "odd"),
                              (515, 4, 32, "fused")]:
        pages = -(-T // size) + 3
        rows, slots = problem(rng, T, Hkv, d, size, pages, dtype)
        slots[1::7] = [-1, pages * size, 2**31 - 1, -2**31][T % 4]
        kp, vp, ksp, vsp = pool(rng, pages, Hkv, size, d)
        gpu = [up(x) for x in (kp, vp, ksp, vsp)]
        kvq.slot_write(*layout(rows, how), up(slots), *gpu)
        torch.cuda.synchronize()
        ok = (slots >= 0) & (slots < pages * size)
        p, o = rows_at(slots[ok], size)
        for c, s, x in ((kp, ksp, rows[0]), (vp, vsp, rows[1])):
            c[p, :, o], s[p, :, o] = ref.quantise(x.float().numpy()[ok])
        for got, want in zip(gpu, (kp, vp, ksp, vsp)):
            got = got.cpu().numpy()
            assert np.array_equal(got.view(np.uint8), want.view(np.uint8)), (T, Hkv, size, how)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", DIMS)
def test_read_values(d, dtype):
    rng = np.random.default_rng(d + 1)
    for T, Hkv, size, how in [(1, 1, 16, "thd"), (37, 8, 16, "htd"), (70, 3, 5, "thd"), (130, 2, 64, "odd"), (515, 4, 32, "htd")]:
        pages = 9
        kp, vp, ksp, vsp = pool(rng, pages, Hkv, size, d)
        slots = rng.integers(0, pages * size, T).astype(np.int32)  # some more than once
        slots[1::7] = [-1, pages * size, 2**31 - 1, -2**31][T % 4]
        if how == "thd":
            outs = [torch.full((T, Hkv, d), float("nan"), dtype=dtype, device="cuda") for _ in "kv"]
            whole = outs
        elif how == "htd":
            whole = [torch.full((Hkv, T, d), float("nan"), dtype=dtype, device="cuda") for _ in "kv"]
            outs = [x.transpose(0, 1) for x in whole]
        else:
            whole = [torch.full((T, Hkv, d + 3), 7.0, dtype=dtype, device="cuda") for _ in "kv"]
            outs = [x[..., 1:1 + d] for x in whole]
        kvq.slot_read(up(slots), *(up(x) for x in (kp, vp, ksp, vsp)), *outs)
        torch.cuda.synchronize()
        ok = (slots >= 0) & (slots < pages * size)
        p, o = rows_at(slots[ok], size)
        for c, s, out in ((kp, ksp, outs[0]), (vp, vsp, outs[1])):
            want = np.zeros((T, Hkv, d), np.float32)
            want[ok] = c[p, :, o].astype(np.float32) * s[p, :, o][..., None]  # one fp32 rounding, as the operator's
            want = torch.from_numpy(want).to(dtype)
            assert torch.equal(out.cpu(), want), (T, Hkv, size, how)
        if how == "odd":
            for x in whole:
                assert bool((x[..., 0] == 7).all()) and bool((x[..., -2:] == 7).all())


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_read_of_scales_that_are_not_finite(bad):
    """A scale that is not finite gives its rows alone values that are not."""
    rng = np.random.default_rng(2)
    kp, vp, ksp, vsp = pool(rng, 3, 2, 16, 64)
    kp[kp == 0] = 1
    ksp[1, :, 3] = bad
    out = [torch.empty((48, 2, 64), device="cuda") for _ in "kv"]
    kvq.slot_read(up(np.arange(48, dtype=np.int32)), *(up(x) for x in (kp, vp, ksp, vsp)), *out)
    fine = torch.isfinite(out[0]).all(-1).cpu()
    assert not fine[16 + 3].any() and fine[torch.arange(48) != 19].all() and bool(torch.isfinite(out[1]).all())


def test_write_then_read_in_a_graph():
    """Captured write and read, replayed with other rows and slots."""
    rng = np.random.default_rng(4)
    T, Hkv, size, d, pages = 50, 4, 16, 128, 8
    k, v = (torch.empty((T, Hkv, d), dtype=torch.bfloat16, device="cuda") for _ in "kv")
    slots = torch.empty(T, dtype=torch.int32, device="cuda")
    gpu = [up(x) for x in pool(rng, pages, Hkv, size, d)]
    out = [torch.empty((T, Hkv, d), device="cuda") for _ in "kv"]

    def step():
        kvq.slot_write(k, v, slots, *gpu)
        kvq.slot_read(slots, *gpu, *out)

    graph = None
    for i in range(5):
        rows, at = problem(rng, T, Hkv, d, size, pages, torch.bfloat16)
        k.copy_(rows[0]), v.copy_(rows[1]), slots.copy_(torch.from_numpy(at))
        torch.cuda.synchronize()
        if graph is None:
            step()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
        graph.replay()
        torch.cuda.synchronize()
        for x, o in zip(rows, out):
            code, s = ref.quantise(x.float().numpy())
            assert np.array_equal(o.cpu().numpy(), code.astype(np.float32) * s[..., None]), i


def test_write_matches_append_bits():
    """The same bits as kvq_paged_append_launch for the same rows."""
    rng = np.random.default_rng(6)
    B, Hkv, d, size = 6, 4, 128, 16
    rows = torch.from_numpy((rng.standard_normal((2, B, Hkv, d)) * 4).astype(np.float32)).cuda()
    table = up(rng.permutation(12).reshape(B, 2).astype(np.int32))
    pos = rng.integers(0, 32, B).astype(np.int32)
    a = [up(x) for x in pool(rng, 12, Hkv, size, d)]
    b = [x.clone() for x in a]
    kvq.paged_append(rows[0], rows[1], *a, table, positions=up(pos))
    slots = table.cpu().numpy()[np.arange(B), pos // size] * size + pos % size
    kvq.slot_write(rows[0], rows[1], up(slots.astype(np.int32)), *b)
    for x, y in zip(a, b):
        assert torch.equal(x, y)


def test_no_rows():
    rng = np.random.default_rng(1)
    gpu = [up(x) for x in pool(rng, 2, 2, 16, 64)]
    none = torch.empty((0, 2, 64), device="cuda")
    slots = torch.empty(0, dtype=torch.int32, device="cuda")
    kvq.slot_write(none, none, slots, *gpu)
    kvq.slot_read(slots, *gpu, none, none)


def test_pool_past_4_gib():
    """Rows whose byte offset in the pool passes 2^32."""
    Hkv, d, size = 8, 128, 64
    pages = (5 << 30) // (Hkv * d * size)
    k = torch.zeros((pages, Hkv, size, d), dtype=torch.int8, device="cuda")
    v = torch.zeros((pages, Hkv, size, d), dtype=torch.int8, device="cuda")
    ks, vs = (torch.zeros((pages, Hkv, size), device="cuda") for _ in "kv")
    rng = np.random.default_rng(9)
    x = torch.from_numpy(rng.standard_normal((2, 40, Hkv, d)).astype(np.float32))
    slots = (pages * size - 1 - np.arange(40) * 37).astype(np.int32)
    kvq.slot_write(x[0].cuda(), x[1].cuda(), up(slots), k, v, ks, vs)
    out = [torch.empty((40, Hkv, d), device="cuda") for _ in "kv"]
    kvq.slot_read(up(slots), k, v, ks, vs, *out)
    for i in range(2):
        code, s = ref.quantise(x[i].numpy())
        assert np.array_equal(out[i].cpu().numpy(), code.astype(np.float32) * s[..., None])
    assert int((ks != 0).sum()) == 40 * Hkv
