"""Chunk attention and shared pages without a GPU: struct layouts, what the C ABI
and the Python wrappers refuse, workspace sizes (host-only), and the restatements
that the GPU tests compare with."""
import ctypes
import subprocess

import pytest
import torch

import _share_ref as ref
from test_pages_cpu import HEADER, INVALID, filled, kvq, launch

STRUCTS = {"kvq_chunk_attention_params": kvq.ChunkAttentionParams, "kvq_page_fork_params": kvq.PageForkParams,
           "kvq_page_copy_params": kvq.PageCopyParams, "kvq_page_compact_params": kvq.PageCompactParams}


def test_struct_layout_matches_c(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void){"]
    for name, cls in STRUCTS.items():
        lines.append(f'printf("{name} sizeof %zu\\n", sizeof({name}));')
        lines += [f'printf("{name} {f} %zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    lines.append('printf("limits %d %d\\n", KVQ_CHUNK_MAX_BATCH, KVQ_FORK_MAX_BATCH);')
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines():
        name, field, off = line.split()
        if name == "limits":
            assert (int(field), int(off)) == (kvq.CHUNK_MAX_BATCH, kvq.FORK_MAX_BATCH)
            continue
        cls = STRUCTS[name]
        assert int(off) == (ctypes.sizeof(cls) if field == "sizeof" else getattr(cls, field).offset), line


def chunk(**kw):
    return filled(kvq.ChunkAttentionParams, **{**dict(batch=3, num_q_heads=8, num_kv_heads=2, head_dim=64, page_size=16,
                                                      num_pages=100, max_pages_per_seq=8, max_seq_len=0, tokens=50, dtype=1,
                                                      causal=1, q_stride=0, out_stride=0, softmax_scale=0.0), **kw})


def fork(**kw):
    return filled(kvq.PageForkParams, **{**dict(batch=3, page_size=16, num_pages=100, max_pages_per_seq=8), **kw})


def copy(**kw):
    return filled(kvq.PageCopyParams, **{**dict(copies=3, layers=2, num_kv_heads=2, head_dim=64, page_size=16, num_pages=9), **kw})


def compact(**kw):
    return filled(kvq.PageCompactParams, **{**dict(batch=3, page_size=16, num_pages=100, max_pages_per_seq=8, max_moves=7), **kw})


TABLE = [dict(batch=0), dict(batch=-1), dict(batch=4097), dict(page_size=0), dict(page_size=-1), dict(max_pages_per_seq=0),
         dict(max_pages_per_seq=1 << 28), dict(batch=4096, max_pages_per_seq=1 << 20), dict(num_pages=0), dict(num_pages=-3)]
POOL = [dict(page_size=1 << 16, num_pages=1 << 15)]


def pointers(cls, but=()):
    return [{n: None} for n, kind in cls._fields_ if kind is ctypes.c_void_p and n not in but]


@pytest.mark.parametrize("bad", TABLE + pointers(kvq.ChunkAttentionParams, ("granted",)) + [
    dict(num_q_heads=0), dict(num_q_heads=7), dict(num_kv_heads=0), dict(head_dim=0), dict(head_dim=4097), dict(tokens=-1),
    dict(tokens=1 << 28, num_q_heads=16), dict(max_seq_len=-1), dict(max_seq_len=129), dict(dtype=2), dict(dtype=-1),
    dict(q_stride=511), dict(out_stride=511), dict(q_stride=-512), dict(q_stride=1 << 60), dict(out_stride=1 << 45),
    dict(max_pages_per_seq=1 << 27)])
def test_chunk_refusals(bad):
    p = chunk(**bad)
    assert launch("kvq_chunk_attention_launch", p, 4096, 1 << 40) == INVALID
    assert kvq.lib().kvq_chunk_attention_workspace_size(ctypes.byref(p)) == 0


@pytest.mark.parametrize("bad", TABLE + POOL + pointers(kvq.PageForkParams, ("keep",)))
def test_fork_refusals(bad):
    p = fork(**bad)
    assert launch("kvq_page_fork_launch", p, 4096, 1 << 40) == INVALID
    assert kvq.lib().kvq_page_fork_workspace_size(ctypes.byref(p)) == 0


@pytest.mark.parametrize("bad", [dict(copies=-1), dict(layers=0), dict(layers=65536), dict(copies=1 << 20, layers=16),
                                 dict(num_kv_heads=0), dict(head_dim=0), dict(head_dim=4097), dict(page_size=0),
                                 dict(num_pages=0), dict(bounds=None), dict(bound_scale=None)] + POOL +
                         pointers(kvq.PageCopyParams, ("bounds", "bound_scale")))
def test_copy_refusals(bad):
    assert launch("kvq_page_copy_launch", copy(**bad)) == INVALID


@pytest.mark.parametrize("bad", TABLE + POOL + pointers(kvq.PageCompactParams) + [dict(max_moves=0), dict(max_moves=-1)])
def test_compact_refusals(bad):
    p = compact(**bad)
    assert launch("kvq_page_compact_launch", p, 4096, 1 << 40) == INVALID
    assert kvq.lib().kvq_page_compact_workspace_size(ctypes.byref(p)) == 0


def test_null_params():
    for fn in ("kvq_chunk_attention_launch", "kvq_page_fork_launch", "kvq_page_compact_launch"):
        assert launch(fn, None, 4096, 1 << 40) == INVALID
    assert launch("kvq_page_copy_launch", None) == INVALID


@pytest.mark.parametrize("make,name", [(fork, "kvq_page_fork"), (compact, "kvq_page_compact"),
                                       (lambda: chunk(batch=1, tokens=4, max_pages_per_seq=500), "kvq_chunk_attention")])
def test_workspace_is_wanted_whole(make, name):
    p = make()
    n = getattr(kvq.lib(), name + "_workspace_size")(ctypes.byref(p))
    assert n > 0
    assert launch(name + "_launch", p, None, n) == INVALID
    assert launch(name + "_launch", p, 4096, n - 1) == INVALID


def test_chunk_workspace_sizes():
    size = lambda **kw: kvq.lib().kvq_chunk_attention_workspace_size(ctypes.byref(chunk(**kw)))  # noqa: E731
    assert size(tokens=0) == 0
    # Many tiles, short sequences and the generic kernel split nothing.
    assert size(batch=300, tokens=300, num_q_heads=16, num_kv_heads=16) == 0
    assert size(max_pages_per_seq=8) == 0   # 128 tokens: a split has two key tiles of 64 at least
    assert size(max_pages_per_seq=16) > 0   # 256 tokens
    assert size(head_dim=20, batch=1, max_pages_per_seq=1 << 16) == 0
    # At most 256 records of 256 rows (128 from d = 256 on) and the counters.
    for d, rows, padded in ((64, 256, 64), (80, 256, 96), (128, 256, 128), (192, 128, 192), (256, 128, 256)):
        n = size(head_dim=d, batch=1, tokens=4, max_pages_per_seq=1 << 16, num_kv_heads=1)
        assert (256 << 10) < n <= (256 << 10) + 256 * rows * (padded + 2) * 4, d
    for b in (1, 7, 500):
        for t in (1, 33, 4096):
            for h in (1, 8, 32):
                assert size(batch=b, tokens=t, num_q_heads=h, num_kv_heads=h, max_pages_per_seq=4096) <= (256 << 10) + 256 * 256 * 66 * 4


def test_wrappers_refuse_what_is_not_on_a_gpu():
    z = lambda *s, dt=torch.int32: torch.zeros(s, dtype=dt)  # noqa: E731
    pool = (z(4, 1, 2, 8, dt=torch.int8), z(4, 1, 2, 8, dt=torch.int8), z(4, 1, 2, dt=torch.float32), z(4, 1, 2, dt=torch.float32))
    q = z(3, 1, 8, dt=torch.float32)
    with pytest.raises(ValueError):
        kvq.chunk_attention(q, *pool, z(1, 2), z(1), z(2))
    with pytest.raises(ValueError):
        kvq.page_fork(z(1), z(1), z(1, 2), z(4), z(4), z(1), 2)
    with pytest.raises(ValueError):
        kvq.page_copy(z(1), z(1), *pool)
    with pytest.raises(ValueError):
        kvq.page_compact(z(1), z(1, 2), z(4), z(4), z(1), 2)


# ---- the restatements ------------------------------------------------------------
def test_reference_attention_on_closed_forms():
    i = ref.batch(1, [(7, 3), (1, 1), (0, 0)], 4, 2, 8, 4, torch.float32, device="cpu")
    out, tol, written = ref.chunk(i, True)
    assert written.tolist() == [True] * 4 + [False] * 3
    # One token to attend: its V row.
    p, at = int(i["block_table"][1, 0]), 0
    v = i["v"][p, :, at].double() * i["vs"][p, :, at, None].double()
    assert torch.allclose(out[3], v.repeat_interleave(2, 0))
    # q = 0: the mean of the rows up to the token's own.
    i["q"].zero_()
    out, tol, _ = ref.chunk(i, True)
    v = ref.values(i["v"], i["vs"], i["block_table"][0], 7)
    for r in range(3):
        assert torch.allclose(out[r], v[:, :5 + r].mean(1).repeat_interleave(2, 0))
    assert (tol > 0).any() and torch.isfinite(tol).all()


def test_reference_attention_counts_what_a_mistake_costs():
    """One key too many, a missing scale, a wrong head: far outside the tolerance."""
    i = ref.batch(2, [(60, 9)], 4, 2, 16, 4, torch.bfloat16, device="cpu")
    out, tol, _ = ref.chunk(i, True)
    off, _, _ = ref.chunk(i, False)
    assert ((off - out).abs() > tol)[:8].any(-1).any(-1).all()  # (in some head: a key's weight may be next to nothing)
    scaled, _, _ = ref.chunk(i, True, scale=0.26)
    assert ((scaled - out).abs() > tol)[:9].any(-1).all()
    assert ((out.flip(1) - out).abs() > tol)[:9].any(-1).all()


def test_reference_fork_and_compaction_by_hand():
    st = {"lengths": [10, 4, 9], "block_table": [[0, 1, 2], [3, 9, 9], [0, 1, 4]], "shares": [1, 1, 0, 0, 0, 0, 0],
          "free_pages": [6, 5, 0, 0, 0, 0, 0], "free_count": [2], "parents": [0, 0, -1], "keep": [10, 9, 0]}
    r = ref.fork(st, 4)
    # Row 1 goes on from row 0's 9 tokens: its own page 3 and row 2's page 4 become free, and it copies page 2 to 4.
    assert r["new_lengths"] == [10, 9, 0] and r["copy_src"] == [-1, 2, -1] and r["copy_dst"] == [-1, 4, -1]
    assert r["rows"] == [[0, 1, 2], [0, 1, 4], []] and r["new_shares"] == [1, 1, 0, 0, 0, 0, 0]
    assert r["new_free_count"] == [3] and r["free_pages"][:3] == [6, 5, 3]
    st = {"lengths": [5], "block_table": [[5, 2, 0]], "shares": [0, 0, 0, 0, 0, 2, 0], "free_pages": [0, 1, 3, 4, 6, 9, 9], "free_count": [5]}
    r = ref.compact(st, 4, 9)
    assert r["rows"] == [[0, 1]] and r["copy_src"][:2] == [5, 2] and r["copy_dst"][:2] == [0, 1] and r["moved"] == [2]
    assert r["free_pages"] == [6, 5, 4, 3, 2] and r["new_shares"] == [2, 0, 0, 0, 0, 0, 0]
