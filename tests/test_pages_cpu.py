"""The operators around a paged cache without a GPU: struct layouts, what the C
ABI and the Python wrappers refuse, workspace sizes and plans (host-only)."""
import ctypes
import importlib
import os
import subprocess

import pytest
import torch

from _util import REPO

kvq = importlib.import_module("cuda-operators_amd").kvq
HEADER = os.path.join(REPO, "include", "kvq.h")
INVALID = kvq.HIP_ERROR_INVALID_VALUE
BIG = 2**31 - 1

STRUCTS = {"kvq_page_map_params": kvq.PageMapParams, "kvq_slot_write_params": kvq.SlotWriteParams,
           "kvq_slot_read_params": kvq.SlotReadParams, "kvq_page_bounds_params": kvq.PageBoundsParams,
           "kvq_sparse_decode_params": kvq.SparseDecodeParams}


def test_struct_layout_matches_c(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void){"]
    for name, cls in STRUCTS.items():
        lines.append(f'printf("{name} sizeof %zu\\n", sizeof({name}));')
        lines += [f'printf("{name} {f} %zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines():
        name, field, off = line.split()
        cls = STRUCTS[name]
        assert int(off) == (ctypes.sizeof(cls) if field == "sizeof" else getattr(cls, field).offset), line


def filled(cls, **values):
    """A struct whose pointers are stand-ins (never followed) and whose numbers are `values`."""
    p = cls()
    for i, (name, kind) in enumerate(cls._fields_):
        if kind is ctypes.c_void_p:
            setattr(p, name, 4096 * (i + 1))
    for k, x in values.items():
        setattr(p, k, x)
    return p


def map_params(**kw):
    return filled(kvq.PageMapParams, **{**dict(batch=3, page_size=16, num_pages=100, max_pages_per_seq=8, max_tokens=50), **kw})


def write_params(**kw):
    return filled(kvq.SlotWriteParams, **{**dict(tokens=5, num_kv_heads=2, head_dim=64, page_size=16, num_pages=9, dtype=0), **kw})


def read_params(**kw):
    return filled(kvq.SlotReadParams, **{**dict(tokens=5, num_kv_heads=2, head_dim=64, page_size=16, num_pages=9, dtype=0,
                                               token_stride=128, head_stride=64), **kw})


def bounds_params(**kw):
    return filled(kvq.PageBoundsParams, **{**dict(batch=2, num_kv_heads=2, head_dim=64, page_size=16, num_pages=9,
                                                 max_pages_per_seq=4, max_seq_len=0), **kw})


def sparse_params(decode=None, **kw):
    step = filled(kvq.PagedDecodeParams, **{**dict(batch=2, num_q_heads=8, num_kv_heads=2, head_dim=64, page_size=16,
                                                  num_pages=99, max_pages_per_seq=40, max_seq_len=0, softmax_scale=0.0,
                                                  num_splits=0), **(decode or {})})
    return filled(kvq.SparseDecodeParams, **{**dict(decode=step, max_selected=8, keep_first=1, keep_last=1), **kw})


def launch(fn, p, *more):
    return getattr(kvq.lib(), fn)(None if p is None else ctypes.byref(p), *more, None)


BAD_POOL = [dict(page_size=0), dict(page_size=-1), dict(num_pages=0), dict(num_pages=-3), dict(page_size=1 << 16, num_pages=1 << 15)]


@pytest.mark.parametrize("bad", BAD_POOL + [
    dict(batch=0), dict(batch=-1), dict(batch=4097), dict(max_pages_per_seq=0), dict(max_pages_per_seq=BIG),
    dict(max_pages_per_seq=1 << 27), dict(batch=4096, max_pages_per_seq=1 << 20, page_size=1), dict(max_tokens=-1)] +
    [{n: None} for n in ("new_tokens", "lengths", "block_table", "free_pages", "free_count", "new_lengths",
                         "new_free_count", "granted", "token_offsets")])
def test_page_map_refuses(bad):
    p = map_params(**bad)
    assert launch("kvq_page_map_launch", p, None, 0) == INVALID
    assert kvq.lib().kvq_page_map_workspace_size(ctypes.byref(p)) == 0


def test_page_map_workspace_is_wanted():
    p = map_params(batch=64, max_tokens=1 << 20)
    n = kvq.lib().kvq_page_map_workspace_size(ctypes.byref(p))
    if n:
        assert launch("kvq_page_map_launch", p, None, n) == INVALID
        assert launch("kvq_page_map_launch", p, 4096, n - 1) == INVALID
    assert kvq.lib().kvq_page_map_workspace_size(ctypes.byref(map_params(max_tokens=20))) == 0


ROWS = [dict(tokens=-1), dict(num_kv_heads=0), dict(head_dim=0), dict(head_dim=4097), dict(dtype=2), dict(dtype=-1),
        dict(tokens=1 << 30, num_kv_heads=2)]


@pytest.mark.parametrize("bad", BAD_POOL + ROWS + [dict(k_stride=127), dict(v_stride=-1), dict(k_stride=1 << 45)] +
                         [{n: None} for n in ("k_new", "v_new", "slots", "k_pages", "v_pages", "k_scale_pages", "v_scale_pages")])
def test_slot_write_refuses(bad):
    assert launch("kvq_slot_write_launch", write_params(**bad)) == INVALID


@pytest.mark.parametrize("bad", BAD_POOL + ROWS + [
    dict(token_stride=127), dict(token_stride=-128), dict(head_stride=63), dict(head_stride=0), dict(token_stride=0, head_stride=64),
    dict(token_stride=64, head_stride=319), dict(token_stride=63, head_stride=320), dict(token_stride=1 << 45)] +
    [{n: None} for n in ("k_out", "v_out", "slots", "k_pages", "v_pages", "k_scale_pages", "v_scale_pages")])
def test_slot_read_refuses(bad):
    assert launch("kvq_slot_read_launch", read_params(**bad)) == INVALID


@pytest.mark.parametrize("bad", [
    dict(batch=0), dict(num_kv_heads=0), dict(head_dim=0), dict(head_dim=4097), dict(page_size=0), dict(num_pages=0),
    dict(max_pages_per_seq=0), dict(max_pages_per_seq=1 << 28), dict(max_seq_len=-1), dict(max_seq_len=65),
    dict(lengths=None), dict(page_size=1 << 26, max_pages_per_seq=17), dict(batch=1 << 30), dict(num_kv_heads=1 << 30)] +
    [{n: None} for n in ("block_table", "k_pages", "k_scale_pages", "bounds", "bound_scale")])
def test_page_bounds_refuses(bad):
    assert launch("kvq_page_bounds_launch", bounds_params(**bad)) == INVALID


@pytest.mark.parametrize("bad", [
    dict(max_selected=0), dict(max_selected=1), dict(keep_first=-1), dict(keep_last=0), dict(keep_first=8),
    dict(keep_first=BIG, keep_last=BIG), dict(max_selected=1 << 27), dict(max_selected=1 << 30)] +
    [{n: None} for n in ("bounds", "bound_scale", "selected", "selected_lengths")] +
    [dict(decode=x) for x in (dict(batch=0), dict(num_q_heads=7), dict(head_dim=0), dict(page_size=0), dict(num_pages=0),
                              dict(max_seq_len=641), dict(num_splits=-1), dict(q=None), dict(out=None), dict(v_new=None),
                              dict(block_table=None), dict(lengths=None), dict(num_pages=1 << 30), dict(k_scale_pages=None))])
def test_sparse_decode_refuses(bad):
    p = sparse_params(**bad)
    info = kvq.PlanInfo()
    assert launch("kvq_sparse_decode_launch", p, 4096, 1 << 40) == INVALID
    assert kvq.lib().kvq_sparse_decode_workspace_size(ctypes.byref(p)) == 0
    assert kvq.lib().kvq_sparse_decode_plan(ctypes.byref(p), ctypes.byref(info)) == INVALID


def test_null_params():
    for fn, more in (("kvq_page_map_launch", (None, 0)), ("kvq_slot_write_launch", ()), ("kvq_slot_read_launch", ()),
                     ("kvq_page_bounds_launch", ()), ("kvq_sparse_decode_launch", (None, 0))):
        assert launch(fn, None, *more) == INVALID
    assert kvq.lib().kvq_page_map_workspace_size(None) == 0 and kvq.lib().kvq_sparse_decode_workspace_size(None) == 0


@pytest.mark.parametrize("decode,budget", [(dict(), 8), (dict(max_pages_per_seq=8192, num_pages=9000), 64),
                                           (dict(batch=256, num_q_heads=64, num_kv_heads=8, max_pages_per_seq=300), 16)])
def test_sparse_decode_wants_its_workspace(decode, budget):
    p = sparse_params(decode=decode, max_selected=budget)
    n = kvq.lib().kvq_sparse_decode_workspace_size(ctypes.byref(p))
    assert kvq.sparse_decode_plan(p).workspace_bytes == n
    if n:
        assert launch("kvq_sparse_decode_launch", p, None, n) == INVALID
        assert launch("kvq_sparse_decode_launch", p, 4096, n - 1) == INVALID


def test_python_wrappers_refuse():
    """Wrong devices, dtypes, shapes and strides raise before any launch (these tensors are on the CPU)."""
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    pool = (torch.zeros(4, 2, 16, 64, dtype=torch.int8),) * 2 + (torch.zeros(4, 2, 16),) * 2
    rows = torch.zeros(5, 2, 64)
    with pytest.raises(ValueError, match="new_tokens: want contiguous cuda"):
        kvq.PageMapper(i32(3), i32(3), i32(3, 4), i32(9), i32(1), 16)
    with pytest.raises(ValueError, match="k_pages: want contiguous cuda"):
        kvq.slot_write(rows, rows, i32(5), *pool)
    with pytest.raises(ValueError, match="k_pages: want contiguous cuda"):
        kvq.slot_read(i32(5), *pool, rows, rows)
    with pytest.raises(ValueError, match="k_pages: want contiguous cuda"):
        kvq.page_bounds(pool[0], pool[2], i32(1, 4), i32(1), torch.zeros(4, 2, 2, 64, dtype=torch.int8), torch.zeros(4, 2))
    with pytest.raises(ValueError, match="q: want contiguous cuda"):
        kvq.SparseDecoder(torch.zeros(1, 4, 64), *pool, i32(1, 4), i32(1), torch.zeros(4, 2, 2, 64, dtype=torch.int8),
                          torch.zeros(4, 2), torch.zeros(1, 4, 64), i32(1, 2, 3), i32(1, 2))


def _mutated(op):
    return {a.name for a in op.default._schema.arguments if a.alias_info is not None and a.alias_info.is_write}


def test_torch_operators_register_and_trace():
    from torch._subclasses.fake_tensor import FakeTensorMode
    importlib.import_module("cuda-operators_amd.torch_ops")
    ops = torch.ops.kvq
    pool_names = {"k_pages", "v_pages", "k_scale_pages", "v_scale_pages"}
    assert _mutated(ops.page_map) == {"lengths", "block_table", "free_pages", "free_count"}
    assert _mutated(ops.slot_write) == pool_names and _mutated(ops.slot_read) == set()
    assert _mutated(ops.page_bounds) == {"bounds", "bound_scale"}
    assert _mutated(ops.sparse_decode) == pool_names | {"bounds", "bound_scale"}
    with FakeTensorMode():
        i32 = lambda *s: torch.empty(s, dtype=torch.int32)  # noqa: E731
        got = ops.page_map(i32(3), i32(3), i32(3, 8), i32(90), i32(1), 16, 50)
        assert [t.shape[0] for t in got] == [3, 4, 50, 50, 50] and all(t.dtype == torch.int32 for t in got)
        kp, sp = torch.empty(9, 2, 16, 64, dtype=torch.int8), torch.empty(9, 2, 16)
        rows = torch.empty(5, 2, 64, dtype=torch.bfloat16)
        ops.slot_write(rows, rows, i32(5), kp, kp.clone(), sp, sp.clone())
        k, v = ops.slot_read(i32(5), kp, kp, sp, sp, torch.float32, True)
        assert k.shape == v.shape == (2, 5, 64) and k.dtype == torch.float32
        b, s = torch.empty(9, 2, 2, 64, dtype=torch.int8), torch.empty(9, 2)
        ops.page_bounds(kp, sp, i32(3, 8), i32(3), b, s, None, 0)
        out, sel, n = ops.sparse_decode(torch.empty(3, 8, 64), kp, kp.clone(), sp, sp.clone(), i32(3, 8), i32(3), b, s, 4, 1,
                                        1, 0, 0.0, 0, None, None)
        assert out.shape == (3, 8, 64) and sel.shape == (3, 2, 4) and n.shape == (3, 2)
