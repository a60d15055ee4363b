"""kvq_chunk_attention_plan without a GPU: which kernel a shape takes, whether its
keys are split, and that it refuses what the launch refuses."""
import ctypes

import pytest

from test_pages_cpu import INVALID, kvq
from test_share_cpu import chunk


def plan(**kw):
    p = chunk(**kw)
    info = kvq.chunk_attention_plan(p)
    assert info.workspace_bytes == kvq.lib().kvq_chunk_attention_workspace_size(ctypes.byref(p))
    return info


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("d", [8, 64, 72, 96, 128, 192, 256])
def test_shapes_of_the_matrix_cores(d, dtype):
    info = plan(head_dim=d, dtype=dtype)
    assert (info.kernel, info.heads_per_group, info.tile_tokens) == (kvq.KERNEL_CHUNK_MFMA, 4, 64)
    assert info.query_block == (256 if d <= (128 if dtype else 96) else 128)


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("kw", [
    dict(head_dim=20), dict(head_dim=264), dict(head_dim=4096), dict(num_q_heads=258), dict(q=4096 + 4), dict(out=4096 + 8),
    dict(k_pages=4096 + 4), dict(v_pages=4096 + 1), dict(q_stride=8 * 64 + 2), dict(out_stride=8 * 64 + 1),
    dict(tokens=1 << 22, num_q_heads=256, num_kv_heads=2)])
def test_shapes_of_the_generic_kernel(kw, dtype):
    info = plan(dtype=dtype, **kw)
    assert (info.kernel, info.query_block, info.tile_tokens) == (kvq.KERNEL_CHUNK_GENERIC, 1, 0)
    assert (info.splits, info.split_plan, info.workspace_bytes) == (1, kvq.SPLITS_STATIC, 0)


def test_splits():
    for kw in (dict(max_pages_per_seq=16), dict(batch=1, tokens=4, max_pages_per_seq=500)):
        info = plan(**kw)
        assert (info.splits, info.split_plan) == (0, kvq.SPLITS_IN_KERNEL) and info.workspace_bytes > 0
    for kw in (dict(), dict(tokens=0), dict(batch=300, tokens=300, num_q_heads=16, num_kv_heads=16)):
        info = plan(**kw)
        assert (info.splits, info.split_plan, info.workspace_bytes) == (1, kvq.SPLITS_STATIC, 0)


@pytest.mark.parametrize("bad", [dict(batch=0), dict(tokens=-1), dict(head_dim=4097), dict(q=None), dict(max_seq_len=129),
                                 dict(dtype=2), dict(q_stride=511)])
def test_refusals(bad):
    info = kvq.PlanInfo()
    assert kvq.lib().kvq_chunk_attention_plan(ctypes.byref(chunk(**bad)), ctypes.byref(info)) == INVALID
    assert kvq.lib().kvq_chunk_attention_plan(ctypes.byref(chunk()), None) == INVALID
    assert kvq.lib().kvq_chunk_attention_plan(None, ctypes.byref(info)) == INVALID
    with pytest.raises(kvq.KvqError):
        kvq.chunk_attention_plan(chunk(**bad))
