"""Shapes around a paged cache that no grid holds are refused, and those just
below are not (host-only: plans and workspace sizes, no launch)."""
import ctypes

import pytest

from test_pages_cpu import INVALID, bounds_params, kvq, launch, sparse_params


@pytest.mark.parametrize("batch", [1 << 24, (1 << 24) + 5, 1 << 29])
def test_page_bounds_of_too_many_sequences(batch):
    assert launch("kvq_page_bounds_launch", bounds_params(batch=batch, max_pages_per_seq=1)) == INVALID


def sparse_of(batch, heads):
    return sparse_params(decode=dict(batch=batch, num_q_heads=heads, num_kv_heads=heads, max_pages_per_seq=3, num_pages=9),
                         max_selected=2)


@pytest.mark.parametrize("batch,heads", [(1 << 23, 1), (1 << 20, 8), (1, 1 << 23), ((1 << 22) + 1, 2)])
def test_sparse_decode_of_too_many_units(batch, heads):
    p, info = sparse_of(batch, heads), kvq.PlanInfo()
    assert launch("kvq_sparse_decode_launch", p, 4096, 1 << 40) == INVALID
    assert kvq.lib().kvq_sparse_decode_workspace_size(ctypes.byref(p)) == 0
    assert kvq.lib().kvq_sparse_decode_plan(ctypes.byref(p), ctypes.byref(info)) == INVALID


@pytest.mark.parametrize("batch,heads", [((1 << 23) - 1, 1), ((1 << 20) - 1, 8)])
def test_sparse_decode_of_many_units(batch, heads):
    p = sparse_of(batch, heads)
    assert kvq.sparse_decode_plan(p).workspace_bytes == kvq.lib().kvq_sparse_decode_workspace_size(ctypes.byref(p))
