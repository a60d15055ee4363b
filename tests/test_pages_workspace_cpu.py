"""Which shapes around a paged cache need a workspace, how much of it, and that
they do not launch without it (host-only): a map of many workgroups without its
arrival counter would update lengths in place while others still read them."""
import ctypes

import pytest

from test_pages_cpu import INVALID, kvq, launch, map_params, sparse_params

COUNTERS = 256 * 1024  # the prefix that arrival counters of every shape share


def wants(fn, p, n):
    assert launch(fn, p, None, n) == INVALID
    assert launch(fn, p, 4096, n - 1) == INVALID
    assert launch(fn, p, None, 0) == INVALID


@pytest.mark.parametrize("shape", [dict(batch=64, max_tokens=1 << 20), dict(max_tokens=33), dict(batch=4096, max_tokens=4096, num_pages=9000),
                                   dict(slot_map=None, token_pos=None, max_tokens=1 << 20),
                                   dict(slot_map=None, token_seq=None, token_pos=None, batch=40, max_tokens=1 << 20)])
def test_page_map_of_several_workgroups(shape):
    p = map_params(**shape)
    n = kvq.lib().kvq_page_map_workspace_size(ctypes.byref(p))
    assert n == 256
    wants("kvq_page_map_launch", p, n)


@pytest.mark.parametrize("shape", [dict(max_tokens=32), dict(max_tokens=0), dict(batch=4096, max_tokens=20, num_pages=9000),
                                   dict(slot_map=None, token_seq=None, token_pos=None, batch=20, max_tokens=100)])
def test_page_map_of_one_workgroup(shape):
    assert kvq.lib().kvq_page_map_workspace_size(ctypes.byref(map_params(**shape))) == 0


@pytest.mark.parametrize("decode,budget,ranks", [
    (dict(max_pages_per_seq=8192, num_pages=9000), 64, 4 * 8192),                    # several workgroups a unit, several splits
    (dict(max_pages_per_seq=300), 4, 4 * 300),                                       # several workgroups a unit, attention unsplit
    (dict(batch=256, num_q_heads=64, num_kv_heads=8, max_pages_per_seq=6145), 16, 2048 * 6145),  # one a unit, ranks beyond LDS
    (dict(head_dim=20, max_pages_per_seq=40), 8, 4 * 40)])                            # the generic selection
def test_sparse_decode_with_ranks_in_memory(decode, budget, ranks):
    p = sparse_params(decode=decode, max_selected=budget)
    n = kvq.lib().kvq_sparse_decode_workspace_size(ctypes.byref(p))
    assert n >= COUNTERS + 4 * ranks and kvq.sparse_decode_plan(p).workspace_bytes == n  # ranks lie behind the counters
    wants("kvq_sparse_decode_launch", p, n)


@pytest.mark.parametrize("decode,budget", [(dict(), 8), (dict(max_pages_per_seq=8), 8),
                                           (dict(batch=256, num_q_heads=64, num_kv_heads=8, max_pages_per_seq=300), 16)])
def test_sparse_decode_without_a_workspace(decode, budget):
    """Ranks in LDS, or none, and an attention of one split."""
    assert kvq.lib().kvq_sparse_decode_workspace_size(ctypes.byref(sparse_params(decode=decode, max_selected=budget))) == 0
