"""kvq_page_map_launch against a sequential restatement: every output integer
is equal, entries without a meaning are left as they were."""
import numpy as np
import pytest
import torch

import _paged_ref as ref
from _gpu import kvq, up

pytestmark = pytest.mark.gpu

OUTS = ("block_table", "free_pages", "new_lengths", "new_free_count", "granted", "token_offsets", "slot_map", "token_seq",
        "token_pos")


def state(rng, B, size, hi, new, spare):
    """A pool in use; spare: free pages relative to what the round needs (0: none at all)."""
    cap_pages = ref.pages_of(hi + new, size)
    lens = rng.integers(0, hi + 1, B)
    lens[rng.random(B) < 0.2] = 0
    add = rng.integers(1, new + 1, B)
    fate = rng.random(B)
    add = np.where(fate < 0.1, 0, add)
    add = np.where((fate >= 0.1) & (fate < 0.25), -lens, add)
    add = np.where((fate >= 0.25) & (fate < 0.4), -rng.integers(1, hi + 2, B), add)
    used = np.array([ref.pages_of(x, size) for x in lens])
    num = B * cap_pages + 3
    ids = rng.permutation(num)
    table = rng.integers(-5, num + 5, (B, cap_pages))  # entries behind the last page mean nothing
    at = 0
    for b in range(B):
        table[b, :used[b]] = ids[at:at + used[b]]
        at += used[b]
    need = sum(max(0, ref.pages_of(x + max(n, 0), size) - ref.pages_of(x, size)) for x, n in zip(lens, add))
    count = min(num - at, int(need * spare))
    free = np.concatenate([ids[at:at + count], rng.integers(-9, 9, num - count)])
    return {"new_tokens": add, "lengths": lens, "block_table": table, "free_pages": free, "free_count": np.array([count])}


def run(st, size, T, in_place=False):
    g = {k: up(np.asarray(v, np.int32)) for k, v in st.items()}
    B = len(st["lengths"])
    fill = lambda n: torch.full((n,), -77, dtype=torch.int32, device="cuda")  # noqa: E731
    more = {} if in_place else {"new_lengths": fill(B), "new_free_count": fill(1)}
    m = kvq.PageMapper(*(g[n] for n in ("new_tokens", "lengths", "block_table", "free_pages", "free_count")), size,
                       slot_map=fill(T), token_seq=fill(T), token_pos=fill(T), **more)
    m()
    torch.cuda.synchronize()
    got = {n: getattr(m, n).cpu().numpy() for n in OUTS}
    if not in_place:
        for n in ("lengths", "free_count", "new_tokens"):
            assert np.array_equal(g[n].cpu().numpy(), st[n]), n
    return got, m


def check(st, size, T, in_place=False):
    want = ref.page_map(*(st[n].tolist() for n in ("new_tokens", "lengths", "block_table", "free_pages")),
                        int(st["free_count"][0]), size, T)
    got, _ = run(st, size, T, in_place)
    for n in OUTS:
        assert np.array_equal(got[n], np.asarray(want[n], np.int64)), n
    return want


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("spare", [0, 0.4, 1.0, 1.5])
@pytest.mark.parametrize("B,size,hi,new", [(1, 16, 40, 1), (1, 1, 1, 1), (7, 16, 100, 1), (64, 16, 300, 30), (65, 5, 90, 33),
                                           (300, 64, 500, 200), (1023, 16, 40, 1), (1025, 7, 33, 9), (4096, 16, 20, 3)])
def test_matches_sequential(B, size, hi, new, spare, in_place):
    rng = np.random.default_rng(B * 31 + size)
    st = state(rng, B, size, hi, new, spare)
    rows = int(np.maximum(st["new_tokens"], 0).sum())
    check(st, size, rows + 11, in_place)


@pytest.mark.parametrize("seed", range(12))
def test_random_rounds(seed):
    rng = np.random.default_rng(seed)
    B, size = int(rng.integers(1, 200)), int(rng.choice([1, 3, 16, 64, 128]))
    st = state(rng, B, size, int(rng.integers(1, 700)), int(rng.integers(1, 400)), float(rng.choice([0.3, 0.9, 1.2])))
    rows = int(np.maximum(st["new_tokens"], 0).sum())
    check(st, size, max(1, int(rows * rng.choice([0.5, 1.0, 1.1]))), bool(seed % 2))


def test_many_rows():
    """Tens of thousands of packed rows."""
    st = state(np.random.default_rng(3), 50, 64, 3000, 4000, 1.0)
    check(st, 64, int(np.maximum(st["new_tokens"], 0).sum()) + 100)


def test_no_rows_and_no_arrays():
    st = state(np.random.default_rng(5), 33, 16, 100, 20, 1.0)
    want = ref.page_map(*(st[n].tolist() for n in ("new_tokens", "lengths", "block_table", "free_pages")),
                        int(st["free_count"][0]), 16, 0)
    got, _ = run(st, 16, 0)
    for n in OUTS:
        assert np.array_equal(got[n], np.asarray(want[n], np.int64)), n
    g = {k: up(np.asarray(v, np.int32)) for k, v in st.items()}
    m = kvq.page_map(g["new_tokens"], g["lengths"], g["block_table"], g["free_pages"], g["free_count"], 16)
    want = ref.page_map(*(st[n].tolist() for n in ("new_tokens", "lengths", "block_table", "free_pages")),
                        int(st["free_count"][0]), 16, 10**6)
    assert m.granted.tolist() == want["granted"] and m.lengths.tolist() == want["new_lengths"]
    assert m.free_count.tolist() == want["new_free_count"] and m.slot_map is None


def test_lengths_and_requests_at_the_ends_of_32_bits():
    """Lengths and counts outside their range are clamped; requests near 2^31 saturate the offsets and are refused."""
    big = 2**31 - 1
    st = {"new_tokens": np.array([big, 3, -big - 1, big, 2, -1]), "lengths": np.array([5, -7, big, big, 3, -big - 1]),
          "block_table": np.arange(24).reshape(6, 4), "free_pages": np.arange(100, 130), "free_count": np.array([big])}
    check(st, 16, 50)
    st["free_count"] = np.array([-3])
    check(st, 16, 50)


def test_bad_page_ids_give_no_slot():
    st = {"new_tokens": np.array([2, 3]), "lengths": np.array([3, 0]), "block_table": np.array([[99, 0], [0, 0]]),
          "free_pages": np.array([0, -4, 1]), "free_count": np.array([2])}
    check(st, 16, 6)


def test_rounds_in_place_in_a_graph():
    """A step captured once and replayed: each replay goes on from the state that the one before left."""
    B, size, steps = 40, 16, 25
    rng = np.random.default_rng(11)
    num, per = 200, 12
    free = rng.permutation(num)
    g = {"new_tokens": up(np.ones(B, np.int32)), "lengths": up(np.zeros(B, np.int32)),
         "block_table": up(np.zeros((B, per), np.int32)), "free_pages": up(free.astype(np.int32)),
         "free_count": up(np.array([num], np.int32))}
    slots = torch.empty(B, dtype=torch.int32, device="cuda")
    m = kvq.PageMapper(*(g[n] for n in ("new_tokens", "lengths", "block_table", "free_pages", "free_count")), size,
                       slot_map=slots)
    m()  # eager, then a replay for each step
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m()
    want = {"lengths": [0] * B, "block_table": [[0] * per] * B, "free_pages": free.tolist(), "free_count": num}
    for step in range(steps):
        add = [1] * B if step % 7 else [1 if b % 3 else -5 for b in range(B)]
        if step:
            g["new_tokens"].copy_(up(np.array(add, np.int32)))
            graph.replay()
        else:
            add = [1] * B
        torch.cuda.synchronize()
        w = ref.page_map(add, want["lengths"], want["block_table"], want["free_pages"], want["free_count"], size, B)
        want = {"lengths": w["new_lengths"], "block_table": w["block_table"], "free_pages": w["free_pages"],
                "free_count": w["new_free_count"][0]}
        assert slots.tolist() == w["slot_map"], step
        assert g["lengths"].tolist() == want["lengths"] and g["block_table"].tolist() == want["block_table"]
        assert g["free_pages"].tolist() == want["free_pages"] and g["free_count"].tolist() == [want["free_count"]]


def test_on_another_stream():
    st = state(np.random.default_rng(8), 90, 16, 200, 60, 1.0)
    T = int(np.maximum(st["new_tokens"], 0).sum())
    want = ref.page_map(*(st[n].tolist() for n in ("new_tokens", "lengths", "block_table", "free_pages")),
                        int(st["free_count"][0]), 16, T)
    g = {k: up(np.asarray(v, np.int32)) for k, v in st.items()}
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    slots = torch.empty(T, dtype=torch.int32, device="cuda")
    m = kvq.page_map(g["new_tokens"], g["lengths"], g["block_table"], g["free_pages"], g["free_count"], 16, stream=s,
                     slot_map=slots)
    s.synchronize()
    assert slots.tolist() == want["slot_map"] and m.granted.tolist() == want["granted"]
