"""Sparse decode and page maps at the edges of what their headers allow:
workspaces shared by different shapes, misaligned tensors, pages shared by
sequences, ranks kept in memory, many workgroups in place."""
import ctypes

import numpy as np
import pytest
import torch

import _paged_ref as ref
from _gpu import down, kvq, poisoned, up
from test_gpu_page_map import state as map_state
from test_gpu_sparse import Problem, decoder, verify

pytestmark = pytest.mark.gpu


def shared_workspace_step(p, ws, budget):
    g = p.gpu()
    dec, out, sel, n = decoder(p, g, budget, workspace=lambda nbytes: ws)
    assert dec.ws_bytes <= ws.numel()
    dec()
    torch.cuda.synchronize()
    verify(p, out, sel, n, budget, 1, 1)
    return dec.ws_bytes


def test_one_workspace_for_every_shape():
    """A workspace zero-filled once serves shapes whose ranks lie in it and shapes that count arrivals in it, in any order."""
    rng = np.random.default_rng(1)
    ws = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    kvq.workspace_init(ws)
    generic = Problem(rng, [16 * 300, 700], 2, 2, 20, 16)       # one workgroup a unit, ranks in memory
    split = Problem(rng, [16 * 700, 16 * 130 + 1], 4, 2, 64, 16)  # several workgroups a unit
    short = Problem(rng, [50, 20], 4, 2, 64, 16)
    many = Problem(rng, [16 * 13000], 1, 1, 32, 16)               # ranks beyond LDS
    used = [shared_workspace_step(p, ws, 8) for p in (split, generic, split, many, short, generic, split, many, split)]
    assert used[0] and used[1]


@pytest.mark.parametrize("which", ["q", "k", "v", "bounds", "ks", "scale"])
def test_misaligned_tensors(which):
    """Contiguous tensors at addresses that are not multiples of 16 bytes."""
    rng = np.random.default_rng(2)
    p = Problem(rng, [1000, 16 * 30 + 1], 4, 2, 64, 16)
    g = p.gpu()
    t = g[which]
    moved = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape)
    moved.copy_(t)
    g[which] = moved
    assert moved.data_ptr() % 16 and moved.is_contiguous()
    dec, out, sel, n = decoder(p, g, 9)
    dec()
    torch.cuda.synchronize()
    verify(p, out, sel, n, 9, 1, 1)
    b, s = kvq.new_bounds(g["k"])
    if which in ("k", "bounds", "ks"):
        kvq.page_bounds(g["k"], g["ks"], g["table"], g["lengths"], g["bounds"], g["scale"])
        kvq.page_bounds(up(p.k), up(p.ks), g["table"], g["lengths"], b, s)
        for i, m in enumerate(p.lens):
            ids = torch.from_numpy(p.table[i, :ref.pages_of(m, 16)].astype(np.int64)).cuda()
            assert torch.equal(g["bounds"][ids], b[ids]) and torch.equal(g["scale"][ids], s[ids])


def test_ranks_in_memory_of_unsplit_units():
    """256 sequences that share more pages than LDS holds ranks of, each in another order."""
    rng = np.random.default_rng(3)
    pages, B, d = 12500, 256, 32
    p = Problem(rng, [pages], 1, 1, d, 1, spare=0)
    p.lens = [pages - int(x) for x in rng.integers(0, 300, B)]
    p.table = np.stack([rng.permutation(pages) for _ in range(B)]).astype(np.int32)
    p.q = rng.standard_normal((B, 1, d)).astype(np.float32)
    g = p.gpu()
    dec, out, sel, n = decoder(p, g, 20)
    dec()
    torch.cuda.synchronize()
    verify(p, out, sel, n, 20, 1, 1)


def test_pages_shared_by_sequences():
    """A common prefix, whose last page becomes whole for both sequences in the same step."""
    rng = np.random.default_rng(4)
    p = Problem(rng, [16 * 20 + 1, 16 * 20 + 1], 4, 2, 64, 16)
    p.table[1, :20] = p.table[0, :20]
    p.set_bounds()
    before = p.table[0, 19]
    p.bounds[before], p.scale[before] = 1, 1e9  # stale: this step writes them
    g = p.gpu()
    dec, out, sel, n = decoder(p, g, 6)
    dec()
    torch.cuda.synchronize()
    p.set_bounds()
    verify(p, out, sel, n, 6, 1, 1)
    assert np.array_equal(down(g["bounds"])[before], p.bounds[before])


@pytest.mark.parametrize("last", [1, 2, 3])
def test_opened_page_with_kept_pages(last):
    """The page that becomes whole is written whether it is ranked, kept, or the sequence is attended whole."""
    rng = np.random.default_rng(5)
    p = Problem(rng, [16 * 30 + 1, 16 * 2 + 1, 17, 16 * 30], 2, 2, 64, 16)
    stale = [p.table[b, (n - 1) // 16 - 1] for b, n in enumerate(p.lens) if n > 1 and n % 16 == 1]
    for x in stale:
        p.bounds[x], p.scale[x] = -3, 7.0
    g = p.gpu()
    dec, out, sel, n = decoder(p, g, 8, last=last)
    dec()
    torch.cuda.synchronize()
    p.set_bounds()
    verify(p, out, sel, n, 8, 1, last)
    for x in stale:
        assert np.array_equal(down(g["bounds"])[x], p.bounds[x]) and np.array_equal(down(g["scale"])[x], p.scale[x])


def test_single_tokens_and_pages_of_one_token():
    rng = np.random.default_rng(6)
    for size in (1, 16):
        p = Problem(rng, [1, 2, 3, 1], 4, 2, 64, size)
        g = p.gpu()
        dec, out, sel, n = decoder(p, g, 2)
        dec()
        torch.cuda.synchronize()
        verify(p, out, sel, n, 2, 1, 1)


def test_page_map_in_place_over_many_workgroups():
    """Replays of a captured map of many rows, in place: lengths and counts are written when every workgroup has read them."""
    rng = np.random.default_rng(7)
    B, size, T, per, num = 64, 16, 20000, 400, 9000
    st = {"lengths": [0] * B, "block_table": [[0] * per] * B, "free_pages": rng.permutation(num).tolist(), "free_count": num}
    g = {k: up(np.asarray([v] if k == "free_count" else v, np.int32)) for k, v in st.items()}
    add = up(np.zeros(B, np.int32))
    rows = [torch.empty(T, dtype=torch.int32, device="cuda") for _ in range(3)]
    m = kvq.PageMapper(add, g["lengths"], g["block_table"], g["free_pages"], g["free_count"], size, slot_map=rows[0],
                       token_seq=rows[1], token_pos=rows[2])
    assert m.params.max_tokens == T and m.ws is not None
    m()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m()
    for step in range(6):
        n = rng.integers(0, 500, B)
        n[rng.random(B) < 0.2] *= -3
        add.copy_(up(n.astype(np.int32)))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        w = ref.page_map(n, st["lengths"], st["block_table"], st["free_pages"], st["free_count"], size, T)
        st = {"lengths": w["new_lengths"], "block_table": w["block_table"], "free_pages": w["free_pages"],
              "free_count": w["new_free_count"][0]}
        assert rows[0].tolist() == w["slot_map"] and rows[1].tolist() == w["token_seq"] and rows[2].tolist() == w["token_pos"]
        assert g["lengths"].tolist() == st["lengths"] and g["block_table"].tolist() == st["block_table"]
        assert g["free_pages"].tolist() == st["free_pages"] and g["free_count"].tolist() == [st["free_count"]]


def test_tensors_dropped_while_a_side_stream_is_busy():
    """Inputs, outputs and workspaces of a launch on another stream are not handed out again before it has run."""
    st = map_state(np.random.default_rng(8), 90, 16, 200, 60, 1.0)
    T = int(np.maximum(st["new_tokens"], 0).sum())
    want = ref.page_map(*(st[n].tolist() for n in ("new_tokens", "lengths", "block_table", "free_pages")),
                        int(st["free_count"][0]), 16, T)
    g = {k: up(np.asarray(v, np.int32)) for k, v in st.items()}
    slots = [torch.empty(T, dtype=torch.int32, device="cuda") for _ in range(3)]
    s = torch.cuda.Stream()
    busy = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        for _ in range(20):
            busy = busy @ busy * 1e-4
    junk = []
    for out in slots:
        args = [g[n].clone() for n in ("new_tokens", "lengths", "block_table", "free_pages", "free_count")]
        s.wait_stream(torch.cuda.current_stream())
        kvq.page_map(*args, 16, stream=s, slot_map=out)
        sizes = [a.numel() for a in args] + [90, 91]
        del args
        junk += [torch.full((n,), 123456, dtype=torch.int32, device="cuda") for n in sizes]
    torch.cuda.current_stream().synchronize()
    s.synchronize()
    for out in slots:
        assert out.tolist() == want["slot_map"]
    for x in junk:
        assert bool((x == 123456).all())


def test_slot_read_of_one_token_or_one_head_with_any_strides():
    rng = np.random.default_rng(9)
    pool = [up(rng.integers(-127, 128, (3, 1, 16, 64)).astype(np.int8)) for _ in "kv"] + \
           [up(rng.random((3, 1, 16)).astype(np.float32)) for _ in "kv"]
    k = torch.empty((5, 1, 64), device="cuda")
    v = torch.empty((5, 7, 64), device="cuda")[:, :1].contiguous().as_strided((5, 1, 64), (64, 1, 1))
    kvq.slot_read(up(np.arange(5, dtype=np.int32)), *pool, k, v)
    want = pool[1][0, 0, :5].float() * pool[3][0, 0, :5, None]
    assert torch.equal(v[:, 0], want)


def test_plan_and_workspace_agree():
    rng = np.random.default_rng(10)
    p = Problem(rng, [3000, 100], 4, 2, 128, 16)
    dec, *_ = decoder(p, p.gpu(), 20)
    info = kvq.sparse_decode_plan(dec.params)
    assert info.workspace_bytes == dec.ws_bytes
    assert info.kernel == kvq.KERNEL_DECODE_MFMA
    assert kvq.lib().kvq_sparse_decode_launch(ctypes.byref(dec.params), None, 0, None) == (kvq.HIP_ERROR_INVALID_VALUE if dec.ws_bytes else 0)


@pytest.mark.parametrize("G", [64, 65])
def test_many_heads_over_many_pages(G):
    """The most columns and ranks that a workgroup keeps, and one head more (which takes the generic selection)."""
    rng = np.random.default_rng(11)
    p = Problem(rng, [5900, 64], G, 1, 256, 1)
    g = p.gpu()
    dec, out, sel, n = decoder(p, g, 300)
    dec()
    torch.cuda.synchronize()
    verify(p, out, sel, n, 300, 1, 1)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("d", [64, 20])
def test_queries_that_are_not_finite(d, bad):
    """Their own heads give NaN; whatever is selected are pages of the sequence, and the other heads attend those."""
    rng = np.random.default_rng(12)
    p = Problem(rng, [16 * 50 + 3, 16 * 40], 4, 2, d, 16)
    p.q[0, 1, 3] = bad     # head 1 of the first kv head
    p.q[1, 4:] = bad       # all of the second kv head
    g = p.gpu()
    dec, out, sel, n = decoder(p, g, 9)
    dec()
    torch.cuda.synchronize()
    picked, out, n = down(sel), down(out), down(n)
    for b, length in enumerate(p.lens):
        of_page = {int(x): i for i, x in enumerate(p.table[b, :ref.pages_of(length, 16)])}
        for h in range(2):
            entries = [of_page[int(x) // 2] for x in picked[b, h]]
            assert (picked[b, h] % 2 == h).all() and entries == sorted(set(entries))
            assert entries[0] == 0 and entries[-1] == len(of_page) - 1 and n[b, h] == 8 * 16 + (length - 1) % 16 + 1
            rows = p.rows(b, h, entries)
            for i in range(4):
                q = p.q[b, 4 * h + i:4 * h + i + 1]
                if not np.isfinite(q).all():
                    assert np.isnan(out[b, 4 * h + i]).all()
                    continue
                exact = ref.attend(q, *rows, 1 / np.sqrt(d))
                assert np.abs(out[b, 4 * h + i] - exact[0]).max() <= ref.attend_tolerance(q, *rows, 1 / np.sqrt(d))


@pytest.mark.parametrize("length", [16 * 40 + 1, 16 * 40 + 9])
def test_uniform_steps_append_as_those_with_lengths(length):
    """Without a lengths array, every sequence of max_seq_len tokens: the same pages, bits, bounds and appended rows."""
    rng = np.random.default_rng(13)
    p = Problem(rng, [length] * 3, 4, 2, 64, 16)
    new = [up(rng.standard_normal((3, 2, 64)).astype(np.float32)) for _ in "kv"]
    got = []
    for lengths in (True, False):
        g = p.gpu()
        dec, out, sel, n = decoder(p, g, 7, lengths=lengths, max_seq_len=length, k_new=new[0], v_new=new[1])
        dec()
        torch.cuda.synchronize()
        got.append([out, sel, n] + [g[x] for x in ("k", "v", "ks", "vs", "bounds", "scale")])
    for a, b in zip(*got):
        assert torch.equal(a, b)
    at = p.table[:, (length - 1) // 16], (length - 1) % 16
    want, scale = ref.quantise(down(new[0]))
    assert np.array_equal(down(got[1][3])[at[0], :, at[1]], want)
    assert np.array_equal(down(got[1][5])[at[0], :, at[1]], scale)
