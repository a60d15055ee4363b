"""kvq_chunk_attention_launch against float64 within a tolerance derived from its
roundings (_share_ref.attend): shapes, masks, strides, garbage around the tokens,
value ranges, streams, graphs and shared workspaces."""
import numpy as np
import pytest
import torch

import _share_ref as ref
from _gpu import kvq

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def attention(i, causal=True, out=None, **kw):
    out = i["out"] if out is None else out
    return kvq.ChunkAttention(i["q"], i["k"], i["v"], i["ks"], i["vs"], i["block_table"], i["lengths"], i["token_offsets"],
                              out, granted=i["granted"], causal=causal, **kw)


def check(i, causal=True, scale=None, **kw):
    if scale is not None:
        kw["softmax_scale"] = scale
    h = attention(i, causal, **kw)
    h()
    torch.cuda.synchronize()
    compare(i["out"], i, causal, scale)
    return h


def compare(out, i, causal=True, scale=None):
    want, tol, written = ref.chunk(i, causal, scale)
    assert torch.isnan(out[~written]).all()  # rows behind the last sequence
    bad = ~((out.double() - want).abs() <= tol)
    bad[~written] = False
    assert not bad.any(), (torch.nonzero(bad)[:4].tolist(), (out.double() - want)[bad][:4].tolist(), tol[bad][:4].tolist())


# (length, new tokens): none held, one, a whole prompt, odd ones, single tokens, none new, a length on a page's and a tile's end.
MIXED = [(1, 1), (0, 0), (77, 77), (200, 1), (64, 64), (129, 3), (50, 0), (333, 40), (128, 128), (65, 17), (16, 1)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("Hq,Hkv,d,page", [(4, 4, 64, 16), (8, 2, 128, 64), (6, 2, 96, 16), (5, 1, 80, 32), (14, 2, 128, 5),
                                           (3, 3, 112, 1), (8, 1, 192, 128), (4, 2, 256, 7), (2, 1, 8, 16), (16, 1, 40, 3),
                                           (128, 1, 64, 16), (100, 1, 64, 32)])
@pytest.mark.parametrize("causal", [True, False])
def test_shapes(Hq, Hkv, d, page, dtype, causal):
    check(ref.batch(Hq * d + page, MIXED, Hq, Hkv, d, page, dtype, refused=(3,)), causal)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("Hq,Hkv,d,page", [(2, 2, 20, 16), (3, 1, 33, 5), (2, 1, 264, 16), (1, 1, 1, 4), (4, 2, 300, 9),
                                           (1, 1, 4096, 8), (129, 1, 64, 16)])
def test_generic(Hq, Hkv, d, page, dtype):
    pairs = [(1, 1), (70, 5), (0, 0), (66, 1), (130, 9)]
    check(ref.batch(d, pairs, Hq, Hkv, d, page, dtype, refused=(3,)))
    check(ref.batch(d, pairs, Hq, Hkv, d, page, dtype), causal=False)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("pairs", [[(5000, 1)], [(5003, 700)], [(1, 1)] * 300, [(9000, 5), (64, 64)], [(2500, 2500)],
                                   [(40, 1)] * 63 + [(4000, 300)], [(300, 1)] * 1000])
def test_lengths(pairs, dtype):
    check(ref.batch(len(pairs), pairs, 8, 2, 64, 16, dtype))


@pytest.mark.parametrize("d,Hq,Hkv", [(128, 32, 8), (96, 24, 24), (192, 16, 2), (256, 8, 4)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_split_and_whole(d, Hq, Hkv, dtype):
    """Few rows over many keys (split), and many rows."""
    check(ref.batch(d, [(8200, 9)], Hq, Hkv, d, 64, dtype))
    check(ref.batch(d, [(1100, 600), (700, 513)], Hq, Hkv, d, 16, dtype))


@pytest.mark.parametrize("n,length", [(9, 4), (200, 3), (64, 0), (5, 1)])
@pytest.mark.parametrize("d", [64, 20])
def test_more_rows_than_tokens(n, length, d):
    """A causal row before the sequence's first token attends nothing: zero."""
    i = ref.batch(n, [(length, n), (100, 7)], 4, 2, d, 16, BF16)
    check(i)
    assert (i["out"][:n - length] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_refused_rows_are_zero(dtype):
    i = ref.batch(5, [(100, 30), (90, 20), (80, 1)], 4, 2, 64, 16, dtype, refused=(0, 2))
    i["granted"][2] = -5  # gave tokens up
    check(i)
    assert (i["out"][:30] == 0).all() and (i["out"][50:51] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_strides(dtype):
    """q as a slice of a fused projection, out as one of a wider tensor; the columns beside stay."""
    i = ref.batch(3, MIXED, 8, 2, 128, 16, dtype, fused=True)
    wide = torch.full((i["q"].shape[0], 10, 128), float("nan"), dtype=dtype, device="cuda")
    i["out"] = wide[:, 1:9]
    check(i)
    assert torch.isnan(wide[:, 0]).all() and torch.isnan(wide[:, 9]).all()


def test_misaligned_rows_take_the_generic_kernel():
    for cols, first in ((8 * 64 + 4, 0), (8 * 64 + 8, 3)):
        i = ref.batch(3, [(100, 9), (70, 1)], 8, 2, 64, 16, BF16)
        wide = torch.zeros((i["q"].shape[0], cols), dtype=BF16, device="cuda")
        wide[:, first:first + 512] = i["q"].flatten(1)
        i["q"] = wide[:, first:first + 512].unflatten(1, (8, 64))
        check(i)


@pytest.mark.parametrize("scale", [1.0, 0.01, 3.0])
def test_softmax_scale(scale):
    i = ref.batch(8, [(300, 33)], 8, 2, 64, 16, F32)
    i["q"] *= 0.1
    check(i, scale=scale)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_contiguous_cache_as_pages(dtype):
    """[B, Hkv, capacity, d] is a pool of B pages of `capacity` tokens."""
    i = ref.batch(4, [(150, 20), (150, 1), (150, 150)], 8, 4, 64, 150, dtype)
    i["block_table"] = torch.arange(3, dtype=torch.int32, device="cuda")[:, None].contiguous()
    for c in ("ks", "vs"):
        i[c] = torch.nan_to_num(i[c], nan=0.01)
    check(i)


@pytest.mark.parametrize("d", [64, 128, 20])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_single_tokens_equal_paged_decode(d, dtype):
    i = ref.batch(9, [(L, 1) for L in (1, 17, 400, 1000)], 8, 2, d, 16, dtype, spare=0)
    attention(i)()
    out = torch.empty((4, 8, d), device="cuda")
    kvq.PagedDecoder(i["q"].float().contiguous(), i["k"], i["v"], i["ks"], i["vs"], i["block_table"], i["lengths"], out)()
    want, tol, _ = ref.chunk(i, True)
    assert ((i["out"].double() - want).abs() <= tol).all()
    # Two results within their tolerances of the same numbers (the decode's: 1e-4 + 1e-3).
    assert ((i["out"].double() - out.double()).abs() <= tol + 1e-4 + 1e-3 * want.abs()).all()


# ---- values --------------------------------------------------------------------
def pool_at(i, b, t):
    page = i["k"].shape[2]
    return int(i["block_table"][b, t // page]), t % page


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d", [128, 20])
def test_scales_that_are_not_finite_stay_with_the_rows_that_see_them(dtype, d):
    for what, value in (("ks", float("nan")), ("vs", float("nan")), ("vs", float("inf")), ("ks", float("inf"))):
        i = ref.batch(6, [(90, 40), (30, 30)], 4, 2, d, 16, dtype)
        p, at = pool_at(i, 0, 70)
        i[what][p, 1, at] = value
        attention(i)()
        out = i["out"].double()
        i[what][p, 1, at] = 0.01
        want, tol, _ = ref.chunk(i, True)
        free = torch.ones((70, 4), dtype=torch.bool, device="cuda")
        free[20:40, 2:] = False  # tokens 70 .. 89 of sequence 0, heads of kv head 1
        assert ((out[:70] - want[:70]).abs() <= tol[:70])[free].all(), (what, value)
        seen = ~torch.isfinite(out[20:40, 2:])
        if (what, value) == ("ks", float("inf")):  # a score of -inf is a weight of zero, one of +inf is NaN
            up = (i["q"][20:40, 2:].double() * i["k"][p, 1, at].double()).sum(-1) > 0
            assert torch.equal(seen.all(-1), up) and torch.equal(seen.any(-1), up)
        else:
            assert seen.all(), (what, value)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_queries_that_are_not_finite_give_nan_in_their_rows(dtype):
    i = ref.batch(6, [(90, 40), (30, 30)], 4, 2, 128, 16, dtype)
    i["q"][3, 1, 5] = float("inf")
    i["q"][41, 0, 100] = float("nan")
    attention(i)()
    out = i["out"].double()
    i["q"][3, 1, 5] = i["q"][41, 0, 100] = 0.0
    want, tol, _ = ref.chunk(i, True)
    bad = torch.zeros((70, 4), dtype=torch.bool, device="cuda")
    bad[3, 1] = bad[41, 0] = True
    assert torch.isnan(out[:70][bad]).all()
    assert ((out[:70] - want[:70]).abs() <= tol[:70])[~bad].all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lo,hi", [(-40, -30), (20, 39), (-100, -50), (50, 100), (-45, 45), (-12, 2), (-30, 0)])
def test_v_scales_of_any_size(lo, hi, dtype):
    """Powers of two apart within one sequence; the rows have to keep the bits of what weighs in them."""
    i = ref.batch(11, [(300, 70), (100, 1), (4500, 2)], 4, 2, 64, 16, dtype)
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    e = torch.rand(i["vs"].shape, generator=g, device="cuda") * (hi - lo) + lo
    i["vs"] = torch.where(torch.isnan(i["vs"]), i["vs"], torch.exp2(e))
    check(i)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_first_token_with_a_tiny_value_and_nearly_all_the_weight(dtype):
    """Attention sinks: the token that takes the weight has a far smaller V scale than the others."""
    for ratio in (2.0**-10, 2.0**-13, 2.0**-20, 2.0**-60):
        i = ref.batch(12, [(200, 30)], 4, 1, 64, 16, dtype)
        p, at = pool_at(i, 0, 0)
        q = i["q"][:30].float()
        # The first token's key along the queries' common direction.
        q[:, :, 0] = 30.0
        i["q"][:30] = q.to(dtype)
        i["k"][p, 0, at] = 0
        i["k"][p, 0, at, 0] = 127
        i["ks"][p, 0, at] = 0.04
        i["vs"][p, 0, at] *= ratio
        check(i)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_zero_and_negative_scales(dtype):
    i = ref.batch(13, [(200, 30), (64, 64)], 4, 2, 64, 16, dtype)
    i["vs"][:, :, ::3] = 0.0
    i["ks"][:, 0, ::4] = 0.0
    i["vs"][:, :, 1::5] *= -1.0
    i["ks"][:, :, 1::7] *= -1.0
    for c in ("ks", "vs"):
        i[c] = torch.nan_to_num(i[c], nan=0.0)
    check(i)
    i["vs"].zero_()
    check(i)
    assert (i["out"][:94] == 0).all()


@pytest.mark.parametrize("size", [1e-38, 1e-20, 1e20, 1e30])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_queries_and_key_scales_of_any_size(size, dtype):
    i = ref.batch(14, [(200, 30)], 4, 2, 64, 16, dtype)
    i["q"] *= size
    i["ks"] = i["ks"] * (0.1 / size)
    check(i)
    i["q"].zero_()
    check(i)


def test_outlier_channels_in_bf16():
    """One channel of q a thousand times the others, and a small one in K: no bits of the others are lost."""
    i = ref.batch(15, [(300, 40)], 8, 2, 128, 16, BF16)
    i["q"][:, :, 7] *= 1000.0
    i["k"][..., 7] = (i["k"][..., 7].float() / 127).round().to(torch.int8)
    i["ks"] *= 0.2
    check(i)


# ---- memory, streams, graphs -----------------------------------------------------
def test_offsets_past_32_bits():
    """A pool of more than 4 GB: pages at its end."""
    Hkv, page, d = 8, 64, 128
    P = (1 << 32) // (Hkv * page * d) + 40
    small = ref.batch(16, [(500, 20), (70, 1)], 16, Hkv, d, page, BF16)
    n = small["k"].shape[0]
    big = dict(small)
    for c in "kv":
        big[c] = torch.empty((P, Hkv, page, d), dtype=torch.int8, device="cuda")
        big[c][-n:] = small[c]
        big[c + "s"] = torch.full((P, Hkv, page), float("nan"), device="cuda")
        big[c + "s"][-n:] = small[c + "s"]
    big["block_table"] = small["block_table"] + (P - n)
    attention(big)()
    compare(big["out"], small)


def test_ids_outside_the_pool_are_clamped():
    i = ref.batch(17, [(100, 10)], 4, 2, 64, 16, BF16)
    i["ks"], i["vs"] = (torch.nan_to_num(i[c], nan=0.01) for c in ("ks", "vs"))
    last = i["k"].shape[0] - 1
    i["block_table"][0, 2], i["block_table"][0, 4] = 1 << 30, -7
    attention(i)()
    got = i["out"].clone()
    i["block_table"][0, 2], i["block_table"][0, 4] = last, 0
    compare(got, i)


def test_other_stream_and_two_calls_at_once():
    i, j = (ref.batch(s, [(4000, 30), (900, 1)], 8, 2, 128, 16, BF16) for s in (18, 19))
    a, b = attention(i), attention(j)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for h, s in zip((a, b), streams):
            h(s)
    torch.cuda.synchronize()
    compare(i["out"], i)
    compare(j["out"], j)


def test_one_workspace_for_all_shapes():
    shapes = [([(8000, 9)], 8, 2, 128, BF16), ([(300, 40)] * 3, 8, 8, 64, F32), ([(5000, 3), (70, 2)], 4, 1, 256, F32),
              ([(6000, 1)] * 5, 32, 8, 96, BF16)]
    batches = [ref.batch(20 + n, pairs, Hq, Hkv, d, 16, dtype) for n, (pairs, Hq, Hkv, d, dtype) in enumerate(shapes)]
    sizes = [attention(i).ws_bytes for i in batches]
    ws = torch.empty(max(sizes), dtype=torch.uint8, device="cuda")
    kvq.workspace_init(ws, max(sizes))
    handles = [attention(i, workspace=lambda n: ws) for i in batches]
    for order in ((0, 1, 2, 3), (3, 1, 0, 2), (2, 2, 3, 0)):
        for n in order:
            batches[n]["out"].fill_(float("nan"))
            handles[n]()
            compare(batches[n]["out"], batches[n])


@pytest.mark.parametrize("pairs", [[(3000, 20)], [(100, 1)] * 40 + [(900, 200)]])
def test_graph_replays_with_new_lengths(pairs):
    """A captured call reads lengths, offsets and tables at every replay."""
    i = ref.batch(25, pairs, 8, 2, 128, 16, BF16)
    h = attention(i, max_seq_len=int(i["lengths"].max()))
    h()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        h()
    full, offsets = i["lengths"].clone(), i["token_offsets"].clone()
    for step in range(4):
        i["lengths"].copy_((full - 17 * step).clamp(min=0))
        i["token_offsets"].copy_((offsets - step).clamp(min=0))
        i["out"].fill_(float("nan"))
        g.replay()
        torch.cuda.synchronize()
        compare(i["out"], i)
        i["out"].fill_(float("nan"))
        h()
        compare(i["out"], i)


def test_results_do_not_depend_on_the_run():
    i = ref.batch(26, [(7000, 11), (300, 90)], 8, 2, 128, 16, F32)
    h = attention(i)
    h()
    first = i["out"].clone()
    for _ in range(5):
        h()
        assert torch.equal(i["out"][:101], first[:101])


def test_no_rows():
    i = ref.batch(27, [(100, 0), (0, 0)], 4, 2, 64, 16, BF16)
    check(i)
    i["q"], i["out"] = i["q"][:0], i["out"][:0]
    attention(i)()
    torch.cuda.synchronize()


def test_function_and_lengths_over_the_bound():
    i = ref.batch(28, [(100, 10), (300, 20)], 4, 2, 64, 16, BF16, spare=0)
    args = [i[n] for n in ("q", "k", "v", "ks", "vs", "block_table", "lengths", "token_offsets")]
    out = kvq.chunk_attention(*args)
    want, tol, _ = ref.chunk(i, True)
    assert ((out.double() - want).abs() <= tol).all()
    out = kvq.chunk_attention(*args, max_seq_len=150)  # the longer one counts as 150 tokens
    i["lengths"][1] = 150
    want, tol, _ = ref.chunk(i, True)
    assert ((out.double() - want).abs() <= tol).all()
