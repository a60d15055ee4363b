"""kvq_chunk_attention_launch where V's scales differ: a row keeps the bits of the
tokens that weigh in it, whatever the scales of the others.  Results are held
against float64 within half a step of their type and the roundings counted in
`tolerance`, tighter than the tests of shapes."""
import pytest
import torch

import _share_ref as ref
from _gpu import kvq
from test_gpu_chunk import BF16, F32, attention, pool_at

pytestmark = pytest.mark.gpu


def half_step(x, dtype):
    """Half the distance between neighbouring values of dtype at x (float64)."""
    bits = {BF16: 8, F32: 24}[dtype]
    return torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0**-126))) - bits)


def tolerance(q, k, v, vs, scale, keys, dtype):
    """Float64 result of rows q [n, d] over keys k, values v (float64 [L, d]) with scales vs, and what may be off:
    * a score: its sum's fp32 roundings and q's limbs, as _share_ref.attend counts them, then 2^-21 for exponentials
      (one of a weight and those of two joins);
    * bf16: a weight is rounded to f16, V's scale too, and their product with a code: 3 times 2^-11; fp32: weights in
      two f16 limbs, 2^-22;
    * a weight below f16's normal range is off by 2^-25 where the largest is 2^-1 at least (fp32: its low limb, 2^6);
    * sums: 2^-23 for each 16 keys and a few for the joins."""
    L, d = k.shape
    t = torch.arange(L, device=q.device)
    s = torch.where(t < keys[:, None], q @ k.T.contiguous() * scale, -torch.inf)
    p = s.softmax(-1)
    mag = q.abs() @ k.abs().T.contiguous() * scale
    bf16 = dtype is BF16
    eps = mag * ((d + 24) * 2.0**-24 + 2.0**-23 + 6 * 2.0**-24) + 3 * 2.0**-21
    size = p @ v.abs()
    err = ((p * eps) @ v.abs() + (p * eps).sum(-1, keepdim=True) * size + size * (3 * 2.0**-11 if bf16 else 2.0**-22)
           + size * (L / 16 + 24) * 2.0**-23 + L * (2.0**-24 if bf16 else 2.0**-31) * 127 * (p * vs.abs()).amax(-1, keepdim=True))
    out = p @ v
    return out, err + half_step(out.abs() + err, dtype)


def check(i, **kw):
    attention(i, **kw)()
    torch.cuda.synchronize()
    q, offsets, dtype = i["q"], i["token_offsets"].tolist(), i["q"].dtype
    d, Hkv = q.shape[2], i["k"].shape[1]
    G = q.shape[1] // Hkv
    worst = 0.0
    for b, length in enumerate(i["lengths"].tolist()):
        r0, r1 = offsets[b], offsets[b + 1]
        keys = (torch.arange(r1 - r0, device="cuda") + length - (r1 - r0) + 1).repeat_interleave(G)
        k, v = (ref.values(i[c], i[c + "s"], i["block_table"][b], length) for c in "kv")
        vs = ref.values(torch.ones_like(i["v"][..., :1]), i["vs"], i["block_table"][b], length)[..., 0]
        for h in range(Hkv):
            x = q[r0:r1, h * G:(h + 1) * G].double().flatten(0, 1)
            want, tol = tolerance(x, k[h], v[h], vs[h], d**-0.5, keys, dtype)
            got = i["out"][r0:r1, h * G:(h + 1) * G].double().flatten(0, 1)
            off = ((got - want).abs() / tol).nan_to_num(nan=1e9, posinf=1e9)
            worst = max(worst, off.max().item())
            assert worst <= 1.0, (b, h, worst, torch.nonzero(off > 1)[0].tolist())
    return worst


def sink(i, b, at, ratio):
    """Token `at` of sequence b takes nearly all the weight of every row, with a V scale `ratio` of what it was."""
    p, at = pool_at(i, b, at)
    q = i["q"].float()
    q[:, :, 0] = 30.0
    i["q"] = q.to(i["q"].dtype)
    i["k"][:, :, :, 0] = 0
    i["k"][p, :, at] = 0
    i["k"][p, :, at, 0] = 127
    i["ks"][p, :, at] = 0.1
    i["vs"][p, :, at] *= ratio


# ---- ratios of scales -----------------------------------------------------------
@pytest.mark.parametrize("half_steps", range(-36, -25))
@pytest.mark.parametrize("n", [30, 3])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_the_token_with_the_weight_has_a_tiny_scale(half_steps, n, dtype):
    for seed, d in ((0, 64), (1, 128), (2, 96)):
        i = ref.batch(seed, [(200, n)], 4, 1, d, 16, dtype)
        sink(i, 0, 5 + seed, 2.0 ** (half_steps / 2))
        check(i)


@pytest.mark.parametrize("bits", [-19, -23, -30, -41, -57, -70])
@pytest.mark.parametrize("n", [30, 3])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_the_token_with_the_weight_has_a_scale_far_below(bits, n, dtype):
    for seed, d in ((0, 64), (1, 192), (2, 256)):
        i = ref.batch(seed, [(200, n), (900, n)], 4, 1, d, 16, dtype)
        sink(i, 0, 5 + seed, 2.0**bits)
        check(i)


@pytest.mark.parametrize("gap", [4.0, 12.0, 20.0, 26.0, 40.0])
@pytest.mark.parametrize("n", [30, 3])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_the_token_with_the_weight_has_the_value_zero(gap, n, dtype):
    """Its score is about `gap` (log2) above the others', of whose weights the output then consists."""
    for seed, d in ((0, 64), (1, 128)):
        i = ref.batch(seed, [(200, n)], 4, 1, d, 16, dtype)
        sink(i, 0, 5, 0.0)
        p, at = pool_at(i, 0, 5)
        i["v"][p, :, at] = 0
        i["ks"][p, :, at] = gap * 0.6931 * d**0.5 / (30.0 * 127)
        check(i)


@pytest.mark.parametrize("low,high", [(-80, 58), (-85, -30), (-20, 59), (-70, 10)])
@pytest.mark.parametrize("pairs", [[(2000, 1)], [(2000, 70)], [(700, 1)] * 130, [(700, 40)] * 130])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_scales_of_two_sizes(low, high, pairs, dtype):
    """The first and the second half of the tokens far apart: the weights' sum keeps both."""
    for first, second in ((low, high), (high, low)):
        i = ref.batch(21, pairs, 4, 2, 64, 16, dtype)
        g = torch.Generator(device="cuda")
        g.manual_seed(5)
        r = torch.rand(i["vs"].shape, generator=g, device="cuda")
        x = torch.exp2(r + second)
        page = i["k"].shape[2]
        for b, (length, _) in enumerate(pairs):
            ids = i["block_table"][b, :length // 2 // page].long()
            x[ids] = torch.exp2(r[ids] + first)
        i["vs"] = torch.where(torch.isnan(i["vs"]), i["vs"], x)
        check(i)


@pytest.mark.parametrize("step", [0.25, -0.25, 0.07, -0.07])
@pytest.mark.parametrize("pairs", [[(230, 230)], [(230, 9)], [(200, 200), (230, 64), (7, 7)] * 20])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_scales_that_grow_from_token_to_token(step, pairs, dtype):
    """The largest scales of a tile belong to tokens that its first rows do not see, or the smallest."""
    for d in (64, 128, 256):
        i = ref.batch(d, pairs, 4, 2, d, 16, dtype)
        page = i["k"].shape[2]
        for b, (length, _) in enumerate(pairs):
            t = torch.arange(length, device="cuda")
            i["vs"][i["block_table"][b, t // page].long(), :, t % page] = torch.exp2(step * t - 20.0)[:, None]
        check(i)


@pytest.mark.parametrize("tiny", [1e-7, 1e-20, 0.0])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_token_of_tiny_value_does_not_slow_its_sequence(tiny, dtype):
    """A padding token's V row next to nothing; 512 tokens over 4096 stay on the matrix cores (in fp32, a row at a time,
    they take hundreds of times as long)."""
    i = ref.batch(22, [(4096, 512)], 8, 2, 128, 16, dtype)
    ms = []
    for value in (0.01, tiny):
        p, at = pool_at(i, 0, 3)
        i["vs"][p, :, at] = value
        h = attention(i)
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        times = []
        for _ in range(5):
            begin.record()
            h()
            end.record()
            torch.cuda.synchronize()
            times.append(begin.elapsed_time(end))
        ms.append(min(times))
    assert ms[1] < 5 * ms[0], ms


# ---- scales of zero -------------------------------------------------------------
def values_of_zero(i, tokens, low):
    """V scales of 2^low to 2^(low + 1), but zero for `tokens` of every sequence."""
    g = torch.Generator(device="cuda")
    g.manual_seed(-low)
    small = torch.exp2(torch.rand(i["vs"].shape, generator=g, device="cuda") + low)
    i["vs"] = torch.where(torch.isnan(i["vs"]), i["vs"], small)
    page = i["k"].shape[2]
    t = torch.tensor(list(tokens), device="cuda")
    ids = i["block_table"].long()[:, t // page]
    i["vs"][ids, :, t % page] = 0.0
    i["v"][ids, :, t % page] = 0


@pytest.mark.parametrize("tokens", [range(0, 64), range(0, 256), range(1000, 1100), range(960, 1024), range(1930, 2000)])
@pytest.mark.parametrize("low", [-40, -36, -30, -20])
@pytest.mark.parametrize("n", [70, 5, 1])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_tokens_of_value_zero_beside_small_scales(tokens, low, n, dtype):
    i = ref.batch(7, [(2000, n)], 4, 2, 64, 16, dtype)
    values_of_zero(i, tokens, low)
    check(i)


@pytest.mark.parametrize("tokens", [range(0, 32), range(0, 64), range(256, 330)])
@pytest.mark.parametrize("low", [-40, -30, -20])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_tokens_of_value_zero_in_a_batch_that_fills_the_chip(tokens, low, dtype):
    """Nothing is split, so a wave has blocks behind the one whose values are zero."""
    i = ref.batch(8, [(600, 1)] * 130, 4, 2, 64, 16, dtype)
    values_of_zero(i, tokens, low)
    check(i)
