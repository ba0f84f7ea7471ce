"""Scores of the 4-bit decode where they are hard to hold: keys with a large zero, scores far beyond
the weights' range, and queries up to the end of bf16's."""
import numpy as np
import pytest
import torch

import tqkv

from int4_reference import HALF_STEP, VALID, f64, pack, spread, unpack, values

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _signs(S, D, bs, seed):
    """A V cache [1, 1, S, D] of rows of -1 and +1 (0.1333 * 15 - 1), and each row's sign."""
    sign = np.random.default_rng(seed).integers(0, 2, S)
    codes = pack(np.repeat((15 * sign)[:, None], D, 1).astype(np.uint8))
    params = np.tile(np.array([2 / 15, -1], np.float16), (S, D // bs, 1))
    return torch.from_numpy(codes)[None, None].cuda(), torch.from_numpy(params)[None, None].cuda(), sign


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("G", [1, 3, 6, 12])
@pytest.mark.parametrize("D,bs", VALID)
def test_keys_whose_zero_is_large_beside_their_scale(D, bs, G, dtype):
    """Zeros of +-4000 times a block's sum of q.  The block holds 1 and -1 beside multiples of 2^-18, so
    that its sum, U 2^-14 with U a multiple of 1 / 16 that is none of 1, is exact in fp32 in every
    order, and its zero terms, which decide the scores, are exact in fp32 too.

    Bound.  A score's terms are those products and codes * scale * q with a scale of 2^-12: with fp32
    sums, which a tensor core may truncate, it is off by (D + 16) 2^-23 of the sum of their magnitudes;
    the argument and the value of 2^x by (|score| + 64) 2^-23 + 2^-22; p * scale by fp16's half step."""
    S, nb = 100, D // bs
    g = np.random.default_rng(D + bs + G)
    U = np.array([20.4375, 5.4375, 1.4375])[{1: 0, 2: 1, 4: 1}[nb]]
    q = np.zeros((G, D))
    for h in range(G):
        for b in range(nb):
            part = np.zeros(bs)
            part[0], part[1] = 1, -1
            n = int(U * 16)
            part[2:12] = n // 10
            part[2:2 + n % 10] += 1
            part[2:12] *= 2.0 ** -18
            q[h, b * bs:(b + 1) * bs] = g.permutation(part)
    qt = torch.from_numpy(q)[None].to(dtype).cuda()
    assert np.array_equal(f64(qt)[0], q)
    vq, vs, sign = _signs(S, D, bs, D + G)
    kc = g.integers(0, 16, (S, D)).astype(np.uint8)
    ks = np.empty((S, nb, 2), np.float16)
    ks[..., 0] = 2.0 ** -12
    ks[..., 1] = np.where(sign, 4000, -4000)[:, None]
    kq = torch.from_numpy(pack(kc))[None, None].cuda()
    o = tqkv.decode_int4(qt, kq, torch.from_numpy(ks)[None, None].cuda(), vq, vs, bs)

    s, z = spread(ks, bs)
    v = values(vq, vs, bs)[0, 0]
    for h in range(G):
        t = (kc * s + z) @ q[h] / np.sqrt(D)
        assert 0.05 < np.abs(t).max() < 2
        p = np.exp(t - t.max())
        p /= p.sum()
        want = p @ v
        blocks = np.abs(q[h].reshape(nb, bs).sum(-1) * ks[..., 1].astype(float)).sum(-1)
        terms = (blocks + (15 * s * np.abs(q[h])).sum(-1)) / np.sqrt(D)
        score = (D + 16) * 2.0 ** -23 * terms.max()
        weight = 2 * (score + (np.abs(t).max() + 64) * 2.0 ** -23 + 2.0 ** -22 + S / 8 * 2.0 ** -24)
        tol = (2.0 ** -11 + weight) * 2.0 + weight * (1 + np.abs(want)) + HALF_STEP[dtype] * np.abs(want)
        err = np.abs(f64(o)[0, h] - want)
        assert (err <= tol).all(), (h, float(err.max()), float(tol.min()))


def _one_hot(q, kq, ks, vq, vs, bs, dtype, gap):
    """O is the row of V whose score is the largest by `gap` relative to the scores' terms: exact up to
    p * scale's and O's rounding."""
    o = tqkv.decode_int4(q, kq, ks, vq, vs, bs)
    k, v = values(kq, ks, bs)[0, 0], values(vq, vs, bs)[0, 0]
    s, z = spread(ks, bs)
    for h in range(q.shape[1]):
        qh = f64(q)[0, h]
        t = k @ qh
        terms = ((15 * s + np.abs(z))[0, 0] @ np.abs(qh)).max()
        order = np.argsort(t)
        assert t[order[-1]] - t[order[-2]] > gap * terms, "the case does not hold what it is for"
        want = v[order[-1]]
        scaled = (unpack(vq) * spread(vs, bs)[0])[0, 0, order[-1]]
        tol = 2.0 ** -11 * scaled + (HALF_STEP[dtype] + 2.0 ** -20) * (np.abs(want) + scaled)
        err = np.abs(f64(o)[0, h] - want)
        assert (err <= tol).all(), (h, float(err.max()), f64(o)[0, h, :4])


def _keys(S, D, bs, seed, mul, peaks):
    """Keys of +-mul, of which the rows `peaks` follow one pattern each that the queries have too."""
    g = np.random.default_rng(seed)
    k = np.where(g.integers(0, 2, (S, D)), mul, -mul) * 0.5
    pattern = np.where(g.integers(0, 2, (len(peaks), D)), 1.0, -1.0)
    for i, r in enumerate(peaks):
        k[r] = pattern[i] * mul
    return tqkv.kv_compress_int4(torch.from_numpy(k)[None, None].half().cuda(), bs), pattern


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("qmul,kmul", [(3.0, 5.0), (1000, 1000), (30000, 300), (60000, 30000), (1e-3, 60000)])
@pytest.mark.parametrize("D,bs", VALID)
@pytest.mark.parametrize("S,peaks", [(90, [0, 17, 89, 40, 63]), (5000, [4999, 0, 2500, 64, 3000])])
def test_scores_far_beyond_the_weights_range(S, peaks, D, bs, qmul, kmul, dtype):
    """Scores up to 2^38 in one piece and in many that are joined, where a number in fp32 has steps far
    above 1: weights and sums stay finite, and the token with the largest score answers."""
    (kq, ks), pattern = _keys(S, D, bs, S + D + bs, kmul, peaks)
    g = torch.Generator(device="cuda").manual_seed(S)
    vq, vs = tqkv.kv_compress_int4(torch.randn((1, 1, S, D), generator=g, device="cuda").half(), bs)
    for G in (1, 5):
        q = torch.from_numpy(pattern[:G] * qmul * np.linspace(0.7, 1, D))[None].to(dtype).cuda()
        _one_hot(q, kq, ks, vq, vs, bs, dtype, 2.0 ** -7)
    o = tqkv.decode_int4(torch.from_numpy(pattern * qmul)[None].to(dtype).cuda().repeat(1, 3, 1)[:, :12].contiguous(),
                         kq, ks, vq, vs, bs)
    assert torch.isfinite(o).all()


@pytest.mark.parametrize("D,bs", VALID)
@pytest.mark.parametrize("qmul", [2.0 ** 90, 8e34, 1e38, 3.38e38])
@pytest.mark.parametrize("kmul", [1e-6, 1.0, 60000.0])
def test_bf16_queries_up_to_the_end_of_their_range(D, bs, qmul, kmul):
    S, peaks = 300, [3, 299, 128]
    (kq, ks), pattern = _keys(S, D, bs, D, kmul, peaks)
    g = torch.Generator(device="cuda").manual_seed(S)
    vq, vs = tqkv.kv_compress_int4(torch.randn((1, 1, S, D), generator=g, device="cuda").half(), bs)
    q = torch.from_numpy(pattern * qmul)[None].to(BF16).cuda()
    _one_hot(q, kq, ks, vq, vs, bs, BF16, 2.0 ** -7)


@pytest.mark.parametrize("D,bs", [(64, 32), (128, 128)])
@pytest.mark.parametrize("qmul,kmul", [(1.0, 1.0), (60000.0, 60000.0), (1e-30, 1.0), (3e38, 1.0), (3e38, 60000.0)])
def test_equal_scores_of_any_size_share_the_weight(D, bs, qmul, kmul):
    """All keys alike, in one piece and in many: O is the mean of V."""
    for S in (70, 4000):
        vq, vs, sign = _signs(S, D, bs, S)
        (kq, ks), pattern = _keys(S, D, bs, 1, kmul, [0])
        for t in (kq, ks):
            t[:, :, 1:] = t[:, :, :1]
        q = torch.from_numpy(pattern * qmul)[None].to(BF16).cuda()
        o = f64(tqkv.decode_int4(q, kq, ks, vq, vs, bs))[0, 0]
        want = values(vq, vs, bs)[0, 0].mean(0)
        # weights 2^x of equal x: each off by 2^-22 and the same 2^-11 of p * scale
        assert (np.abs(o - want) <= 2.0 ** -11 * 2 + 2.0 ** -8 * np.abs(want) + S * 2.0 ** -24).all()


def test_an_infinite_query_gives_nan_in_its_head_alone():
    D, bs, S = 128, 64, 200
    g = torch.Generator(device="cuda").manual_seed(1)
    cache = [t for _ in "kv" for t in
             tqkv.kv_compress_int4(torch.randn((1, 1, S, D), generator=g, device="cuda").half(), bs)]
    for dtype in (F16, BF16):
        q = torch.randn((1, 4, D), generator=g, device="cuda").to(dtype)
        o = tqkv.decode_int4(q, *cache, bs)
        for bad in (float("inf"), -float("inf"), float("nan")):
            r = q.clone()
            r[0, 2, 5] = bad
            again = tqkv.decode_int4(r, *cache, bs)
            assert torch.isnan(again[0, 2]).all()
            assert torch.equal(again[0, [0, 1, 3]], o[0, [0, 1, 3]])
