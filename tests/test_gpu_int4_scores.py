"""Scores of the 4-bit decode where they are hard to hold: keys with a large zero."""
import numpy as np
import pytest
import torch

import tqkv

from int4_reference import HALF_STEP, VALID, f64, pack, spread, values

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
