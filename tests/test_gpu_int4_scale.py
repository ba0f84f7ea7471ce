"""The scale of a 4-bit block is the correctly rounded (max - min) / 15."""
import numpy as np
import pytest
import torch

import tqkv

from int4_reference import VALID, unpack

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _check(x, bs, exact):
    """x [rows, D] of values that its type holds.  The range is one fp32 difference; its fifteenth, in 64
    bits here, is rounded once to fp16.  A code is the nearest integer to (x - zero) / scale: for
    `exact` (differences of few bits) always, else where none of the two fp32 roundings, of the
    difference and of the quotient over 16, crosses a half: 15 * 2^-24 and 16 * 2^-24."""
    codes, params = tqkv.kv_compress_int4(x[None, None].cuda(), bs)
    b = x.double().numpy().reshape(x.shape[0], -1, bs)
    lo, hi = b.min(-1), b.max(-1)
    zero = lo.astype(np.float16)
    scale = ((hi.astype(np.float32) - lo.astype(np.float32)).astype(np.float64) / 15).astype(np.float16)
    got = params[0, 0].cpu().numpy()
    assert np.array_equal(got[..., 0], scale)
    assert np.array_equal(got[..., 1], zero)
    s = scale.astype(np.float64)[..., None]
    ideal = np.clip(np.where(s == 0, 0, (b - zero.astype(np.float64)[..., None]) / np.where(s == 0, 1, s)), 0, 15)
    c = unpack(codes[0, 0]).reshape(b.shape).astype(np.float64)
    if exact:
        assert np.array_equal(c, np.rint(ideal))
    else:
        assert (np.abs(c - ideal) <= 0.5 + 31 * 2.0 ** -24).all()


@pytest.mark.parametrize("D,bs", VALID)
@pytest.mark.parametrize("e", [-12, -4, 0])
def test_ranges_whose_fifteenth_is_a_tie(D, bs, e):
    """Ranges 15 (2 m + 1) 2^e over all mantissas: the quotient lies exactly between two fp16 values
    and goes to the even one.  The largest element is the range's leading 11 bits, the smallest
    takes the rest off: both are exact in fp16."""
    m = np.arange(1024, 2048)
    rng = 15.0 * (2 * m + 1)
    hi = np.floor(rng / 32) * 32
    x = np.zeros((len(m), D))
    g = np.random.default_rng(bs)
    for b in range(D // bs):
        part = np.rint(g.random((len(m), bs)) * hi[:, None] / 64) * 64
        part = np.minimum(part, hi[:, None])
        part[:, 1], part[:, bs - 2] = hi, hi - rng
        x[:, b * bs:(b + 1) * bs] = part
    x = torch.from_numpy(x * 2.0 ** e).half()
    assert float(x.double().max()) < 65504 and float(x.double().min()) < 0
    _check(x, bs, True)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,bs", VALID)
def test_one_sided_blocks(D, bs, dtype):
    """Blocks between a small and a large positive number, whose range has more bits than either."""
    g = np.random.default_rng(D + bs)
    x = np.abs(g.standard_normal((4000, D)))
    _check(torch.from_numpy(x).to(dtype), bs, False)
    _check(torch.from_numpy(-x * 37).to(dtype), bs, False)


@pytest.mark.parametrize("bs", [32, 128])
def test_ranges_below_the_normal_numbers(bs):
    """bf16 holds ranges of n / 2 smallest fp16 steps: quotients at and around the middle between two
    of fp16's subnormal numbers."""
    n = np.arange(1, 512)
    x = np.zeros((len(n), 128))
    x[:, ::bs] = (n * 2.0 ** -25)[:, None]
    x = torch.from_numpy(x).bfloat16()
    _check(x, bs, False)
