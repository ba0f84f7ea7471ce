"""The 4-bit cache as it is written and read back (tqkv_kv_append_int4, tqkv_kv_compress_int4,
tqkv_kv_reconstruct_int4), against the format's definition in float64."""
import numpy as np
import pytest
import torch

import tqkv

from int4_reference import HALF_STEP, TINY, VALID, f64, pack, quantise, unpack, values

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _rand(shape, seed, dtype=F16, mul=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * mul).to(dtype)


def _check_written(x, codes, scales, bs):
    """Codes and parameters are the definition's: quotients of 16-bit inputs that are half-integers
    are exactly so, and no others come within the kernel's 2^-45 of one."""
    want_c, want_s = quantise(f64(x), bs)
    got_s = scales.cpu().numpy()
    assert np.array_equal(np.isnan(got_s), np.isnan(want_s))
    ok = ~np.isnan(want_s)
    assert np.array_equal(got_s[ok], want_s[ok])
    assert np.array_equal(codes.cpu().numpy(), pack(want_c))


def _check_read(y, codes, scales, bs):
    want, got = values(codes, scales, bs), f64(y)
    nan = np.isnan(want)
    assert np.array_equal(nan, np.isnan(got))
    u = HALF_STEP[y.dtype]
    # one rounding (bf16: one to fp32 before it)
    err = np.abs(got - want)[~nan]
    lim = (u + 2.0 ** -23) * np.abs(want[~nan]) + TINY[y.dtype]
    assert (err <= lim).all(), float((err - lim).max())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,bs", VALID)
@pytest.mark.parametrize("B,H,S", [(1, 1, 1), (2, 3, 17), (1, 2, 257), (5, 1, 64)])
def test_compress_and_reconstruct(B, H, S, D, bs, dtype):
    x = _rand((B, H, S, D), S + D + bs, dtype)
    codes, scales = tqkv.kv_compress_int4(x, bs)
    _check_written(x, codes, scales, bs)
    for out in (F16, BF16):
        _check_read(tqkv.kv_reconstruct_int4(codes, scales, bs, dtype=out), codes, scales, bs)


@pytest.mark.parametrize("D,bs", VALID)
def test_ties_round_to_even(D, bs):
    """Multiples of half a step: every second quotient is exactly a half-integer."""
    B, H, S = 1, 1, 64
    x = torch.zeros((S, D))
    for t in range(S):
        step = float(np.float16((1 + t / 64) * 2.0 ** (t % 9 - 4)))
        n = torch.randint(0, 31, (D,), generator=torch.Generator().manual_seed(t)).float()
        n[::bs], n[1::bs] = 0, 30
        x[t] = n * (step / 2) - step * (t % 5)
    x = x.half().view(B, H, S, D).cuda()
    codes, scales = tqkv.kv_compress_int4(x, bs)
    _check_written(x, codes, scales, bs)
    c, s = quantise(f64(x), bs)
    q = (f64(x).reshape(S, -1, bs) - s[..., 1].reshape(S, -1, 1).astype(float)) / \
        s[..., 0].reshape(S, -1, 1).astype(float)
    assert (np.abs(q % 1 - 0.5) == 0).mean() > 0.05   # the case holds what it is for


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,bs", VALID)
def test_every_magnitude_and_constant_blocks(D, bs, dtype):
    mags = [0.0, 1e-7, 6e-6, 1e-4, 1.0, 300.0, 1e4, 6e4]
    x = torch.cat([_rand((1, 2, 3, D), i, torch.float32).clamp(-1, 1) * m
                   for i, m in enumerate(mags)], 2).to(dtype)
    x[0, 1, :, :] = x[0, 1, :, :1]          # every element of the row the same
    codes, scales = tqkv.kv_compress_int4(x, bs)
    _check_written(x, codes, scales, bs)
    y = tqkv.kv_reconstruct_int4(codes, scales, bs, dtype=dtype)
    _check_read(y, codes, scales, bs)
    assert torch.equal(y[0, 1].float(), x[0, 1].half().float().to(dtype).float())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), 1e5])
def test_blocks_that_fp16_cannot_hold_read_as_nan(bad, dtype):
    D, bs = 128, 32
    x = _rand((1, 1, 4, D), 3, dtype)
    x[0, 0, 1, 40] = bad          # fp16: 1e5 is an infinity already
    x[0, 0, 2, :32] = bad
    codes, scales = tqkv.kv_compress_int4(x, bs)
    y = f64(tqkv.kv_reconstruct_int4(codes, scales, bs)).reshape(4, 4, 32)
    want = np.zeros((4, 4), bool)
    want[2, 0] = True
    # one value of 1e5 above others: the range fits fp16, and so does its zero
    want[1, 1] = not (dtype == BF16 and bad == 1e5)
    assert np.array_equal(np.isnan(y).all(-1), want) and np.array_equal(np.isnan(y).any(-1), want)
    assert not unpack(codes).reshape(4, 4, 32)[want].any()
    _check_written(x, codes, scales, bs)


@pytest.mark.parametrize("D,bs", [(128, 128), (128, 32), (64, 64)])
@pytest.mark.parametrize("T,t0,S_cap", [(1, 0, 1), (1, 99, 100), (7, 13, 64), (300, 5, 2048)])
def test_append_leaves_other_rows(D, bs, T, t0, S_cap):
    B, H = 2, 3
    x = _rand((B, H, T, D), T + t0)
    codes = torch.full((B, H, S_cap, D // 2), 0xA5, dtype=torch.uint8, device="cuda")
    scales = torch.full((B, H, S_cap, D // bs, 2), 7.0, dtype=F16, device="cuda")
    tqkv.kv_append_int4(x, codes, scales, t0, bs)
    _check_written(x, codes[:, :, t0:t0 + T], scales[:, :, t0:t0 + T], bs)
    rest = torch.ones(S_cap, dtype=torch.bool, device="cuda")
    rest[t0:t0 + T] = False
    assert bool((codes[:, :, rest] == 0xA5).all()) and bool((scales[:, :, rest] == 7.0).all())
    y = tqkv.kv_reconstruct_int4(codes, scales, bs, t0=t0, T=T)
    assert torch.equal(y, tqkv.kv_reconstruct_int4(codes, scales, bs)[:, :, t0:t0 + T])


def test_starts_of_each_sequence_and_rows_outside():
    """Rows that a sequence's start puts outside the cache are not written and read as zero."""
    B, H, T, S_cap, D, bs = 6, 2, 3, 10, 64, 32
    x = _rand((B, H, T, D), 1)
    first = [0, 7, 8, -2, 10, -2147483648]
    starts = torch.tensor(first, dtype=torch.int32, device="cuda")
    codes = torch.full((B, H, S_cap, D // 2), 0x5A, dtype=torch.uint8, device="cuda")
    scales = torch.full((B, H, S_cap, D // bs, 2), 3.0, dtype=F16, device="cuda")
    tqkv.kv_append_int4(x, codes, scales, starts, bs)
    y = tqkv.kv_reconstruct_int4(codes, scales, bs, t0=starts, T=T)
    ref_c, ref_s = tqkv.kv_compress_int4(x, bs)
    ref_y = tqkv.kv_reconstruct_int4(ref_c, ref_s, bs)
    for b, f in enumerate(first):
        written = set()
        for t in range(T):
            if 0 <= f + t < S_cap:
                written.add(f + t)
                assert torch.equal(codes[b, :, f + t], ref_c[b, :, t])
                assert torch.equal(scales[b, :, f + t], ref_s[b, :, t])
                assert torch.equal(y[b, :, t], ref_y[b, :, t])
            else:
                assert not y[b, :, t].any()
        for r in set(range(S_cap)) - written:
            assert bool((codes[b, :, r] == 0x5A).all()) and bool((scales[b, :, r] == 3.0).all())


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_strided_inputs(dtype):
    """Values as a slice of a fused projection, and other orders of the dimensions."""
    B, H, T, D, bs = 3, 2, 5, 128, 64
    qkv = _rand((B, T, 8, D), 5, dtype)
    x = qkv.transpose(1, 2)[:, 3:3 + H]
    want_c, want_s = tqkv.kv_compress_int4(x.contiguous(), bs)
    for view in (x, x.permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3), x[:, :1].expand(B, H, T, D)):
        c, s = tqkv.kv_compress_int4(view, bs)
        ref_c, ref_s = tqkv.kv_compress_int4(view.contiguous(), bs)
        assert torch.equal(c, ref_c) and torch.equal(s, ref_s)
    assert torch.equal(tqkv.kv_compress_int4(x, bs)[0], want_c)
    wide = _rand((B, H, T, D + 8), 6, dtype)[..., :D]      # rows further apart than D
    c, s = tqkv.kv_compress_int4(wide, bs)
    ref_c, ref_s = tqkv.kv_compress_int4(wide.contiguous(), bs)
    assert torch.equal(c, ref_c) and torch.equal(s, ref_s) and want_s.isfinite().all()


def test_offsets_past_32_bits():
    """A cache of more than 2^32 bytes of codes: the last rows of its last head."""
    D, bs, S_cap = 128, 128, 1 << 25
    codes = torch.empty((1, 3, S_cap, D // 2), dtype=torch.uint8, device="cuda")
    scales = torch.empty((1, 3, S_cap, 1, 2), dtype=F16, device="cuda")
    x = _rand((1, 3, 5, D), 9)
    t0 = S_cap - 5
    assert (2 * S_cap + t0) * (D // 2) > 2 ** 32
    tqkv.kv_append_int4(x, codes, scales, t0, bs)
    c, s = tqkv.kv_compress_int4(x, bs)
    assert torch.equal(codes[:, :, t0:], c) and torch.equal(scales[:, :, t0:], s)
    assert torch.equal(tqkv.kv_reconstruct_int4(codes, scales, bs, t0=t0, T=5),
                       tqkv.kv_reconstruct_int4(c, s, bs))
