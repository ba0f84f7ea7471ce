"""The 4-bit KV cache's operators in numpy float64, from their definitions, with the error bounds
that the kernels' roundings allow.

Half a step of rounding, relative to the value: fp16 2^-11, bf16 2^-8, fp32 2^-24.
"""
import numpy as np
import torch

VALID = [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)]
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# half the smallest step of a type: what rounding loses below its normal range
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}


def f64(t: torch.Tensor) -> np.ndarray:
    return t.detach().cpu().double().numpy()


def element_places(D):
    """(byte, shift) of every element in a packed row."""
    i = np.arange(D)
    word = (i % 32) // 8 * (D // 32) + i // 32
    return 4 * word + (i % 8) // 2, 4 * (i % 2)


def unpack(codes) -> np.ndarray:
    """uint8 [..., D/2] -> codes [..., D]."""
    c = codes.cpu().numpy() if isinstance(codes, torch.Tensor) else codes
    byte, shift = element_places(2 * c.shape[-1])
    return (c[..., byte] >> shift.astype(np.uint8)) & 15


def pack(codes: np.ndarray) -> np.ndarray:
    """codes [..., D] -> uint8 [..., D/2]."""
    D = codes.shape[-1]
    byte, shift = element_places(D)
    out = np.zeros(codes.shape[:-1] + (D // 2,), dtype=np.uint8)
    for i in range(D):
        out[..., byte[i]] |= (codes[..., i].astype(np.uint8) << shift[i]).astype(np.uint8)
    return out


def spread(scales, bs):
    """(scale, zero) of every element, float64 [..., D], from [..., D/bs, 2]."""
    s = f64(scales) if isinstance(scales, torch.Tensor) else np.asarray(scales, np.float64)
    return np.repeat(s[..., 0], bs, -1), np.repeat(s[..., 1], bs, -1)


def values(codes, scales, bs) -> np.ndarray:
    s, z = spread(scales, bs)
    return unpack(codes) * s + z


def quantise(x: np.ndarray, bs):
    """float64 x [..., D] -> (codes [..., D], scales float16 [..., D/bs, 2])."""
    b = x.reshape(x.shape[:-1] + (-1, bs))
    with np.errstate(all="ignore"):
        lo, hi = b.min(-1), b.max(-1)
        zero = lo.astype(np.float16)
        rng = hi.astype(np.float32) - lo.astype(np.float32)
        scale = (rng * (np.float32(1) / np.float32(15))).astype(np.float16)
        bad = ~(np.isfinite(zero) & np.isfinite(scale))
        zero[bad], scale[bad] = np.nan, np.nan
        s = np.where(bad | (scale == 0), 1, scale).astype(np.float64)
        q = np.rint((b - zero[..., None].astype(np.float64)) / s[..., None])
        q = np.where((bad | (scale == 0))[..., None], 0, q)
    return np.clip(q, 0, 15).astype(np.uint8).reshape(x.shape), np.stack((scale, zero), -1)


def check_quantised(x: np.ndarray, codes, scales, bs, slack):
    """The cache rows of x (float64, exact to `slack` relative to its block's largest): zero and
    scale are the block's rounded to fp16, and every code is the nearest one to its element."""
    b = x.reshape(x.shape[:-1] + (-1, bs))
    lo, hi = b.min(-1), b.max(-1)
    big = np.maximum(np.abs(lo), np.abs(hi))
    s, z = f64(scales)[..., 0], f64(scales)[..., 1]
    assert (np.abs(z - lo) <= 2.0 ** -11 * np.abs(lo) + 2.0 ** -25 + 2 * slack * big).all()
    want = (hi - lo) / 15
    # roundings of the difference, of 1 / 15 and of the product, and one to fp16
    assert (np.abs(s - want) <= (2.0 ** -11 + 2.0 ** -22) * want + 2.0 ** -25 + slack * big).all()
    got = unpack(codes).reshape(b.shape).astype(np.float64)
    sz = s[..., None]
    ideal = np.clip((b - z[..., None]) / np.where(sz == 0, 1, sz), 0, 15)
    # half a code, the quotient's own rounding, and what x may be off
    allowed = 0.5 + 16 * 2.0 ** -22 + (2 * slack * big)[..., None] / np.where(sz == 0, 1, sz)
    off = np.abs(got - np.where(sz == 0, 0, ideal))
    assert (off <= np.where(sz == 0, 0, allowed)).all(), float(off.max())


def attention(q, kq, ks, vq, vs, bs, lengths):
    """float64 (O [B, Hq, D], bound on |error| before the output's rounding) over the first
    lengths[b] rows; numpy views of the caches, rows behind the lengths are not looked at."""
    q = f64(q)
    B, Hq, D = q.shape
    Hkv = kq.shape[1]
    G = Hq // Hkv
    o, tol = np.zeros_like(q), np.zeros_like(q)
    for b in range(B):
        n = int(lengths[b])
        if n == 0:
            continue
        k = values(kq[b, :, :n], ks[b, :, :n], bs)
        vc = unpack(vq[b, :, :n])
        s, z = spread(vs[b, :, :n], bs)
        for h in range(Hq):
            kv = h // G
            t = k[kv] @ q[b, h] / np.sqrt(D)
            p = np.exp(t - t.max())
            p /= p.sum()
            scaled, zero = vc[kv] * s[kv], z[kv]
            o[b, h] = p @ (scaled + zero)
            # a score: D products and 2 D / bs + 4 more operations in fp32, whose sums a tensor core
            # may truncate (2^-23); its terms are codes * scale * q and zero * q, and q itself is
            # kept to 2^-24 of its head's largest element
            ksc, kz = spread(ks[b, kv, :n], bs)
            terms = (15 * ksc + np.abs(kz)) @ np.abs(q[b, h]) / np.sqrt(D)
            terms += (15 * ksc + np.abs(kz)).sum(-1) * np.abs(q[b, h]).max() / np.sqrt(D)
            score = (D + 16) * 2.0 ** -23 * terms.max()
            # its argument of 2^x: one rounding of up to |score| + 64; 2^x itself 2^-22; sums of p
            weight = 2 * (score + (np.abs(t).max() + 64) * 2.0 ** -23 + 2.0 ** -22 + n / 8 * 2.0 ** -24)
            # the product's operand p * scale in fp16: half a step, or 2^-35 of the largest one
            tol[b, h] = (2.0 ** -11 + weight) * (p @ scaled) + weight * (p @ np.abs(zero)) + \
                weight * np.abs(o[b, h]) + n * 15 * s[kv].max() * 2.0 ** -34
    return o, tol


def check_attention(out, q, kq, ks, vq, vs, bs, lengths):
    want, tol = attention(q, kq.cpu().numpy(), ks.float().cpu().numpy(), vq.cpu().numpy(),
                          vs.float().cpu().numpy(), bs, lengths)
    got, u = f64(out), HALF_STEP[out.dtype]
    bad = ~(np.abs(got - want) <= tol * (1 + u) + u * np.abs(want) + TINY[out.dtype])
    assert not bad.any(), (int(bad.sum()), float(np.abs(got - want)[bad].max()),
                           np.argwhere(bad)[:3].tolist())


def norm_rope(x, w, cos, sin, eps, interleaved, exact=False):
    """float64 x [B, H, T, D], cos and sin [B, 1, T, pairs] -> (out, bound before rounding);
    `exact`: the root mean square is correct to fp32, as where the values go to a cache."""
    D, P = x.shape[-1], cos.shape[-1]
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    if w is not None:
        y = y * w
    out, mag = y.copy(), np.abs(y)
    ia = np.arange(P) * 2 if interleaved else np.arange(P)
    ib = ia + 1 if interleaved else ia + P
    a, b = y[..., ia], y[..., ib]
    out[..., ia], out[..., ib] = a * cos - b * sin, b * cos + a * sin
    mag[..., ia] = np.abs(a * cos) + np.abs(b * sin)
    mag[..., ib] = np.abs(b * cos) + np.abs(a * sin)
    # 1/rms, times x, times w, times cos or sin, the sum: five roundings to fp32.  A sum of squares in
    # fp32 passes at most 8 FMAs, 1 and 3 sums, of positive terms: 12 roundings, of which the root
    # keeps half, and eps one, of which it keeps half
    return out, (5.1 if exact else 5.1 + 6 + 0.5 + 0.5) * 2.0 ** -24 * mag
