"""The 4-bit KV cache's operators as they are measured: writing and reading back, decode attention over the cache, and
the head norms with the position rotation that come before it.

A case names an operator (`op`) and its sizes.  `run` computes it in plain torch operations, or, where `own` is true,
with this repository's kernels.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
BLOCKS = {64: (32, 64), 128: (32, 64, 128)}
EPS = 1e-6


def _tqkv():
    try:
        import tqkv
    except ImportError:
        sys.path.insert(0, os.path.join(os.getcwd(), "parallel-final-project_b200"))
        import tqkv
    return tqkv


# --------------------------------------------------------------------------
# Cases
# --------------------------------------------------------------------------
def listed():
    return [
        # the keys of four prompts of 4096 tokens, quantised as they enter the cache
        dict(name="write_prompt", op="write", B=4, H=8, T=4096, cap=4096, D=128, bs=64, dtype="bf16"),
        # one new token for each of 64 sequences, each at its own row of the cache
        dict(name="write_token", op="write", B=64, H=8, T=1, cap=2048, D=128, bs=128, dtype="fp16"),
        # a short cache of odd length, read back
        dict(name="read_short", op="read", B=2, H=8, T=257, cap=300, D=64, bs=32, dtype="fp16"),
        # a long context's keys, read back whole (this repository's long-context slice)
        dict(name="read_long", op="read", B=4, H=32, T=16384, cap=16384, D=128, bs=128, dtype="fp16"),
        # the smallest decode step of this repository's workloads: latency
        dict(name="decode_small", op="decode", B=1, Hq=4, Hkv=4, cap=128, ragged=False, D=64, bs=64, dtype="fp16"),
        # a served batch: 32 sequences of all lengths, four query heads to a key head
        dict(name="decode_served", op="decode", B=32, Hq=32, Hkv=8, cap=4099, ragged=True, D=128, bs=32, dtype="bf16"),
        # one user's long conversation: few heads, many tokens
        dict(name="decode_one_user", op="decode", B=1, Hq=32, Hkv=8, cap=32769, ragged=False, D=128, bs=64, dtype="bf16"),
        # this repository's long-context workload
        dict(name="decode_long", op="decode", B=4, Hq=32, Hkv=32, cap=131072, ragged=False, D=128, bs=128, dtype="fp16"),
        # q and k of one new token for each of 64 sequences
        dict(name="rotate_token", op="rotate", B=64, Hq=32, Hkv=8, T=1, axes=1, interleaved=False, D=128, dtype="bf16"),
        # q and k of two prompts with images: positions in time, height and width
        dict(name="rotate_image", op="rotate", B=2, Hq=32, Hkv=8, T=4097, axes=3, interleaved=False, D=128, dtype="bf16"),
        # norm, rotation and cache write of one new token for each of 32 sequences
        dict(name="step_token", op="step", B=32, Hq=32, Hkv=8, T=1, cap=1024, axes=1, interleaved=False, D=128, bs=32,
             dtype="bf16"),
        # norm, rotation and cache write of a prompt
        dict(name="step_prompt", op="step", B=1, Hq=32, Hkv=8, T=2049, cap=2049, axes=1, interleaved=True, D=64, bs=32,
             dtype="fp16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    D = rng.choice((64, 128))
    c = dict(op=rng.choice(("write", "read", "decode", "decode", "rotate", "step")), D=D, dtype=rng.choice(("fp16", "bf16")))
    if c["op"] != "rotate":
        c["bs"] = rng.choice(BLOCKS[D])
    if c["op"] in ("write", "read"):
        c.update(B=_log(rng, 1, 64), H=_log(rng, 1, 32), T=1)
        if rng.random() < 0.7:
            c["T"] = _log(rng, 2, max(3, min(16384, (1 << 21) // (c["B"] * c["H"]))))
        c["cap"] = c["T"] + _log(rng, 1, 1024) - 1
    elif c["op"] == "decode":
        Hkv = _log(rng, 1, 16)
        c.update(B=_log(rng, 1, 64), Hq=Hkv * rng.choice((1, 1, 2, 3, 4, 5, 8, 16)), Hkv=Hkv, ragged=rng.random() < 0.6)
        c["cap"] = _log(rng, 1, max(2, min(131072, (1 << 22) // (c["B"] * Hkv))))
    else:
        Hkv = _log(rng, 1, 8)
        c.update(B=_log(rng, 1, 64), Hq=Hkv * rng.choice((1, 2, 4, 8)), Hkv=Hkv, T=1, axes=rng.choice((1, 1, 3)),
                 interleaved=rng.random() < 0.4)
        if rng.random() < 0.6:
            most = (1 << 18) // (c["B"] * (c["Hq"] + Hkv)) if c["op"] == "rotate" else (1 << 14) // (c["B"] * Hkv)
            c["T"] = _log(rng, 2, max(3, most))
        if c["op"] == "step":
            c["cap"] = c["T"] + _log(rng, 1, 512) - 1
    return c


def _lengths(c):
    """How many tokens of its cache each sequence holds: part of the case, so that its work is known."""
    if not c["ragged"]:
        return [c["cap"]] * c["B"]
    r = random.Random(c["B"] * 1_000_003 + c["cap"])
    n = [r.randint(1, c["cap"]) for _ in range(c["B"])]
    if c["B"] > 3:
        n[r.randrange(c["B"])] = 0  # a slot of the batch that is idle
    return n


def _starts(c):
    r = random.Random(c["B"] * 7919 + c["cap"])
    return [r.randint(0, c["cap"] - c["T"]) for _ in range(c["B"])]


def _sections(c):
    P = c["D"] // 2
    return None if c["axes"] == 1 else (P // 4, P * 3 // 8, P - P // 4 - P * 3 // 8)


# --------------------------------------------------------------------------
# The 4-bit format in plain torch
# --------------------------------------------------------------------------
def _quantise(x, bs):
    """x [..., D] -> (codes uint8 [..., D], scales fp16 [..., D/bs, 2] = (scale, zero))."""
    x = x.float().unflatten(-1, (-1, bs))
    lo, hi = x.amin(-1), x.amax(-1)
    scale, zero = ((hi - lo) / 15).half(), lo.half()
    bad = ~(scale.isfinite() & zero.isfinite())
    scale, zero = (t.masked_fill(bad, math.nan) for t in (scale, zero))
    q = ((x - zero.float().unsqueeze(-1)) / scale.float().unsqueeze(-1)).round().clamp(0, 15)
    q = q.masked_fill((bad | (scale == 0)).unsqueeze(-1), 0)
    return q.to(torch.uint8).flatten(-2), torch.stack((scale, zero), -1)


def _pack(codes):
    """uint8 [..., D] in 0..15 -> packed rows uint8 [..., D/2]."""
    w = codes.unflatten(-1, (-1, 4, 4, 2)).transpose(-4, -3)  # [..., eighths, 32s, bytes, nibbles]
    return (w[..., 0] | (w[..., 1] << 4)).flatten(-3)


def _unpack(packed):
    w = packed.unflatten(-1, (4, -1, 4))
    return torch.stack((w & 15, w >> 4), -1).transpose(-4, -3).flatten(-4)


def _values(packed, scales, bs):
    """fp32 values of packed rows."""
    c = _unpack(packed).float().unflatten(-1, (-1, bs))
    s = scales.float()
    return (c * s[..., 0:1] + s[..., 1:2]).flatten(-2)


# --------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------
def _randn(seed, which, shape, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed * 1009 + which)
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _heads(seed, which, shape, dtype):
    """Keys or values [B, H, T, D]: N(0, 1) with each head's channels spread log-normally."""
    spread = torch.exp(0.5 * _randn(seed, which + 50, (shape[1], 1, shape[3]), torch.float32))
    return (_randn(seed, which, shape, torch.float32) * spread).to(dtype)


def _cache(seed, which, B, H, S, D, bs):
    codes, scales = _quantise(_heads(seed, which, (B, H, S, D), torch.float16), bs)
    return _pack(codes), scales


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _empty_cache(c):
    codes = torch.zeros((c["B"], c.get("H", c.get("Hkv")), c["cap"], c["D"] // 2), dtype=torch.uint8, device="cuda")
    return codes, torch.zeros((*codes.shape[:3], c["D"] // c["bs"], 2), dtype=torch.float16, device="cuda")


def prepare(case, seed):
    c, dt = case, DTYPES[case["dtype"]]
    s = dict(case=c)
    if c["op"] == "write":
        s.update(x=_heads(seed, 1, (c["B"], c["H"], c["T"], c["D"]), dt), starts=_ints(_starts(c)))
        s["kq"], s["ks"] = _empty_cache(c)
    elif c["op"] == "read":
        s["starts"] = _ints(_starts(c))
        s["kq"], s["ks"] = _cache(seed, 1, c["B"], c["H"], c["cap"], c["D"], c["bs"])
    elif c["op"] == "decode":
        s.update(q=_randn(seed, 3, (c["B"], c["Hq"], c["D"]), dt), lengths=_ints(_lengths(c)))
        s["kq"], s["ks"] = _cache(seed, 1, c["B"], c["Hkv"], c["cap"], c["D"], c["bs"])
        s["vq"], s["vs"] = _cache(seed, 2, c["B"], c["Hkv"], c["cap"], c["D"], c["bs"])
    else:
        B, T, D, Hq, Hkv, P = c["B"], c["T"], c["D"], c["Hq"], c["Hkv"], c["D"] // 2
        qkv = _randn(seed, 1, (B, T, Hq + 2 * Hkv, D), dt).transpose(1, 2)  # heads of one projection, as views
        s["q"], s["k"], s["v"] = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
        s["qw"], s["kw"] = (1 + 0.1 * _randn(seed, n, (D,), torch.float32).to(dt) for n in (2, 3))
        t = torch.arange(T, device="cuda", dtype=torch.int32)
        far = 8192  # rows of the table before the first token: the conversation so far
        off = torch.randint(0, far, (B, 1), generator=torch.Generator().manual_seed(seed), dtype=torch.int32).cuda()
        wide = max(1, int(math.sqrt(T)))
        s["positions"] = off + t if c["axes"] == 1 else torch.stack((off + 0 * t, off + t // wide, off + t % wide))
        angle = torch.arange(far + T, device="cuda", dtype=torch.float64)[:, None] * \
            10000.0 ** (-torch.arange(P, device="cuda", dtype=torch.float64) / P)
        s["table"] = torch.stack((angle.cos(), angle.sin()), -1).float()
        s["sections"] = _sections(c)
        if c["op"] == "step":
            s["starts"] = _ints(_starts(c))
            (s["kq"], s["ks"]), (s["vq"], s["vs"]) = _empty_cache(c), _empty_cache(c)
    return s


# --------------------------------------------------------------------------
# The operators
# --------------------------------------------------------------------------
def _at(s):
    """Index of the rows [start, start + T) of every sequence of a cache [B, H, cap, ...]."""
    c = s["case"]
    b = torch.arange(c["B"], device="cuda")[:, None, None]
    h = torch.arange(c.get("H", c.get("Hkv")), device="cuda")[None, :, None]
    return b, h, s["starts"].long()[:, None, None] + torch.arange(c["T"], device="cuda")


def _store(s, x, codes, scales):
    q, p = _quantise(x, s["case"]["bs"])
    codes[_at(s)], scales[_at(s)] = _pack(q), p


def _load(s, codes, scales):
    at = _at(s)
    return _values(codes[at], scales[at], s["case"]["bs"]).to(DTYPES[s["case"]["dtype"]])


def _norm_rotate(s, x, w):
    """fp32 [B, H, T, D]; the root mean square is taken in 64 bits, as the values go to the borders of 4-bit codes."""
    c, P = s["case"], s["case"]["D"] // 2
    inv = (x.double().square().mean(-1, keepdim=True) + EPS).rsqrt().float()
    y = x.float() * inv * w.float()
    pair = torch.arange(P, device="cuda")
    if s["sections"] is None:
        row = s["positions"].long()[..., None]
    else:
        axis = torch.bucketize(pair, torch.tensor(s["sections"], device="cuda").cumsum(0), right=True)
        row = s["positions"].long()[axis].permute(1, 2, 0)
    cos, sin = (s["table"][row, pair, i][:, None] for i in (0, 1))  # [B, 1, T, P]
    a, b = (y[..., 0::2], y[..., 1::2]) if c["interleaved"] else (y[..., :P], y[..., P:])
    out = (a * cos - b * sin, b * cos + a * sin)
    return torch.stack(out, -1).flatten(-2) if c["interleaved"] else torch.cat(out, -1)


def _attend(s):
    c, bs = s["case"], s["case"]["bs"]
    q = s["q"].float().unflatten(1, (c["Hkv"], -1))
    score = q @ _values(s["kq"], s["ks"], bs).transpose(-1, -2) / math.sqrt(c["D"])
    n = s["lengths"].view(-1, 1, 1, 1)
    score = score.masked_fill(torch.arange(c["cap"], device="cuda") >= n, -math.inf)
    p = (score - score.amax(-1, keepdim=True)).exp()
    o = (p / p.sum(-1, keepdim=True)) @ _values(s["vq"], s["vs"], bs)
    return o.masked_fill(n == 0, 0).flatten(1, 2).to(s["q"].dtype)


def run(s):
    c, op = s["case"], s["case"]["op"]
    dt = DTYPES[c["dtype"]]
    if own:
        t = _tqkv()
        if op == "write":
            t.kv_append_int4(s["x"], s["kq"], s["ks"], s["starts"], c["bs"])
            return t.kv_reconstruct_int4(s["kq"], s["ks"], c["bs"], t0=s["starts"], T=c["T"], dtype=dt)
        if op == "read":
            return t.kv_reconstruct_int4(s["kq"], s["ks"], c["bs"], t0=s["starts"], T=c["T"], dtype=dt)
        if op == "decode":
            return t.decode_int4(s["q"], s["kq"], s["ks"], s["vq"], s["vs"], c["bs"], lengths=s["lengths"])
        how = dict(q_weight=s["qw"], k_weight=s["kw"], eps=EPS, interleaved=c["interleaved"], sections=s["sections"])
        if op == "rotate":
            return t.qk_norm_rope(s["q"], s["k"], s["positions"], s["table"], **how)
        q = t.qk_norm_rope_append_int4(s["q"], s["k"], s["v"], s["positions"], s["table"], s["kq"], s["ks"], s["vq"],
                                       s["vs"], s["starts"], c["bs"], **how)
        return [q] + [t.kv_reconstruct_int4(s[a], s[b], c["bs"], t0=s["starts"], T=c["T"], dtype=dt)
                      for a, b in (("kq", "ks"), ("vq", "vs"))]
    if op == "write":
        _store(s, s["x"], s["kq"], s["ks"])
        return _load(s, s["kq"], s["ks"])
    if op == "read":
        return _load(s, s["kq"], s["ks"])
    if op == "decode":
        return _attend(s)
    q, k = _norm_rotate(s, s["q"], s["qw"]), _norm_rotate(s, s["k"], s["kw"])
    if op == "rotate":
        return q.to(dt), k.to(dt)
    _store(s, k, s["kq"], s["ks"])
    _store(s, s["v"], s["vq"], s["vs"])
    return [q.to(dt), _load(s, s["kq"], s["ks"]), _load(s, s["vq"], s["vs"])]


def work(case):
    c = case
    D, op = c["D"], c["op"]
    if op in ("write", "read"):
        n = c["B"] * c["H"] * c["T"]
        cache = D // 2 + 4 * (D // c["bs"])
        return {"bytes": n * (cache + 2 * D * (2 if op == "write" else 1)), "flops": 6.0 * n * D}
    if op == "decode":
        tokens = sum(_lengths(c))
        row = D // 2 + 4 * (D // c["bs"])
        return {"bytes": 2 * tokens * c["Hkv"] * row + 4 * c["B"] * c["Hq"] * D, "flops": 4.0 * tokens * c["Hq"] * D}
    n = c["B"] * c["T"]
    bytes_, heads = 4 * n * D * c["Hq"] + 4 * n * D + 4 * n * c["axes"], c["Hq"] + c["Hkv"]
    if op == "rotate":
        bytes_ += 4 * n * D * c["Hkv"]
    else:
        bytes_ += 2 * n * c["Hkv"] * (4 * D + D // 2 + 4 * (D // c["bs"]))
        heads += 2 * c["Hkv"]
    return {"bytes": bytes_, "flops": 8.0 * n * heads * D}


# --------------------------------------------------------------------------
# The operators' definitions in 64 bits
# --------------------------------------------------------------------------
def _exact_codes(x, bs):
    """Each element's value after the cache, of x float64 [..., D]: the definition, block by block."""
    out = torch.empty_like(x)
    for j in range(x.shape[-1] // bs):
        b = x[..., j * bs:(j + 1) * bs]
        zero = b.min(-1, keepdim=True).values.half().double()
        scale = ((b.max(-1, keepdim=True).values - b.min(-1, keepdim=True).values) / 15).half().double()
        step = torch.where(scale > 0, scale, torch.ones_like(scale))
        code = torch.where(scale > 0, torch.round((b - zero) / step), torch.zeros_like(b))
        out[..., j * bs:(j + 1) * bs] = torch.clamp(code, 0, 15) * scale + zero
    return out


def _exact_read(packed, scales, bs):
    """Values in 64 bits, element by element: where each one's nibble stands, and its block's parameters."""
    D = 2 * packed.shape[-1]
    i = torch.arange(D, device=packed.device)
    byte = ((i % 32 // 8) * (D // 32) + i // 32) * 4 + i % 8 // 2
    code = (packed[..., byte].to(torch.int16) >> (4 * (i % 2)).to(torch.int16)) & 15
    p = scales.double()[..., i // bs, :]
    return code.double() * p[..., 0] + p[..., 1]


def _exact_rotate(s, x, w):
    D = x.shape[-1]
    x = x.double()
    y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + EPS) * w.double()
    out = torch.empty_like(y)
    pos, sec = s["positions"], s["sections"]
    for j in range(D // 2):
        if sec is None:
            p = pos
        else:
            p = pos[0] if j < sec[0] else pos[1] if j < sec[0] + sec[1] else pos[2]
        cos, sin = (s["table"][p.long(), j, i].double()[:, None] for i in (0, 1))
        m, n = (2 * j, 2 * j + 1) if s["case"]["interleaved"] else (j, j + D // 2)
        out[..., m] = y[..., m] * cos - y[..., n] * sin
        out[..., n] = y[..., n] * cos + y[..., m] * sin
    return out


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] == "write":
        return _exact_codes(s["x"].double(), c["bs"])
    if c["op"] == "read":
        return torch.stack([_exact_read(s["kq"][b, :, t:t + c["T"]], s["ks"][b, :, t:t + c["T"]], c["bs"])
                            for b, t in enumerate(_starts(c))])
    if c["op"] == "decode":
        out = torch.zeros((c["B"], c["Hq"], c["D"]), dtype=torch.float64, device="cuda")
        for b, n in enumerate(_lengths(c)):
            if n == 0:
                continue
            k, v = (_exact_read(s[x][b, :, :n], s[y][b, :, :n], c["bs"]) for x, y in (("kq", "ks"), ("vq", "vs")))
            q = s["q"][b].double().view(c["Hkv"], -1, c["D"])
            p = torch.softmax(torch.einsum("hgd,htd->hgt", q, k) / c["D"] ** 0.5, -1)
            out[b] = torch.einsum("hgt,htd->hgd", p, v).reshape(c["Hq"], c["D"])
        return out
    q, k = _exact_rotate(s, s["q"], s["qw"]), _exact_rotate(s, s["k"], s["kw"])
    return (q, k) if c["op"] == "rotate" else [q, _exact_codes(k, c["bs"]), _exact_codes(s["v"].double(), c["bs"])]
