"""Head norms with the position rotation (tqkv_qk_norm_rope), the same into the 4-bit cache
(tqkv_qk_norm_rope_append_int4), and a run of all the 4-bit operators together."""
import math

import numpy as np
import pytest
import torch

import tqkv

from int4_reference import (HALF_STEP, TINY, VALID, check_attention, check_quantised, f64, norm_rope,
                            unpack)

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _rand(shape, seed, dtype=F16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _positions(B, T, axes, max_pos, seed):
    g = torch.Generator().manual_seed(seed)
    shape = (B, T) if axes == 1 else (axes, B, T)
    return torch.randint(0, max_pos, shape, generator=g, dtype=torch.int32).cuda()


def _sections(pairs, axes):
    if axes == 1:
        return None
    s = [pairs // axes + (i % 2) for i in range(axes - 1)]
    return tuple(s + [pairs - sum(s)])


def _cos_sin(table, positions, sections):
    """float64 [B, 1, T, pairs] each."""
    t, pos = f64(table), positions.cpu().numpy()
    pairs = np.arange(t.shape[1])
    if sections is None:
        row = pos[..., None]
    else:
        axis = np.searchsorted(np.cumsum(sections), pairs, side="right")
        row = np.moveaxis(pos[axis], 0, -1)
    cs = t[row, pairs]
    return cs[..., 0][:, None], cs[..., 1][:, None]


def _check(out, x, w, cos, sin, eps, interleaved, exact=False):
    want, tol = norm_rope(f64(x), None if w is None else f64(w), cos, sin, eps, interleaved, exact)
    u = HALF_STEP[out.dtype]
    err = np.abs(f64(out) - want)
    lim = tol * (1 + u) + u * np.abs(want) + TINY[out.dtype]
    assert (err <= lim).all(), float((err - lim).max())
    return want


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,rot", [(64, 64), (64, 16), (128, 128), (128, 96), (128, 32)])
@pytest.mark.parametrize("B,Hq,Hkv,T,axes", [(1, 1, 1, 1, 1), (3, 5, 1, 7, 1), (2, 8, 2, 33, 3),
                                             (1, 3, 3, 130, 2), (2, 4, 4, 9, 4)])
def test_norm_rope(B, Hq, Hkv, T, axes, D, rot, interleaved, dtype):
    max_pos = 5000
    q, k = _rand((B, Hq, T, D), 1, dtype), _rand((B, Hkv, T, D), 2, dtype) * 3
    qw, kw = _rand((D,), 3, dtype), _rand((D,), 4, dtype)
    table = tqkv.rope_table(max_pos, rot)
    sections = _sections(rot // 2, axes)
    pos = _positions(B, T, axes, max_pos, T)
    cos, sin = _cos_sin(table, pos, sections)
    for a, b in ((qw, kw), (None, None)):
        qo, ko = tqkv.qk_norm_rope(q, k, pos, table, a, b, eps=1e-5, interleaved=interleaved,
                                   sections=sections)
        _check(qo, q, a, cos, sin, 1e-5, interleaved)
        _check(ko, k, b, cos, sin, 1e-5, interleaved)


@pytest.mark.parametrize("Hq,Hkv,T", [(32, 8, 700), (7, 7, 1500), (9, 1, 2000)])
def test_many_rows(Hq, Hkv, T):
    """Enough rows that a lane group takes several heads, and head counts that do not divide."""
    B, D = 2, 128
    q, k = _rand((B, Hq, T, D), 1, BF16), _rand((B, Hkv, T, D), 2, BF16)
    table, pos = tqkv.rope_table(T, D), _positions(B, T, 1, T, 3)
    cos, sin = _cos_sin(table, pos, None)
    qo, ko = tqkv.qk_norm_rope(q, k, pos, table)
    _check(qo, q, None, cos, sin, 1e-6, False)
    _check(ko, k, None, cos, sin, 1e-6, False)


def test_rope_table_angles():
    t = f64(tqkv.rope_table(70000, 128, base=500000.0))
    p = np.arange(70000, dtype=np.float64)[:, None] * 500000.0 ** (-np.arange(64) / 64)
    assert np.abs(t[..., 0] - np.cos(p)).max() <= 2.0 ** -25 + 1e-10
    assert np.abs(t[..., 1] - np.sin(p)).max() <= 2.0 ** -25 + 1e-10


def test_zero_rows_and_large_values():
    q = torch.zeros((1, 2, 3, 128), dtype=BF16, device="cuda")
    q[0, 1] = 3e38
    k = torch.full((1, 1, 3, 128), 1e-30, dtype=BF16, device="cuda")
    table, pos = tqkv.rope_table(8, 128), _positions(1, 3, 1, 8, 0)
    cos, sin = _cos_sin(table, pos, None)
    qo, ko = tqkv.qk_norm_rope(q, k, pos, table)
    _check(qo, q, None, cos, sin, 1e-6, False)
    _check(ko, k, None, cos, sin, 1e-6, False)
    qo, _ = tqkv.qk_norm_rope(q, k, pos, table, eps=0.0)
    assert torch.isnan(qo[0, 0]).all() and not torch.isnan(qo[0, 1]).any()   # 0 / 0


def test_positions_outside_the_table_leave_nan():
    B, H, T, D, rot = 1, 2, 6, 128, 64
    q, k = _rand((B, H, T, D), 1), _rand((B, H, T, D), 2)
    pos = torch.tensor([[0, -1, 9, 10, 2 ** 31 - 1, -2 ** 31]], dtype=torch.int32, device="cuda")
    qo, ko = tqkv.qk_norm_rope(q, k, pos, tqkv.rope_table(10, rot))
    nan = torch.tensor([False, True, False, True, True, True], device="cuda")
    for o in (qo, ko):
        assert torch.equal(torch.isnan(o[..., :rot]).all(-1), nan.expand(B, H, T))
        assert not torch.isnan(o[..., rot:]).any() and not torch.isnan(o[:, :, ~nan]).any()


@pytest.mark.parametrize("interleaved", [False, True])
def test_strided_inputs_and_given_outputs(interleaved):
    B, Hq, Hkv, T, D = 2, 4, 2, 5, 64
    qkv = _rand((B, T, Hq + 2 * Hkv, D), 1, BF16).transpose(1, 2)
    q, k = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv]
    table, pos = tqkv.rope_table(50, D), _positions(B, T, 1, 50, 2)
    want = tqkv.qk_norm_rope(q.contiguous(), k.contiguous(), pos, table, interleaved=interleaved)
    got = tqkv.qk_norm_rope(q, k, pos, table, interleaved=interleaved,
                            q_out=torch.empty_like(want[0]), k_out=torch.empty_like(want[1]))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # one key head for all: a broadcast view
    one = k[:, :1].expand(B, Hkv, T, D)
    a = tqkv.qk_norm_rope(q, one, pos, table, interleaved=interleaved)[1]
    assert torch.equal(a, want[1][:, :1].expand_as(a))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,bs", VALID)
@pytest.mark.parametrize("B,Hq,Hkv,T,axes,interleaved", [(1, 1, 1, 1, 1, False), (3, 6, 2, 5, 3, True),
                                                         (2, 8, 1, 40, 1, False)])
def test_append(B, Hq, Hkv, T, axes, interleaved, D, bs, dtype):
    S_cap = T + 9
    q, k, v = (_rand((B, h, T, D), i, dtype) for i, h in enumerate((Hq, Hkv, Hkv)))
    qw, kw = _rand((D,), 3, dtype), _rand((D,), 4, dtype)
    table = tqkv.rope_table(300, D)
    sections = _sections(D // 2, axes)
    pos = _positions(B, T, axes, 300, T)
    cos, sin = _cos_sin(table, pos, sections)
    first = [4 + (b % 3) for b in range(B)]
    starts = torch.tensor(first, dtype=torch.int32, device="cuda")
    kq, vq = (torch.full((B, Hkv, S_cap, D // 2), 0xC3, dtype=torch.uint8, device="cuda") for _ in "kv")
    ks, vs = (torch.full((B, Hkv, S_cap, D // bs, 2), 5.0, dtype=F16, device="cuda") for _ in "kv")
    qo = tqkv.qk_norm_rope_append_int4(q, k, v, pos, table, kq, ks, vq, vs, starts, bs, q_weight=qw,
                                       k_weight=kw, interleaved=interleaved, sections=sections)
    _check(qo, q, qw, cos, sin, 1e-6, interleaved, exact=True)
    want_k, tol = norm_rope(f64(k), f64(kw), cos, sin, 1e-6, interleaved, exact=True)
    ref_c, ref_s = tqkv.kv_compress_int4(v, bs)
    for b, f in enumerate(first):
        rows = slice(f, f + T)
        # a rotated pair's sum is exact to 5.1 roundings of at most sqrt(2) of its block's largest
        # norm; 2^-20 of the largest element covers pairs that lie in two blocks
        check_quantised(want_k[b], kq[b, :, rows], ks[b, :, rows], bs,
                        slack=float((tol[b] / np.abs(want_k[b]).max(-1, keepdims=True)).max()) * 4)
        assert torch.equal(vq[b, :, rows], ref_c[b]) and torch.equal(vs[b, :, rows], ref_s[b])
        rest = [r for r in range(S_cap) if not f <= r < f + T]
        assert bool((kq[b, :, rest] == 0xC3).all()) and bool((vs[b, :, rest] == 5.0).all())
        assert bool((vq[b, :, rest] == 0xC3).all()) and bool((ks[b, :, rest] == 5.0).all())


def test_append_drops_rows_outside_the_cache():
    B, H, T, D, bs, S_cap = 2, 1, 4, 64, 32, 6
    q, k, v = (_rand((B, H, T, D), i) for i in range(3))
    table, pos = tqkv.rope_table(10, D), _positions(B, T, 1, 10, 0)
    kq, vq = (torch.full((B, H, S_cap, D // 2), 1, dtype=torch.uint8, device="cuda") for _ in "kv")
    ks, vs = (torch.zeros((B, H, S_cap, 2, 2), dtype=F16, device="cuda") for _ in "kv")
    starts = torch.tensor([4, -3], dtype=torch.int32, device="cuda")
    tqkv.qk_norm_rope_append_int4(q, k, v, pos, table, kq, ks, vq, vs, starts, bs)
    assert bool((kq[0, :, :4] == 1).all()) and bool((vq[1, :, 1:] == 1).all())
    full = [torch.empty((B, H, T, D // 2), dtype=torch.uint8, device="cuda") for _ in "kv"]
    fs = [torch.empty((B, H, T, 2, 2), dtype=F16, device="cuda") for _ in "kv"]
    tqkv.qk_norm_rope_append_int4(q, k, v, pos, table, full[0], fs[0], full[1], fs[1], 0, bs)
    assert torch.equal(kq[0, :, 4:], full[0][0, :, :2]) and torch.equal(vq[0, :, 4:], full[1][0, :, :2])
    assert torch.equal(kq[1, :, :1], full[0][1, :, 3:]) and torch.equal(vq[1, :, :1], full[1][1, :, 3:])


def test_an_axis_without_pairs():
    B, H, T, D = 1, 3, 9, 128
    q, k = _rand((B, H, T, D), 1), _rand((B, H, T, D), 2)
    table = tqkv.rope_table(40, D)
    pos = _positions(B, T, 3, 40, 5)
    for sections in ((0, 40, 24), (64, 0, 0), (3, 0, 61)):
        for interleaved in (False, True):
            cos, sin = _cos_sin(table, pos, sections)
            qo, ko = tqkv.qk_norm_rope(q, k, pos, table, sections=sections, interleaved=interleaved)
            _check(qo, q, None, cos, sin, 1e-6, interleaved)
            _check(ko, k, None, cos, sin, 1e-6, interleaved)


@pytest.mark.parametrize("D,rot,bs", [(128, 96, 32), (128, 32, 128), (64, 16, 32), (128, 64, 64)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_with_a_part_of_the_head_rotated(D, rot, bs, interleaved):
    B, Hq, Hkv, T = 2, 3, 2, 11
    q, k, v = (_rand((B, h, T, D), i) for i, h in enumerate((Hq, Hkv, Hkv)))
    table, pos = tqkv.rope_table(50, rot), _positions(B, T, 1, 50, 1)
    cos, sin = _cos_sin(table, pos, None)
    kq, vq = (torch.empty((B, Hkv, T, D // 2), dtype=torch.uint8, device="cuda") for _ in "kv")
    ks, vs = (torch.empty((B, Hkv, T, D // bs, 2), dtype=F16, device="cuda") for _ in "kv")
    qo = tqkv.qk_norm_rope_append_int4(q, k, v, pos, table, kq, ks, vq, vs, 0, bs, interleaved=interleaved)
    _check(qo, q, None, cos, sin, 1e-6, interleaved, exact=True)
    want_k, tol = norm_rope(f64(k), None, cos, sin, 1e-6, interleaved, exact=True)
    check_quantised(want_k, kq, ks, bs, slack=float((tol / np.abs(want_k).max(-1, keepdims=True)).max()) * 4)
    ref_c, ref_s = tqkv.kv_compress_int4(v, bs)
    assert torch.equal(vq, ref_c) and torch.equal(vs, ref_s)


def test_on_another_stream():
    """stream=: inputs made on the current stream, results read on it, ordered by events."""
    B, H, T, D, bs = 2, 4, 300, 128, 64
    table, pos = tqkv.rope_table(T, D), _positions(B, T, 1, T, 3)
    q, k, v = (_rand((B, H, T, D), i) for i in range(3))

    def run(**kw):
        c, s = tqkv.kv_compress_int4(v, bs, **kw)
        y = tqkv.kv_reconstruct_int4(c, s, bs, **kw)
        qo, ko = tqkv.qk_norm_rope(q, k, pos, table, **kw)
        tqkv.kv_append_int4(ko, c, s, 0, bs, **kw)
        return y, qo, ko, c, s, tqkv.decode_int4(qo[:, :, 0].contiguous(), c, s, c, s, bs, **kw)
    want = run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(5):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            q0 = run(stream=side)
        got = q0
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("D,bs,dtype", [(128, 32, BF16), (64, 64, F16)])
def test_prompt_then_tokens(D, bs, dtype, captured):
    """A prompt's K and V into the cache, then tokens one at a time: norm, rotation and append in one
    launch, attention over the grown cache, for sequences of different lengths; the step captured
    once and replayed, or launched each time.  Each answer is checked against float64 attention over
    what the cache holds, and the cache against float64 norms and rotations."""
    B, Hq, Hkv, S_cap, steps = 3, 4, 2, 80, 4
    prompt = [40, 1, 17]
    table = tqkv.rope_table(S_cap, D)
    kq, vq = (torch.zeros((B, Hkv, S_cap, D // 2), dtype=torch.uint8, device="cuda") for _ in "kv")
    ks, vs = (torch.zeros((B, Hkv, S_cap, D // bs, 2), dtype=F16, device="cuda") for _ in "kv")
    kw = _rand((D,), 7, dtype)
    all_k = _rand((B, Hkv, S_cap, D), 8, dtype)
    all_v = _rand((B, Hkv, S_cap, D), 9, dtype)
    T = max(prompt)
    pos = torch.arange(T, dtype=torch.int32, device="cuda").expand(B, T).contiguous()
    zeros = torch.zeros((B, Hq, T, D), dtype=dtype, device="cuda")
    # the padded batch: rows behind each prompt are overwritten token by token later
    tqkv.qk_norm_rope_append_int4(zeros, all_k[:, :, :T], all_v[:, :, :T], pos, table, kq, ks, vq, vs,
                                  0, bs, k_weight=kw)
    lengths = torch.tensor(prompt, dtype=torch.int32, device="cuda")
    after = lengths + 1
    q, k, v = (torch.zeros((B, h, 1, D), dtype=dtype, device="cuda") for h in (Hq, Hkv, Hkv))

    def step():
        p = lengths[:, None].contiguous()
        qr = tqkv.qk_norm_rope_append_int4(q, k, v, p, table, kq, ks, vq, vs, lengths, bs, k_weight=kw)
        return qr[:, :, 0], tqkv.decode_int4(qr[:, :, 0], kq, ks, vq, vs, bs, lengths=after)

    graph = None
    if captured:
        saved = [t.clone() for t in (kq, ks, vq, vs)]
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            qr, o = step()
        for t, s in zip((kq, ks, vq, vs), saved):
            t.copy_(s)
    cos, sin = _cos_sin(table, torch.arange(S_cap)[None].expand(B, S_cap), None)
    want_k, tol = norm_rope(f64(all_k), f64(kw), cos, sin, 1e-6, False, exact=True)
    for i in range(steps):
        n = [p + i for p in prompt]
        q.copy_(_rand((B, Hq, 1, D), 100 + i, dtype))
        for b in range(B):
            k[b, :, 0], v[b, :, 0] = all_k[b, :, n[b]], all_v[b, :, n[b]]
        lengths.copy_(torch.tensor(n, dtype=torch.int32))
        after.copy_(lengths + 1)
        if graph is not None:
            graph.replay()
        else:
            qr, o = step()
        torch.cuda.synchronize()
        check_attention(o, qr, kq, ks, vq, vs, bs, [m + 1 for m in n])
        for b in range(B):
            m = n[b] + 1
            check_quantised(want_k[b, :, :m], kq[b, :, :m], ks[b, :, :m], bs,
                            slack=float((tol[b] / np.abs(want_k[b]).max(-1, keepdims=True)).max()) * 4)
            c, s = tqkv.kv_compress_int4(all_v[b:b + 1, :, :m], bs)
            assert torch.equal(vq[b:b + 1, :, :m], c) and torch.equal(vs[b:b + 1, :, :m], s)
    assert tqkv.read_device_error() == 0
