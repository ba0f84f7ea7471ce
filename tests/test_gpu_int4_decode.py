"""Decode attention over the 4-bit cache (tqkv_decode_int4), against attention over the cache's
values in float64."""
import numpy as np
import pytest
import torch

import tqkv
from tqkv import Workspace

from int4_reference import VALID, check_attention, f64, spread, unpack, values

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _rand(shape, seed, dtype=F16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _cache(B, H, S, D, bs, seed, mul=1.0):
    return tqkv.kv_compress_int4(_rand((B, H, S, D), seed) * mul, bs)


def _run(B, Hq, Hkv, S, D, bs, dtype=F16, lengths=None, seed=0, **kw):
    q = _rand((B, Hq, D), seed + 1, dtype)
    kq, ks = _cache(B, Hkv, S, D, bs, seed + 2)
    vq, vs = _cache(B, Hkv, S, D, bs, seed + 3)
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    o = tqkv.decode_int4(q, kq, ks, vq, vs, bs, lengths=n, **kw)
    assert tqkv.read_device_error() == 0
    return o, q, kq, ks, vq, vs


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,bs", VALID)
@pytest.mark.parametrize("S", [1, 2, 15, 16, 17, 31, 32, 33, 64, 65, 127, 129, 500])
def test_lengths_around_the_tiles(S, D, bs, dtype):
    o, q, *cache = _run(2, 3, 3, S, D, bs, dtype, seed=S)
    check_attention(o, q, *cache, bs, [S, S])


@pytest.mark.parametrize("D,bs", VALID)
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (2, 1), (6, 2), (5, 1), (8, 1), (9, 1), (16, 1), (24, 2),
                                    (17, 1), (40, 1), (33, 3)])
def test_groups_of_query_heads(Hq, Hkv, D, bs):
    o, q, *cache = _run(2, Hq, Hkv, 333, D, bs, seed=Hq)
    check_attention(o, q, *cache, bs, [333, 333])


@pytest.mark.parametrize("D,bs,G", [(128, 128, 1), (128, 32, 4), (64, 32, 16), (64, 64, 7)])
@pytest.mark.parametrize("S", [9000, 20011])
def test_heads_cut_across_many_blocks(S, D, bs, G):
    o, q, *cache = _run(1, G, 1, S, D, bs, BF16, seed=S + G)
    check_attention(o, q, *cache, bs, [S])


@pytest.mark.parametrize("D,bs,G", [(128, 64, 4), (64, 32, 1), (128, 32, 12)])
def test_ragged_lengths(D, bs, G):
    S = 700
    lengths = [700, 0, 1, 33, 0, 699, 256, 64, 0, 5, 128, 31] + list(range(40, 75))
    o, q, *cache = _run(len(lengths), 2 * G, 2, S, D, bs, lengths=lengths, seed=G)
    check_attention(o, q, *cache, bs, lengths)
    for b, n in enumerate(lengths):
        if n == 0:
            assert not o[b].any()


@pytest.mark.parametrize("D,bs", VALID)
@pytest.mark.parametrize("B,Hkv,top", [(3, 2, 150), (2, 1, 40), (7, 3, 90), (40, 2, 60), (40, 4, 17),
                                       (149, 1, 20), (151, 2, 140), (13, 8, 260)])
def test_short_sequences_in_more_blocks_than_tiles(B, Hkv, top, D, bs):
    """Blocks with fewer rows than their warps take; cuts fall at every place of a sequence."""
    g = torch.Generator().manual_seed(B * top)
    for lengths in ([top] * B, torch.randint(0, top + 1, (B,), generator=g).tolist()):
        o, q, *cache = _run(B, 2 * Hkv, Hkv, top, D, bs, lengths=lengths, seed=B)
        check_attention(o, q, *cache, bs, lengths)
    o, q, *cache = _run(B, 2 * Hkv, Hkv, top, D, bs, seed=B)
    check_attention(o, q, *cache, bs, [top] * B)


def test_lengths_are_taken_into_the_range():
    lengths = [-5, 2 ** 31 - 1, -2 ** 31, 41]
    _, q, *cache = _run(4, 2, 1, 100, 128, 64)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    o = tqkv.decode_int4(q, *cache, 64, S=40, lengths=n)
    check_attention(o, q, *cache, 64, [0, 40, 0, 40])


def test_all_sequences_empty():
    q = _rand((3, 4, 64), 1)
    cache = [t for n in (2, 3) for t in _cache(3, 2, 50, 64, 32, n)]
    out = torch.full_like(q, 9.0)
    tqkv.decode_int4(q, *cache, 32, lengths=torch.zeros(3, dtype=torch.int32, device="cuda"), out=out)
    assert not out.any()
    out.fill_(9.0)
    tqkv.decode_int4(q, *cache, 32, S=0, out=out)
    assert not out.any()


@pytest.mark.parametrize("D,bs", VALID)
def test_rows_behind_the_length_are_not_read(D, bs):
    """NaN and arbitrary bytes behind each length change nothing, and the caches stay as they are."""
    B, Hq, Hkv, S = 3, 4, 2, 150
    lengths = [1, 70, 149]
    o, q, kq, ks, vq, vs = _run(B, Hq, Hkv, S, D, bs, lengths=lengths)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    for b, m in enumerate(lengths):
        kq[b, :, m:], vq[b, :, m:] = 0xFF, 0xFF
        ks[b, :, m:], vs[b, :, m:] = float("nan"), float("inf")
    before = [t.clone() for t in (kq, ks, vq, vs)]
    again = tqkv.decode_int4(q, kq, ks, vq, vs, bs, lengths=n)
    assert torch.equal(o, again)
    for t, u in zip((kq, ks, vq, vs), before):
        assert torch.equal(t.view(torch.uint8), u.view(torch.uint8))


def test_nan_reaches_only_its_head():
    o, q, kq, ks, vq, vs = _run(2, 4, 2, 100, 128, 32)
    ks[1, 0, 50, 2] = float("nan")
    vs[0, 1, 7, 1] = float("nan")
    again = tqkv.decode_int4(q, kq, ks, vq, vs, 32)
    assert torch.isnan(again[1, :2]).all()
    assert torch.isnan(again[0, 2:, 32:64]).all() and not torch.isnan(again[0, 2:, :32]).any()
    assert torch.equal(again[0, :2], o[0, :2]) and torch.equal(again[1, 2:], o[1, 2:])


@pytest.mark.parametrize("kmul,vmul,qmul", [(1, 1e-4, 1), (1, 2e4, 1), (30, 1, 1), (1e-3, 1, 1e3),
                                            (1, 1, 0), (200, 1e3, 0.5), (1, 1, 1e-6)])
@pytest.mark.parametrize("D,bs", [(128, 32), (64, 64)])
def test_magnitudes(D, bs, kmul, vmul, qmul):
    """Weights and values of every magnitude, peaked and flat scores."""
    B, Hq, Hkv, S = 1, 4, 2, 400
    q = (_rand((B, Hq, D), 1).float() * qmul).half()
    kq, ks = _cache(B, Hkv, S, D, bs, 2, kmul)
    vq, vs = tqkv.kv_compress_int4((_rand((B, Hkv, S, D), 3).float().clamp(-2.5, 2.5) * vmul).half(), bs)
    o = tqkv.decode_int4(q, kq, ks, vq, vs, bs)
    check_attention(o, q, kq, ks, vq, vs, bs, [S])


def test_one_token_far_above_many_small_ones():
    """A token of a large weight and a small value scale beside thousands of small weights whose
    values are large: their sum must not be lost below fp16's range."""
    S, D, bs = 8000, 128, 128
    q = torch.zeros((1, 1, D), dtype=F16, device="cuda")
    q[..., 0] = 10.0
    k = _rand((1, 1, S, D), 4) * 0.01
    k[0, 0, 4321, 0] = 14.0
    v = _rand((1, 1, S, D), 5) * 30 + 20
    v[0, 0, 4321] *= 1e-4
    kq, ks = tqkv.kv_compress_int4(k, bs)
    vq, vs = tqkv.kv_compress_int4(v, bs)
    o = tqkv.decode_int4(q, kq, ks, vq, vs, bs)
    check_attention(o, q, kq, ks, vq, vs, bs, [S])


@pytest.mark.parametrize("G,copies", [(1, 8), (2, 4), (3, 2), (4, 2)])
def test_small_groups_average_the_rounding_of_their_weights(G, copies):
    """fp16 over many tokens.  The error's root mean square is that of O's own rounding, known
    exactly, and of the weights': a rounding of p * scale is uniform in half a step of at most 2^-11,
    so 2^-11 / sqrt(3) of it at most, independent between tokens and between the copies whose mean is
    taken.  Terms in fp32 are 2^-10 of that.  4096 elements' root mean square has a deviation of
    1 / sqrt(8192); G * 4096 of them are here: four deviations are 4.5 %."""
    S, D, bs, H = 12000, 128, 128, 32
    o, q, kq, ks, vq, vs = _run(1, G * H, H, S, D, bs, seed=G)
    kq, ks, vq, vs = (t.cpu().numpy() for t in (kq, ks, vq, vs))
    got, qd = f64(o)[0], f64(q)[0]
    own, weights, total = 0.0, 0.0, 0.0
    middle = np.where(np.arange(S) % 2, 7.0, 8.0)[:, None]
    for h in range(H):
        s, z = spread(vs[0, h].astype(np.float64), bs)
        c = unpack(vq[0, h]) - middle
        k = values(kq[0, h], ks[0, h].astype(np.float64), bs)
        for i in range(h * G, h * G + G):
            t = k @ qd[i] / np.sqrt(D)
            p = np.exp(t - t.max())
            p /= p.sum()
            want = p @ (c * s + (z + middle * s))
            total += ((got[i] - want) ** 2).sum()
            own += ((want.astype(np.float16) - want) ** 2).sum()
            weights += (p ** 2 @ (c * s) ** 2).sum() * (2.0 ** -11) ** 2 / 3
    assert total <= 1.045 ** 2 * (own + weights / copies), (total, own, weights)


def test_bf16_queries_beyond_fp16():
    q = (_rand((1, 2, 128), 1).float() * 1e5).to(BF16)
    assert float(q.abs().max()) > 65504
    kq, ks = _cache(1, 2, 77, 128, 64, 2, 1e-4)
    vq, vs = _cache(1, 2, 77, 128, 64, 3)
    o = tqkv.decode_int4(q, kq, ks, vq, vs, 64)
    check_attention(o, q, kq, ks, vq, vs, 64, [77])


def test_offsets_past_32_bits():
    D, bs, S_cap = 128, 128, 1 << 25
    codes = [torch.empty((1, 3, S_cap, D // 2), dtype=torch.uint8, device="cuda") for _ in range(2)]
    scales = [torch.empty((1, 3, S_cap, 1, 2), dtype=F16, device="cuda") for _ in range(2)]
    n = 130
    for i in range(2):
        tqkv.kv_append_int4(_rand((1, 3, n, D), i), codes[i], scales[i], 0, bs)
    q = _rand((1, 3, D), 5)
    o = tqkv.decode_int4(q, codes[0], scales[0], codes[1], scales[1], bs, S=n)
    small = [t[:, :, :n].contiguous() for p in zip(codes, scales) for t in p]
    assert torch.equal(o, tqkv.decode_int4(q, *small, bs))
    check_attention(o, q, *small, bs, [n])


def test_results_repeat_and_the_workspace_is_left_zeroed():
    B, Hq, Hkv, S, D, bs = 3, 8, 2, 5000, 128, 64
    lengths = [5000, 17, 3333]
    o, q, *cache = _run(B, Hq, Hkv, S, D, bs, lengths=lengths)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    ws = Workspace()
    for _ in range(20):
        assert torch.equal(o, tqkv.decode_int4(q, *cache, bs, lengths=n, workspace=ws))
    assert not ws.buf.any()


@pytest.mark.parametrize("lengths,G", [([1, 5999], 4), ([3000, 2999], 1), ([2500, 700, 4000], 8),
                                       ([5000, 3], 12)])
def test_sums_keep_their_order(lengths, G):
    """A block that arrives last at two cut units merges both at once, at other times one: the
    bits are the same, call after call, alone and beside another call."""
    B, S = len(lengths), 6000
    sets = []
    for i in range(2):
        q = _rand((B, 2 * G, 128), 10 * i)
        sets.append((q, *_cache(B, 2, S, 128, 64, 10 * i + 1), *_cache(B, 2, S, 128, 64, 10 * i + 2)))
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    want = [tqkv.decode_int4(*s, 64, lengths=n) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for i in range(150):
        got = [tqkv.decode_int4(*s, 64, lengths=n, stream=st if i % 2 else None)
               for s, st in zip(sets, streams)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


def test_workspace_shared_with_the_int8_decode():
    ws = Workspace()
    B, H, S, D, bs = 1, 4, 30000, 128, 64
    q, k, v = _rand((B, H, D), 1), _rand((B, H, S, D), 2), _rand((B, H, S, D), 3)
    c8 = [*tqkv.kv_compress(k, bs), *tqkv.kv_compress(v, bs)]
    c4 = [*tqkv.kv_compress_int4(k, bs), *tqkv.kv_compress_int4(v, bs)]
    o8, o4 = tqkv.decode_int8(q, *c8, bs), tqkv.decode_int4(q, *c4, bs)
    for _ in range(3):
        assert torch.equal(o8, tqkv.decode_int8(q, *c8, bs, workspace=ws))
        assert torch.equal(o4, tqkv.decode_int4(q, *c4, bs, workspace=ws))


@pytest.mark.parametrize("G", [1, 4, 12])
def test_a_workspace_for_the_largest_batch_serves_smaller_ones(G):
    """Its size grows with the sizes, and the kernels take it at every batch below."""
    need = tqkv.load().tqkv_decode_int4_workspace_bytes
    for D in (64, 128):
        for sizes in ([(B, H, S) for S in (1, 40, 700, 5000) for H in (1, 3) for B in range(1, 320)],
                      [(B, 1, S) for B in (1, 149, 160) for S in range(1, 4000, 13)],
                      [(3, H, S) for S in (1, 300, 3000) for H in range(1, 120)]):
            last = 0, None
            for B, H, S in sizes:
                n = need(B, H * G, H, S, D)
                if last[1] is not None and (B, H, S) >= last[1] and sum(
                        x != y for x, y in zip((B, H, S), last[1])) == 1:
                    assert n >= last[0], (B, H, S)
                last = n, (B, H, S)
    S, D, bs = 40, 128, 64
    ws = Workspace()
    _run(160, G, 1, S, D, bs, workspace=ws)
    size = ws.buf.numel()
    for B in (159, 149, 148, 147, 75, 2, 1):
        o, q, *cache = _run(B, G, 1, S, D, bs, workspace=ws)
        check_attention(o, q, *cache, bs, [S] * B)
    assert ws.buf.numel() == size and not ws.buf.any()


def test_streams_side_by_side():
    """Calls on several streams at once, each with the workspace of its stream."""
    sets = []
    for i in range(3):
        q = _rand((1, 8, 128), 10 * i)
        sets.append((q, *_cache(1, 2, 9000, 128, 64, 10 * i + 1), *_cache(1, 2, 9000, 128, 64, 10 * i + 2)))
    want = [tqkv.decode_int4(*s, 64) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(10):
        got = [tqkv.decode_int4(*s, 64, stream=st) for s, st in zip(sets, streams)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_graphs_captured_on_one_stream_replay_side_by_side():
    """Two captured calls own their scratch: replays on different streams do not disturb each
    other, and lengths may change between replays."""
    sets, graphs, outs, lens = [], [], [], []
    for i in range(2):
        q = _rand((2, 8, 128), 10 * i)
        sets.append((q, *_cache(2, 2, 6000, 128, 64, 10 * i + 1), *_cache(2, 2, 6000, 128, 64, 10 * i + 2)))
        lens.append(torch.tensor([6000, 100], dtype=torch.int32, device="cuda"))
    for s, n in zip(sets, lens):
        tqkv.decode_int4(*s, 64, lengths=n)
    torch.cuda.synchronize()
    for s, n in zip(sets, lens):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(tqkv.decode_int4(*s, 64, lengths=n))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in sets]
    for lengths in ([6000, 100], [1, 5999], [0, 3000]):
        for n in lens:
            n.copy_(torch.tensor(lengths))
        want = [tqkv.decode_int4(*s, 64, lengths=n) for s, n in zip(sets, lens)]
        torch.cuda.synchronize()
        for _ in range(5):
            for g, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_workspace_does_not_grow_while_captured():
    q = _rand((1, 8, 128), 1)
    cache = (*_cache(1, 2, 6000, 128, 64, 2), *_cache(1, 2, 6000, 128, 64, 3))
    ws = Workspace()
    tqkv.decode_int4(q, *cache, 64)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(ValueError, match="captured"):
            tqkv.decode_int4(q, *cache, 64, workspace=ws)
    want = tqkv.decode_int4(q, *cache, 64, workspace=ws)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = tqkv.decode_int4(q, *cache, 64, workspace=ws)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
