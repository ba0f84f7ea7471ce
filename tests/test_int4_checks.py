"""The 4-bit operators refuse what they cannot do before anything is launched: the C entries by
status, the Python front end by ValueError.  No GPU is needed: the pointers are never followed."""
import ctypes

import numpy as np
import pytest
import torch

import tqkv
from tqkv import _lib, int4

from int4_reference import element_places, pack, quantise, unpack, values

OK, UNSUPPORTED, SIZE, MISALIGNED, WORKSPACE, CUDA, NULL = range(7)
P = 1 << 20


def test_append_and_compress_refusals():
    lib = tqkv.load()

    def call(x=P, st=(256, 128, 128), cq=P, cs=P, starts=None, t0=0, B=1, H=2, T=1, D=128, bs=64,
             cap=4, dt=0):
        s = (ctypes.c_longlong * 3)(*st) if st else None
        return lib.tqkv_kv_append_int4(x, s, cq, cs, starts, t0, B, H, T, D, bs, cap, dt, None)
    for D, bs in ((96, 32), (64, 128), (128, 16), (256, 128), (0, 0)):
        assert call(D=D, bs=bs) == UNSUPPORTED
    assert call(dt=2) == UNSUPPORTED and call(dt=-1) == UNSUPPORTED
    for kw in (dict(B=0), dict(H=-1), dict(T=0), dict(cap=0), dict(T=5), dict(t0=-1), dict(t0=4),
               dict(T=4, t0=1), dict(T=1 << 20, cap=1 << 20, B=1 << 15), dict(T=5, starts=P)):
        assert call(**kw) == SIZE, kw
    for kw in (dict(x=None), dict(cq=None), dict(cs=None)):
        assert call(**kw) == NULL
    for kw in (dict(x=P + 8), dict(cq=P + 8), dict(cs=P + 4), dict(st=(4, 128, 128)), dict(st=(8, 8, 1))):
        assert call(**kw) == MISALIGNED
    assert lib.tqkv_kv_compress_int4(None, P, P, 1, 1, 1, 128, 64, 0, None) == NULL
    assert lib.tqkv_kv_compress_int4(P, P, P, 1, 1, 0, 128, 64, 0, None) == SIZE


def test_reconstruct_refusals():
    lib = tqkv.load()

    def call(q=P, s=P, y=P, starts=None, t0=0, B=1, H=2, T=1, D=128, bs=64, cap=4, dt=0):
        return lib.tqkv_kv_reconstruct_int4(q, s, y, starts, t0, B, H, T, D, bs, cap, dt, None)
    assert call(D=32, bs=32) == UNSUPPORTED and call(dt=5) == UNSUPPORTED
    assert call(T=0) == SIZE and call(t0=4) == SIZE and call(T=5, starts=P) == SIZE
    assert call(q=None) == NULL and call(s=None) == NULL and call(y=None) == NULL
    assert call(q=P + 4) == MISALIGNED and call(s=P + 4) == MISALIGNED and call(y=P + 2) == MISALIGNED


def test_decode_refusals():
    lib = tqkv.load()

    def call(q=P, kq=P, ks=P, vq=P, vs=P, n=None, o=P, B=1, Hq=2, Hkv=2, S=4, cap=4, D=128, bs=64, dt=0):
        return lib.tqkv_decode_int4(q, kq, ks, vq, vs, n, o, B, Hq, Hkv, S, cap, D, bs, dt, None, 0, None)
    assert call(D=96) == UNSUPPORTED and call(bs=16) == UNSUPPORTED and call(dt=3) == UNSUPPORTED
    for kw in (dict(B=0), dict(Hq=0), dict(Hkv=0), dict(Hq=3), dict(S=-1), dict(S=5), dict(cap=0, S=0),
               dict(B=1 << 20, Hq=1 << 12)):
        assert call(**kw) == SIZE, kw
    for name in ("q", "kq", "ks", "vq", "vs", "o"):
        assert call(**{name: None}) == NULL
        assert call(**{name: P + 8}) == MISALIGNED
    assert lib.tqkv_decode_int4_workspace_bytes(1, 3, 2, 100, 128) == 0
    assert lib.tqkv_decode_int4_workspace_bytes(0, 2, 2, 100, 128) == 0


def _args(**kw):
    a = _lib.NormRopeArgs()
    base = dict(q=P, k=P, v=P, table=P, positions=P, q_out=P, k_out=P, kq=P, vq=P, ks=P, vs=P, eps=1e-6,
                B=1, H_q=2, H_kv=1, T=1, D=128, block_size=64, S_cap=4, rot_dim=128, max_pos=9, axes=1)
    for name, v in {**base, **kw}.items():
        if isinstance(v, (tuple, list)):
            getattr(a, name)[:len(v)] = v
        else:
            setattr(a, name, v)
    return ctypes.byref(a)


def test_packed_arguments_are_the_structure():
    """The front end packs tqkv_norm_rope_args in one step: every field lands where ctypes has it."""
    n = len(_lib.NORM_ROPE_PACK.unpack(bytes(_lib.NORM_ROPE_PACK.size)))
    assert _lib.NORM_ROPE_PACK.size == ctypes.sizeof(_lib.NormRopeArgs) and n == 41
    a = _lib.NormRopeArgs.from_buffer_copy(_lib.NORM_ROPE_PACK.pack(*range(1, n + 1)))
    flat = []
    for name, _ in _lib.NormRopeArgs._fields_:
        v = getattr(a, name)
        flat += list(v) if hasattr(v, "__len__") else [v]
    assert flat == list(range(1, n + 1))


def test_norm_rope_refusals():
    lib = tqkv.load()
    both = (lib.tqkv_qk_norm_rope, lib.tqkv_qk_norm_rope_append_int4)
    for f in both:
        assert f(None, None) == NULL
        for kw in (dict(D=96), dict(dtype=2), dict(rot_dim=0), dict(rot_dim=24), dict(rot_dim=144),
                   dict(D=64, rot_dim=128), dict(axes=0), dict(axes=5)):
            assert f(_args(**kw), None) == UNSUPPORTED, kw
        for kw in (dict(B=0), dict(H_q=0), dict(H_kv=0), dict(T=0), dict(max_pos=0), dict(eps=-1.0),
                   dict(eps=float("nan")), dict(axes=2, sections=(32, 31)), dict(axes=2, sections=(65, -1)),
                   dict(axes=4, sections=(2 ** 31 - 1, 2 ** 31 - 1, 2, 64)),
                   dict(B=1 << 16, T=1 << 16, S_cap=1 << 16)):
            assert f(_args(**kw), None) == SIZE, kw
        for name in ("q", "k", "table", "positions", "q_out"):
            assert f(_args(**{name: None}), None) == NULL
        for kw in (dict(q=P + 8), dict(k=P + 2), dict(q_out=P + 8), dict(q_weight=P + 8), dict(table=P + 8),
                   dict(q_strides=(4, 8, 8)), dict(k_strides=(8, 8, 12))):
            assert f(_args(**kw), None) == MISALIGNED, kw
    plain, append = both
    assert plain(_args(k_out=None), None) == NULL
    for name in ("v", "kq", "ks", "vq", "vs"):
        assert append(_args(**{name: None}), None) == NULL
        assert append(_args(**{name: P + 8}), None) == MISALIGNED
    assert append(_args(v_strides=(1, 8, 8)), None) == MISALIGNED
    assert append(_args(block_size=16), None) == UNSUPPORTED
    for kw in (dict(S_cap=0), dict(T=5), dict(t0=4), dict(t0=-1), dict(T=5, starts=P)):
        assert append(_args(**kw), None) == SIZE, kw


def test_python_refuses_what_does_not_fit():
    q = torch.zeros((1, 2, 64), dtype=torch.float16)
    x = torch.zeros((1, 2, 8, 64), dtype=torch.float16)
    c = torch.zeros((1, 2, 8, 32), dtype=torch.uint8)
    s = torch.zeros((1, 2, 8, 1, 2), dtype=torch.float16)
    t = torch.zeros((8, 32, 2))
    pos = torch.zeros((1, 8), dtype=torch.int32)

    def refused(f, *a, **kw):
        with pytest.raises(ValueError):
            f(*a, **kw)
    # everything fits, but nothing is on a GPU
    refused(int4.kv_append_int4, x, c, s, 0, 64)
    refused(int4.kv_reconstruct_int4, c, s, 64)
    refused(int4.decode_int4, q, c, s, c, s, 64)
    refused(int4.qk_norm_rope, x, x, pos, t)
    refused(int4.qk_norm_rope_append_int4, x, x, x, pos, t, c, s, c, s, 0, 64)
    # types and shapes
    refused(int4.kv_append_int4, x.float(), c, s, 0, 64)
    refused(int4.kv_append_int4, x[..., :32], c, s, 0, 64)
    refused(int4.kv_append_int4, x, c.to(torch.int8), s, 0, 64)
    refused(int4.kv_append_int4, x, c, s[..., 0], 0, 64)
    refused(int4.kv_append_int4, x, c, s, torch.zeros(1, dtype=torch.int64), 64)
    refused(int4.kv_append_int4, x, c, s, torch.zeros(2, dtype=torch.int32), 64)
    refused(int4.kv_append_int4, x, c, s, 0, 0)
    refused(int4.kv_append_int4, x.transpose(2, 3), c, s, 0, 64)
    refused(int4.kv_append_int4, torch.zeros((1, 2, 8, 65), dtype=torch.float16)[..., :64], c, s, 0, 64)
    refused(int4.kv_compress_int4, x[0], 64)
    refused(int4.kv_reconstruct_int4, c, s, 64, t0=torch.zeros(1, dtype=torch.int32))
    refused(int4.kv_reconstruct_int4, c, s, 64, dtype=torch.float32)
    refused(int4.decode_int4, q[..., :32], c, s, c, s, 64)
    refused(int4.decode_int4, torch.zeros((1, 3, 64), dtype=torch.float16), c, s, c, s, 64)
    refused(int4.decode_int4, q, c, s, c[:, :, :4], s, 64)
    refused(int4.decode_int4, q, c, s, c, s, 64, lengths=torch.zeros(1, dtype=torch.int64))
    refused(int4.qk_norm_rope, x, x[:, :, :4], pos, t)
    refused(int4.qk_norm_rope, x, x, pos[:, :4], t)
    refused(int4.qk_norm_rope, x, x, pos, t.half())
    refused(int4.qk_norm_rope, x, x, pos, t, q_weight=torch.zeros(64))
    refused(int4.qk_norm_rope, x, x, pos, t, sections=(16, 15))
    refused(int4.qk_norm_rope, x, x, pos, t, sections=(16, 16))     # positions have one axis
    refused(int4.qk_norm_rope_append_int4, x, x, x[:, :1], pos, t, c, s, c, s, 0, 64)
    refused(int4.rope_table, 8, 24, device="cpu")
    refused(int4.rope_table, 0, 64, device="cpu")


def test_numbers_that_a_c_int_would_cut_short(monkeypatch):
    """ctypes takes the low 32 bits of a number: 2^32 + 1 would be row 1."""
    monkeypatch.setattr(int4, "_device", lambda t, name: -1)
    monkeypatch.setattr(int4, "_current_device", lambda: -1)
    x = torch.zeros((1, 2, 8, 64), dtype=torch.float16)
    c = torch.zeros((1, 2, 8, 32), dtype=torch.uint8)
    s = torch.zeros((1, 2, 8, 1, 2), dtype=torch.float16)
    q, t = torch.zeros((1, 2, 64), dtype=torch.float16), torch.zeros((8, 32, 2))
    pos = torch.zeros((1, 8), dtype=torch.int32)
    for far in (2 ** 32 + 1, 2 ** 31, -2 ** 32, -2 ** 31 - 1):
        for call in (lambda: int4.kv_append_int4(x[:, :, :1], c, s, far, 64),
                     lambda: int4.kv_reconstruct_int4(c, s, 64, t0=far, T=1),
                     lambda: int4.kv_reconstruct_int4(c, s, 64, T=far),
                     lambda: int4.decode_int4(q, c, s, c, s, 64, S=far),
                     lambda: int4.qk_norm_rope_append_int4(x, x, x, pos, t, c, s, c, s, far, 64)):
            with pytest.raises(ValueError, match="32 bits"):
                call()
    with pytest.raises(ValueError, match="does not match"):
        int4.kv_append_int4(x[:, :, :1].expand(1, 2, 2 ** 32 + 1, 64), c, s, 0, 64)


@pytest.mark.parametrize("D", [64, 128])
def test_packed_order(D):
    """The order that include/tqkv.h documents: every nibble once, a 32-element group's four words
    D / 8 bytes apart, and each quarter of a row holding one word of every group."""
    byte, shift = element_places(D)
    assert len({(b, s) for b, s in zip(byte, shift)}) == D
    for i in range(D):
        assert byte[i] // (D // 8) == i % 32 // 8
    c = np.random.default_rng(0).integers(0, 16, (3, D)).astype(np.uint8)
    assert np.array_equal(unpack(pack(c)), c)


def test_quantised_values_are_within_half_a_step():
    x = np.random.default_rng(1).standard_normal((50, 128)).astype(np.float16).astype(np.float64)
    for bs in (32, 64, 128):
        c, s = quantise(x, bs)
        step = np.repeat(s[..., 0].astype(np.float64), bs, -1)
        # half a step, and the ends where the fp16 step times 15 falls short of the range
        assert (np.abs(values(pack(c), s, bs) - x) <= step * (0.5 + 15 * 2.0 ** -10)).all()
