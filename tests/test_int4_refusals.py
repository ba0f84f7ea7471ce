"""What the 4-bit front end refuses, check by check, with the message of the check that is meant.  The
tensors are on the CPU and pass for those of one device; the library is a stand-in that counts calls, so
that a check that is missing shows as a call that goes through."""
import types

import pytest
import torch

from tqkv import int4

F16, BF16, I32, U8 = torch.float16, torch.bfloat16, torch.int32, torch.uint8
B, H, HQ, T, S, D, BS = 2, 2, 4, 3, 8, 64, 32


@pytest.fixture
def calls(monkeypatch):
    made = []

    class Library:
        def __getattr__(self, name):
            return lambda *a: made.append(name) or 0

    library = Library()
    monkeypatch.setattr(int4, "load", lambda: library)
    monkeypatch.setattr(int4, "_device", lambda t, name: t.get_device())
    monkeypatch.setattr(int4, "_current_device", lambda: -1)
    monkeypatch.setattr(int4, "_current_stream", lambda index: 0)
    monkeypatch.setattr(int4, "_workspace", lambda *a: (None, 0))
    return made


def x(h=H, t=T, d=D, b=B, dtype=F16):
    return torch.zeros((b, h, t, d), dtype=dtype)


def cache(s=S, h=H, d=D, b=B, bs=BS):
    return torch.zeros((b, h, s, d // 2), dtype=U8), torch.zeros((b, h, s, d // bs, 2), dtype=F16)


def ints(*shape, dtype=I32):
    return torch.zeros(shape, dtype=dtype)


class Elsewhere(torch.Tensor):
    def get_device(self):
        return 1


def far(*shape, dtype=F16):
    """A tensor of that shape on another device."""
    return torch.zeros(shape, dtype=dtype).as_subclass(Elsewhere)


def append(**kw):
    c, s = cache()
    a = dict(x=x(), cache_q=c, cache_s=s, t0=0, block_size=BS)
    return int4.kv_append_int4(**{**a, **kw})


def compress(**kw):
    return int4.kv_compress_int4(**{**dict(x=x(), block_size=BS), **kw})


def reconstruct(**kw):
    c, s = cache()
    return int4.kv_reconstruct_int4(**{**dict(xq=c, scales=s, block_size=BS), **kw})


def decode(**kw):
    (kq, ks), (vq, vs) = cache(), cache()
    a = dict(q=torch.zeros((B, HQ, D), dtype=F16), kq=kq, ks=ks, vq=vq, vs=vs, block_size=BS)
    return int4.decode_int4(**{**a, **kw})


def rope(**kw):
    a = dict(q=x(HQ), k=x(), positions=ints(B, T), table=torch.zeros((9, D // 2, 2)))
    return int4.qk_norm_rope(**{**a, **kw})


def rope_append(**kw):
    (kq, ks), (vq, vs) = cache(), cache()
    a = dict(q=x(HQ), k=x(), v=x(), positions=ints(B, T), table=torch.zeros((9, D // 2, 2)), kq=kq, ks=ks, vq=vq,
             vs=vs, t0=0, block_size=BS)
    return int4.qk_norm_rope_append_int4(**{**a, **kw})


odd = torch.zeros((B, H, T, D + 4), dtype=F16)[..., :D]         # rows D + 4 apart
gaps = torch.zeros((B, H, T, 2 * D), dtype=F16)[..., ::2]        # elements 2 apart
wide = torch.zeros((B, H, T, D + 8), dtype=F16)[..., :D]

ACCEPTED = [
    (append, {}), (append, dict(x=wide)), (append, dict(t0=ints(B))), (append, dict(x=x(dtype=BF16))),
    (append, dict(x=odd[:1, :1, :1], cache_q=cache(h=1, b=1)[0], cache_s=cache(h=1, b=1)[1])),
    (compress, {}), (compress, dict(xq=cache(T)[0], scales=cache(T)[1])),
    (reconstruct, {}), (reconstruct, dict(t0=ints(B), T=T)), (reconstruct, dict(y=x(t=S, dtype=BF16))),
    (decode, {}), (decode, dict(lengths=ints(B), S=5)), (decode, dict(out=torch.zeros((B, HQ, D), dtype=F16))),
    (rope, {}), (rope, dict(q_weight=torch.zeros(D, dtype=F16), k_weight=torch.zeros(D, dtype=F16))),
    (rope, dict(positions=ints(3, B, T), sections=(8, 12, 12))), (rope, dict(q_out=x(HQ), k_out=x())),
    (rope_append, {}), (rope_append, dict(t0=ints(B), q_out=x(HQ))),
]


@pytest.mark.parametrize("f,kw", ACCEPTED)
def test_what_fits_reaches_the_library(calls, f, kw):
    f(**kw)
    assert len(calls) == 1


REFUSED = [
    # writing
    (append, dict(x=x(dtype=torch.float32)), "x must be fp16 or bf16"),
    (append, dict(x=x()[0]), r"x must be a .* tensor \[B, H, T, D\]"),
    (append, dict(x=gaps), "x: the last dimension must be adjacent"),
    (append, dict(x=odd), "x: strides must be multiples of 8"),
    (append, dict(x=x(d=128)), "does not match x"),
    (append, dict(x=x(h=1)), "does not match x"),
    (append, dict(x=x(b=1)), "does not match x"),
    (append, dict(x=x(t=S + 1)), "does not match x"),
    (append, dict(cache_q=cache()[0].to(torch.int8)), "cache_q must be a contiguous uint8"),
    (append, dict(cache_q=cache()[0][0]), "cache_q must be a contiguous uint8"),
    (append, dict(cache_q=cache(2 * S)[0][:, :, ::2]), "cache_q must be a contiguous uint8"),
    (append, dict(cache_q=far(B, H, S, D // 2, dtype=U8), x=x()), "cache_q must be a contiguous uint8"),
    (append, dict(cache_s=cache()[1][..., 0]), "cache_s must be a contiguous"),
    (append, dict(cache_s=cache()[1].to(BF16)), "cache_s must be a contiguous"),
    (append, dict(cache_s=cache(bs=64)[1]), "cache_s must be a contiguous"),
    (append, dict(cache_s=cache(S - 1)[1]), "cache_s must be a contiguous"),
    (append, dict(cache_s=None), "cache_s is required"),
    (append, dict(block_size=0), "block_size 0 does not divide D 64"),
    (append, dict(block_size=-32), "block_size -32 does not divide D 64"),
    (append, dict(block_size=48), "block_size 48 does not divide D 64"),
    (append, dict(t0=ints(B, dtype=torch.int64)), "t0 must be a contiguous"),
    (append, dict(t0=ints(B + 1)), "t0 must be a contiguous"),
    (append, dict(t0=far(B, dtype=I32)), "t0 must be a contiguous"),
    (append, dict(x=x(b=0), cache_q=torch.zeros((0, H, 2 ** 31, D // 2), dtype=U8)), "S_cap 2147483648 does not fit"),
    (append, dict(t0=2 ** 31), "t0 2147483648 does not fit 32 bits"),
    (compress, dict(x=x()[0]), r"x must be \[B, H, S, D\]"),
    (compress, dict(block_size=0), "block_size 0 does not divide D 64"),
    (compress, dict(block_size=48), "block_size 48 does not divide D 64"),
    (compress, dict(x=x(dtype=torch.float32)), "x must be fp16 or bf16"),
    (compress, dict(xq=cache()[0], scales=cache()[1]), "does not have x's 3 rows"),
    (compress, dict(xq=cache(T)[0][0]), "does not have x's 3 rows"),
    (compress, dict(scales=cache()[1]), "cache_s must be a contiguous"),
    # reading
    (reconstruct, dict(xq=cache()[0].to(torch.int8)), "xq must be a contiguous uint8"),
    (reconstruct, dict(scales=cache(bs=64)[1]), "scales must be a contiguous"),
    (reconstruct, dict(block_size=0), "block_size 0 does not divide D 64"),
    (reconstruct, dict(t0=ints(B)), "T is required with a tensor t0"),
    (reconstruct, dict(t0=ints(B, dtype=torch.int64), T=T), "t0 must be a contiguous"),
    (reconstruct, dict(T=2 ** 31), "T 2147483648 does not fit 32 bits"),
    (reconstruct, dict(dtype=torch.float32), "dtype must be fp16 or bf16"),
    (reconstruct, dict(y=x(t=S, dtype=torch.float32)), "y must be fp16 or bf16"),
    (reconstruct, dict(y=x(t=S - 1)), "y must be a contiguous"),
    (reconstruct, dict(y=x(t=2 * S)[:, :, ::2]), "y must be a contiguous"),
    # decode
    (decode, dict(q=torch.zeros((B, HQ, D))), "q must be fp16 or bf16"),
    (decode, dict(q=torch.zeros((B, HQ, D, 1), dtype=F16)), r"q must be \[B, H_q, D\]"),
    (decode, dict(q=torch.zeros((B, HQ, 2 * D), dtype=F16)), "q must be a contiguous"),
    (decode, dict(q=torch.zeros((B + 1, HQ, D), dtype=F16)), "q must be a contiguous"),
    (decode, dict(q=torch.zeros((B, D, HQ), dtype=F16).transpose(1, 2)), "q must be a contiguous"),
    (decode, dict(q=torch.zeros((B, 3, D), dtype=F16)), "H_q 3 is not a multiple of H_kv 2"),
    (decode, dict(kq=cache()[0].to(torch.int8)), "kq must be a contiguous uint8"),
    (decode, dict(ks=cache(bs=64)[1]), "ks must be a contiguous"),
    (decode, dict(vq=cache(S - 1)[0]), "vq must be a contiguous"),
    (decode, dict(vq=None), "vq is required"),
    (decode, dict(vs=cache(S - 1)[1]), "vs must be a contiguous"),
    (decode, dict(vs=cache()[1].to(BF16)), "vs must be a contiguous"),
    (decode, dict(lengths=ints(B, dtype=torch.int64)), "lengths must be a contiguous"),
    (decode, dict(lengths=ints(B + 1)), "lengths must be a contiguous"),
    (decode, dict(lengths=ints(2 * B)[::2]), "lengths must be a contiguous"),
    (decode, dict(lengths=far(B, dtype=I32)), "lengths must be a contiguous"),
    (decode, dict(S=2 ** 31), "S 2147483648 does not fit 32 bits"),
    (decode, dict(out=torch.zeros((B, HQ, D), dtype=BF16)), "out must be a contiguous"),
    (decode, dict(out=torch.zeros((B, HQ + 1, D), dtype=F16)), "out must be a contiguous"),
    (decode, dict(block_size=48), "block_size 48 does not divide D 64"),
    # norms and rotation, alone and with the cache
    *[(f, kw, m) for f in (rope, rope_append) for kw, m in (
        (dict(q=x(HQ, dtype=torch.float32)), ".* must be (fp16 or bf16|a torch.float32)"),
        (dict(q=x(HQ)[0]), r"q must be a .* tensor \[B, H, T, D\]"),
        (dict(q=torch.zeros((B, HQ, T, D + 4), dtype=F16)[..., :D]), "q: strides must be multiples of 8"),
        (dict(table=torch.zeros((9, D // 2))), r"table must be float32 \[max_pos"),
        (dict(table=torch.zeros((9, D // 2, 2), dtype=F16)), "table must be a contiguous"),
        (dict(table=torch.zeros((9, D // 2, 3))), "table must be a contiguous"),
        (dict(positions=ints(B, T, dtype=torch.int64)), "positions must be a contiguous"),
        (dict(positions=ints(B, T + 1)), "positions must be a contiguous"),
        (dict(positions=ints(T, B).T), "positions must be a contiguous"),
        (dict(positions=ints(1, T).expand(B, T)), "positions must be a contiguous"),
        (dict(sections=(16, 16)), "positions must be a contiguous"),
        (dict(sections=(16, 15), positions=ints(2, B, T)), "sections .* 1 to 4 counts that sum to 32"),
        (dict(sections=(33, -1), positions=ints(2, B, T)), "sections .* 1 to 4 counts that sum to 32"),
        (dict(sections=(8, 8, 8, 4, 4), positions=ints(5, B, T)), "sections .* 1 to 4 counts that sum to 32"),
        (dict(sections=(), positions=ints(0, B, T)), "sections .* 1 to 4 counts that sum to 32"),
        (dict(table=torch.zeros((2 ** 31, 0, 2))), "max_pos 2147483648 does not fit 32 bits"),
        (dict(q_weight=torch.zeros(D)), "q_weight must be a contiguous"),
        (dict(k_weight=torch.zeros(D // 2, dtype=F16)), "k_weight must be a contiguous"),
        (dict(q_out=x(H)), "q_out must be a contiguous"),
        (dict(q_out=x(HQ, dtype=BF16)), "q_out must be a contiguous"),
    )],
    (rope, dict(k=x(t=T + 1)), "does not match q"),
    (rope, dict(k=x(d=128)), "does not match q"),
    (rope, dict(k=x(b=1)), "does not match q"),
    (rope, dict(k=x(dtype=BF16)), "k must be a torch.float16 tensor"),
    (rope, dict(k=gaps), "k: the last dimension must be adjacent"),
    (rope, dict(k_out=x(HQ)), "k_out must be a contiguous"),
    (rope_append, dict(v=x(HQ)), "^v .* does not match k"),
    (rope_append, dict(k=x(1)), "^v .* does not match k"),
    (rope_append, dict(v=x(dtype=BF16)), "v must be a torch.float16 tensor"),
    (rope_append, dict(v=odd), "v: strides must be multiples of 8"),
    (rope_append, dict(k=x(1), v=x(1)), "^kq .* does not match k"),
    (rope_append, dict(kq=cache()[0].to(torch.int8)), "kq must be a contiguous uint8"),
    (rope_append, dict(ks=cache(bs=64)[1]), "ks must be a contiguous"),
    (rope_append, dict(vq=cache(S - 1)[0]), "vq must be a contiguous"),
    (rope_append, dict(vs=cache(S - 1)[1]), "vs must be a contiguous"),
    (rope_append, dict(block_size=48), "block_size 48 does not divide D 64"),
    (rope_append, dict(t0=ints(B + 1)), "t0 must be a contiguous"),
    (rope_append, dict(t0=-2 ** 31 - 1), "t0 -2147483649 does not fit 32 bits"),
]


@pytest.mark.parametrize("f,kw,message", REFUSED, ids=[f"{f.__name__}-{i}" for i, (f, *_) in enumerate(REFUSED)])
def test_what_does_not_fit_is_refused_by_its_check(calls, f, kw, message):
    with pytest.raises(ValueError, match=message):
        f(**kw)
    assert calls == []


def test_tensors_on_the_host_are_refused(monkeypatch):
    for f in (append, compress, reconstruct, decode, rope, rope_append):
        with pytest.raises(ValueError, match="must be on a CUDA device"):
            f()


def test_a_stream_of_another_device_is_refused(calls):
    stream = types.SimpleNamespace(device=torch.device("cuda", 1))
    for f in (append, compress, reconstruct, decode, rope, rope_append):
        with pytest.raises(ValueError, match="stream is on cuda:1"):
            f(stream=stream)
    assert calls == []
