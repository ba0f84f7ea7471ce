"""The KV cache in 4 bits, for torch tensors (C ABI: include/tqkv.h).

    q, o            fp16 or bf16 [B, H_q, D]
    x, k, v         fp16 or bf16 [B, H, T, D], any strides that are multiples of 8, D adjacent
    kq, vq          uint8 [B, H, S_cap, D // 2], packed codes
    ks, vs          fp16 [B, H, S_cap, D // block_size, 2], (scale, zero) of each block

All tensors of a call are on one device, which need not be the current one, and
the call launches on that device's current torch stream (or `stream=`).  A
first row `t0` is an int for all sequences or an int32 tensor [B] on the
device, with which rows outside the cache are not written and read as 0.
Errors raise ValueError or TqkvError before anything is launched.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence, Tuple, Union

import torch

from ._lib import NormRopeArgs, check, load
from .ops import Workspace

_DTYPES = {torch.float16: 0, torch.bfloat16: 1}
_L3 = ctypes.c_longlong * 3


class _Launch:
    """The device and stream of a call: enters the device, gives the stream's handle, and tells
    torch's allocator about tensors that another stream than the current one uses."""

    __slots__ = ("guard", "handle", "other")

    def __init__(self, device: torch.device, stream):
        if device.type != "cuda":
            raise ValueError("tensors must be on a CUDA device")
        if stream is not None and stream.device != device:
            raise ValueError(f"stream is on {stream.device}, tensors are on {device}")
        self.guard = None if torch.cuda.current_device() == device.index \
            else torch.cuda.device(device)
        self.other = None
        if stream is None:
            self.handle = torch._C._cuda_getCurrentRawStream(device.index)
        else:
            self.handle = stream.cuda_stream
            if self.handle != torch._C._cuda_getCurrentRawStream(device.index):
                self.other = stream

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()
        return self

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)

    def used(self, *tensors) -> None:
        if self.other is not None and not torch.cuda.is_current_stream_capturing():
            for t in tensors:
                if t is not None:
                    t.record_stream(self.other)


def _dtype(t: torch.Tensor, name: str) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"{name} must be fp16 or bf16, got {t.dtype}")
    return code


def _is(t: Optional[torch.Tensor], name: str, shape: tuple, dtype: torch.dtype,
        device: torch.device) -> int:
    """The address of a contiguous tensor of exactly this shape, type and device."""
    if t is None:
        raise ValueError(f"{name} is required")
    if t.shape != shape or t.dtype != dtype or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor {shape} on {device}, got "
                         f"{t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _rows(x: torch.Tensor, name: str, dtype: torch.dtype, device: torch.device):
    """(shape, strides of the first three dimensions) of x [B, H, T, D]."""
    if x.dim() != 4 or x.dtype != dtype or x.device != device:
        raise ValueError(f"{name} must be a {dtype} tensor [B, H, T, D] on {device}, got "
                         f"{x.dtype} {tuple(x.shape)} on {x.device}")
    shape, st = x.shape, x.stride()
    if st[3] != 1 and shape[3] != 1:
        raise ValueError(f"{name}: the last dimension must be adjacent in memory")
    # the stride of a dimension of one element means nothing
    strides = tuple(0 if n == 1 else s for n, s in zip(shape[:3], st))
    if strides[0] % 8 or strides[1] % 8 or strides[2] % 8:
        raise ValueError(f"{name}: strides must be multiples of 8 elements, got {tuple(st)}")
    return shape, strides


def _cache(q: torch.Tensor, s: torch.Tensor, qn: str, sn: str, block_size: int,
           device: torch.device) -> Tuple[int, int, int, int]:
    """(B, H, S_cap, D) of a cache's codes and scales."""
    if q.dim() != 4:
        raise ValueError(f"{qn} must be uint8 [B, H, S_cap, D // 2]")
    B, H, S, half = q.shape
    _is(q, qn, (B, H, S, half), torch.uint8, device)
    D = 2 * half
    if block_size <= 0 or D % block_size:
        raise ValueError(f"block_size {block_size} does not divide D {D}")
    _is(s, sn, (B, H, S, D // block_size, 2), torch.float16, device)
    return B, H, S, D


def _starts(t0: Union[int, torch.Tensor], B: int, device: torch.device):
    """(address of the per-sequence first rows or None, first row of all)."""
    if isinstance(t0, torch.Tensor):
        return _is(t0, "t0", (B,), torch.int32, device), 0
    return None, int(t0)


def _bound(**sizes: int) -> None:
    for name, n in sizes.items():
        if n > 0x7fffffff:
            raise ValueError(f"{name} = {n} does not fit 32 bits")


def kv_compress_int4(x: torch.Tensor, block_size: int, xq: Optional[torch.Tensor] = None,
                     scales: Optional[torch.Tensor] = None, stream=None):
    """fp16 or bf16 [B, H, S, D] -> (codes uint8 [B, H, S, D // 2], scales fp16
    [B, H, S, D // block_size, 2])."""
    if x.dim() != 4:
        raise ValueError("x must be [B, H, S, D]")
    B, H, S, D = x.shape
    if block_size <= 0 or D % block_size or D % 2:
        raise ValueError(f"block_size {block_size} does not divide D {D}")
    if xq is None:
        xq = torch.empty((B, H, S, D // 2), dtype=torch.uint8, device=x.device)
    if scales is None:
        scales = torch.empty((B, H, S, D // block_size, 2), dtype=torch.float16, device=x.device)
    kv_append_int4(x, xq, scales, 0, block_size, stream=stream)
    return xq, scales


def kv_append_int4(x: torch.Tensor, cache_q: torch.Tensor, cache_s: torch.Tensor,
                   t0: Union[int, torch.Tensor], block_size: int, stream=None) -> None:
    """Quantise T tokens per head, x [B, H, T, D], into rows [t0, t0 + T) of a 4-bit cache."""
    device = x.device
    dt = _dtype(x, "x")
    shape, strides = _rows(x, "x", x.dtype, device)
    B, H, S_cap, D = _cache(cache_q, cache_s, "cache_q", "cache_s", block_size, device)
    if (B, H, D) != (shape[0], shape[1], shape[3]):
        raise ValueError(f"cache_q {tuple(cache_q.shape)} does not match x {tuple(shape)}")
    _bound(S_cap=S_cap)
    starts, first = _starts(t0, B, device)
    with _Launch(device, stream) as on:
        check("tqkv_kv_append_int4", load().tqkv_kv_append_int4(
            x.data_ptr(), _L3(*strides), cache_q.data_ptr(), cache_s.data_ptr(), starts, first,
            B, H, shape[2], D, block_size, S_cap, dt, on.handle))
        on.used(x, cache_q, cache_s, t0 if starts else None)


def kv_reconstruct_int4(xq: torch.Tensor, scales: torch.Tensor, block_size: int,
                        y: Optional[torch.Tensor] = None, t0: Union[int, torch.Tensor] = 0,
                        T: Optional[int] = None, dtype: torch.dtype = torch.float16,
                        stream=None) -> torch.Tensor:
    """The values of rows [t0, t0 + T) of a 4-bit cache (all of them by default): [B, H, T, D] in
    `dtype`, or in y's."""
    device = xq.device
    B, H, S_cap, D = _cache(xq, scales, "xq", "scales", block_size, device)
    if T is None:
        if isinstance(t0, torch.Tensor):
            raise ValueError("T is required with a tensor t0")
        T = S_cap - t0
    _bound(S_cap=S_cap)
    starts, first = _starts(t0, B, device)
    with _Launch(device, stream) as on:
        if y is None:
            y = torch.empty((B, H, max(T, 0), D), dtype=dtype, device=device)
        dt = _dtype(y, "y")
        _is(y, "y", (B, H, T, D), y.dtype, device)
        check("tqkv_kv_reconstruct_int4", load().tqkv_kv_reconstruct_int4(
            xq.data_ptr(), scales.data_ptr(), y.data_ptr(), starts, first, B, H, T, D, block_size,
            S_cap, dt, on.handle))
        on.used(xq, scales, y, t0 if starts else None)
    return y


_default_ws: dict = {}
_ws_bytes: dict = {}


def _workspace(ws: Optional[Workspace], device: torch.device, handle: int, stream, key):
    """(address, bytes, tensor to keep) of the scratch for a decode of sizes `key`.  Without a
    Workspace of the caller's, every stream has its own; a call that is being captured gets its own
    buffer from the graph's memory, zeroed by the graph, so that graphs may replay side by side."""
    need = _ws_bytes.get((device.index, key))
    if need is None:
        need = int(load().tqkv_decode_int4_workspace_bytes(*key))
        if len(_ws_bytes) < 4096:
            _ws_bytes[(device.index, key)] = need
    if need == 0:
        return None, 0, None
    if ws is not None and ws.device.index not in (None, device.index):
        raise ValueError(f"workspace is on {ws.device}, tensors are on {device}")
    big_enough = ws is not None and ws.buf is not None and ws.buf.numel() >= need
    if big_enough:
        return ws.buf.data_ptr(), ws.buf.numel(), ws.buf
    if torch.cuda.is_current_stream_capturing():
        if ws is not None:
            raise ValueError("a Workspace cannot grow while a graph is captured: call once before "
                             "the capture, or leave the workspace to the call")
        buf = torch.empty(need, dtype=torch.uint8, device=device)
        check("tqkv_workspace_init", load().tqkv_workspace_init(buf.data_ptr(), need, handle))
        return buf.data_ptr(), need, buf
    if ws is None:
        ws = _default_ws.get((device.index, handle))
        if ws is None:
            ws = _default_ws[(device.index, handle)] = Workspace(device)
    ptr, size = ws.get(need, stream)
    return ptr, size, ws.buf


def decode_int4(q: torch.Tensor, kq: torch.Tensor, ks: torch.Tensor, vq: torch.Tensor,
                vs: torch.Tensor, block_size: int, S: Optional[int] = None,
                lengths: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                workspace: Optional[Workspace] = None, stream=None) -> torch.Tensor:
    """Decode attention over a 4-bit cache -> O [B, H_q, D] in q's type.

    q [B, H_q, D]; caches with H_kv heads, H_q a multiple of H_kv.  Sequence b attends over its
    first lengths[b] rows (int32 [B] on the device, taken into [0, S]), or over S rows; S defaults
    to the cache's.  A sequence without rows gives zeros."""
    device = q.device
    dt = _dtype(q, "q")
    if q.dim() != 3:
        raise ValueError("q must be [B, H_q, D]")
    B, H_kv, S_cap, D = _cache(kq, ks, "kq", "ks", block_size, device)
    _is(vq, "vq", kq.shape, torch.uint8, device)
    _is(vs, "vs", ks.shape, torch.float16, device)
    H_q = q.shape[1]
    _is(q, "q", (B, H_q, D), q.dtype, device)
    if S is None:
        S = S_cap
    _bound(S_cap=S_cap, S=S)
    if H_kv == 0 or H_q % H_kv:
        raise ValueError(f"H_q {H_q} is not a multiple of H_kv {H_kv}")
    n = None if lengths is None else _is(lengths, "lengths", (B,), torch.int32, device)
    with _Launch(device, stream) as on:
        if out is None:
            out = torch.empty((B, H_q, D), dtype=q.dtype, device=device)
        else:
            _is(out, "out", (B, H_q, D), q.dtype, device)
        ptr, size, buf = _workspace(workspace, device, on.handle, stream, (B, H_q, H_kv, S, D))
        check("tqkv_decode_int4", load().tqkv_decode_int4(
            q.data_ptr(), kq.data_ptr(), ks.data_ptr(), vq.data_ptr(), vs.data_ptr(), n,
            out.data_ptr(), B, H_q, H_kv, S, S_cap, D, block_size, dt, ptr, size, on.handle))
        on.used(q, kq, ks, vq, vs, lengths, out, buf)
    return out


def rope_table(max_pos: int, rot_dim: int, base: float = 10000.0, device=None) -> torch.Tensor:
    """fp32 [max_pos, rot_dim // 2, 2]: (cos, sin) of position * base ** (-2 j / rot_dim), the
    angles in 64 bits.  A table of any other frequencies serves as well."""
    if max_pos <= 0 or rot_dim <= 0 or rot_dim % 16:
        raise ValueError("max_pos must be positive and rot_dim a positive multiple of 16")
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else device
    j = torch.arange(rot_dim // 2, dtype=torch.float64, device=device)
    p = torch.arange(max_pos, dtype=torch.float64, device=device)
    angle = p[:, None] * base ** (-2.0 * j / rot_dim)
    return torch.stack((angle.cos(), angle.sin()), -1).float()


def _norm_rope(q, k, positions, table, q_weight, k_weight, eps, interleaved, sections):
    """The arguments that both forms share, and (B, H_q, H_kv, T, D)."""
    device = q.device
    a = NormRopeArgs()
    a.dtype = _dtype(q, "q")
    (B, H_q, T, D), qs = _rows(q, "q", q.dtype, device)
    (Bk, H_kv, Tk, Dk), kst = _rows(k, "k", q.dtype, device)
    if (Bk, Tk, Dk) != (B, T, D):
        raise ValueError(f"k {tuple(k.shape)} does not match q {tuple(q.shape)}")
    if table.dim() != 3:
        raise ValueError("table must be float32 [max_pos, rot_dim // 2, 2]")
    max_pos, pairs = table.shape[0], table.shape[1]
    a.table = _is(table, "table", (max_pos, pairs, 2), torch.float32, device)
    if sections is None:
        axes = 1
        a.positions = _is(positions, "positions", (B, T), torch.int32, device)
    else:
        axes = len(sections)
        if not 1 <= axes <= 4 or sum(sections) != pairs or min(sections) < 0:
            raise ValueError(f"sections {tuple(sections)}: 1 to 4 counts that sum to {pairs}")
        a.positions = _is(positions, "positions", (axes, B, T), torch.int32, device)
        a.sections[:axes] = list(sections)
    for w, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if w is not None:
            setattr(a, name, _is(w, name, (D,), q.dtype, device))
    _bound(max_pos=max_pos)
    a.q, a.k = q.data_ptr(), k.data_ptr()
    a.q_strides[:], a.k_strides[:] = qs, kst
    a.eps = eps
    a.B, a.H_q, a.H_kv, a.T, a.D = B, H_q, H_kv, T, D
    a.rot_dim, a.max_pos, a.interleaved, a.axes = 2 * pairs, max_pos, bool(interleaved), axes
    return a, (B, H_q, H_kv, T, D)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, table: torch.Tensor,
                 q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                 eps: float = 1e-6, interleaved: bool = False,
                 sections: Optional[Sequence[int]] = None, q_out: Optional[torch.Tensor] = None,
                 k_out: Optional[torch.Tensor] = None, stream=None):
    """Head norms and position rotation: q [B, H_q, T, D] and k [B, H_kv, T, D] (views of one
    projection will do) -> contiguous (q, k).

    y = x * rsqrt(mean(x^2) + eps) * weight over each head; then each pair (a, b) of the first
    rot_dim = 2 * table.shape[1] elements becomes (a cos - b sin, b cos + a sin).  Pairs are (j, j +
    rot_dim / 2), or (2 j, 2 j + 1) if `interleaved`.  positions: int32 [B, T], or [axes, B, T] with
    `sections`, the number of pairs that follow each axis.  A position outside the table gives
    NaN."""
    device = q.device
    a, (B, H_q, H_kv, T, D) = _norm_rope(q, k, positions, table, q_weight, k_weight, eps,
                                         interleaved, sections)
    with _Launch(device, stream) as on:
        if q_out is None:
            q_out = torch.empty((B, H_q, T, D), dtype=q.dtype, device=device)
        if k_out is None:
            k_out = torch.empty((B, H_kv, T, D), dtype=q.dtype, device=device)
        a.q_out = _is(q_out, "q_out", (B, H_q, T, D), q.dtype, device)
        a.k_out = _is(k_out, "k_out", (B, H_kv, T, D), q.dtype, device)
        check("tqkv_qk_norm_rope", load().tqkv_qk_norm_rope(ctypes.byref(a), on.handle))
        on.used(q, k, positions, table, q_weight, k_weight, q_out, k_out)
    return q_out, k_out


def qk_norm_rope_append_int4(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                             positions: torch.Tensor, table: torch.Tensor, kq: torch.Tensor,
                             ks: torch.Tensor, vq: torch.Tensor, vs: torch.Tensor,
                             t0: Union[int, torch.Tensor], block_size: int,
                             q_weight: Optional[torch.Tensor] = None,
                             k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                             interleaved: bool = False, sections: Optional[Sequence[int]] = None,
                             q_out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """qk_norm_rope with K and V [B, H_kv, T, D] written straight into rows [t0, t0 + T) of their
    4-bit caches, in one launch; returns q [B, H_q, T, D].  K is quantised from fp32, without the
    rounding to its type that qk_norm_rope followed by kv_append_int4 has."""
    device = q.device
    a, (B, H_q, H_kv, T, D) = _norm_rope(q, k, positions, table, q_weight, k_weight, eps,
                                         interleaved, sections)
    shape, vst = _rows(v, "v", q.dtype, device)
    if shape != k.shape:
        raise ValueError(f"v {tuple(shape)} does not match k {tuple(k.shape)}")
    Bc, Hc, S_cap, Dc = _cache(kq, ks, "kq", "ks", block_size, device)
    if (Bc, Hc, Dc) != (B, H_kv, D):
        raise ValueError(f"kq {tuple(kq.shape)} does not match k {tuple(k.shape)}")
    _is(vq, "vq", kq.shape, torch.uint8, device)
    _is(vs, "vs", ks.shape, torch.float16, device)
    _bound(S_cap=S_cap)
    starts, a.t0 = _starts(t0, B, device)
    a.starts = starts
    a.v, a.v_strides[:] = v.data_ptr(), vst
    a.kq, a.ks, a.vq, a.vs = kq.data_ptr(), ks.data_ptr(), vq.data_ptr(), vs.data_ptr()
    a.block_size, a.S_cap = block_size, S_cap
    with _Launch(device, stream) as on:
        if q_out is None:
            q_out = torch.empty((B, H_q, T, D), dtype=q.dtype, device=device)
        a.q_out = _is(q_out, "q_out", (B, H_q, T, D), q.dtype, device)
        check("tqkv_qk_norm_rope_append_int4",
              load().tqkv_qk_norm_rope_append_int4(ctypes.byref(a), on.handle))
        on.used(q, k, v, positions, table, kq, ks, vq, vs, t0 if starts else None, q_weight,
                k_weight, q_out)
    return q_out
