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

from ._lib import NORM_ROPE_PACK, TqkvError, check, load
from .ops import Workspace

_F16 = torch.float16
_U8 = torch.uint8
_DTYPES = {torch.float16: 0, torch.bfloat16: 1}
_L3 = ctypes.c_longlong * 3
_current_device = torch._C._cuda_getDevice
_current_stream = torch._C._cuda_getCurrentRawStream

# A decode step of a served model makes a few of these calls per layer, each
# shorter on the GPU than a careless wrapper is on the host.  So the checks
# below ask each tensor for as little as possible, once.


def _device(t: torch.Tensor, name: str) -> int:
    """The index of t's CUDA device."""
    index = t.get_device()
    if index < 0:
        raise ValueError(f"{name} must be on a CUDA device")
    return index


def _elsewhere(fn, index: int, stream, *args, **kwargs):
    """The call where it does not run on the current device and stream: enters them, so that what
    it allocates belongs to that stream, and tells torch's allocator that the stream uses the
    arguments.  The caller orders the streams, as for any torch operation."""
    if stream is None:
        with torch.cuda.device(index):
            return fn(*args, **kwargs)
    if stream.device.index != index:
        raise ValueError(f"stream is on {stream.device}, tensors are on cuda:{index}")
    with torch.cuda.stream(stream):
        out = fn(*args, **kwargs)
        if not torch.cuda.is_current_stream_capturing():
            for t in (*args, *kwargs.values()):
                if isinstance(t, Workspace):
                    t = t.buf
                if isinstance(t, torch.Tensor):
                    t.record_stream(stream)
    return out


def _dtype(t: torch.Tensor, name: str) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"{name} must be fp16 or bf16, got {t.dtype}")
    return code


def _is(t: Optional[torch.Tensor], name: str, shape: tuple, dtype: torch.dtype, index: int) -> int:
    """The address of a contiguous tensor of exactly this shape, type and device."""
    if t is None:
        raise ValueError(f"{name} is required")
    if t.dtype is not dtype or t.get_device() != index or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor {tuple(shape)} on "
                         f"cuda:{index}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _rows(x: torch.Tensor, name: str, dtype: torch.dtype, index: int):
    """(shape, strides of the first three dimensions) of x [B, H, T, D]."""
    if x.dtype is not dtype or x.get_device() != index or x.dim() != 4:
        raise ValueError(f"{name} must be a {dtype} tensor [B, H, T, D] on cuda:{index}, got "
                         f"{x.dtype} {tuple(x.shape)} on {x.device}")
    shape = x.shape
    sb, sh, st, sd = x.stride()
    if sd != 1 and shape[3] != 1:
        raise ValueError(f"{name}: the last dimension must be adjacent in memory")
    if (sb | sh | st) & 7:
        # the stride of a dimension of one element means nothing
        sb, sh, st = (0 if n == 1 else s for n, s in zip(shape, (sb, sh, st)))
        if (sb | sh | st) & 7:
            raise ValueError(f"{name}: strides must be multiples of 8 elements, got {x.stride()}")
    return shape, (sb, sh, st)


def _cache(q: torch.Tensor, s: torch.Tensor, qn: str, sn: str, block_size: int, index: int):
    """(codes' shape, D, scales' shape) of a cache."""
    if q.dtype is not _U8 or q.get_device() != index or q.dim() != 4 or not q.is_contiguous():
        raise ValueError(f"{qn} must be a contiguous uint8 tensor [B, H, S_cap, D // 2] on "
                         f"cuda:{index}, got {q.dtype} {tuple(q.shape)} on {q.device}")
    shape = q.shape
    B, H, S, half = shape
    D = 2 * half
    if block_size <= 0 or D % block_size:
        raise ValueError(f"block_size {block_size} does not divide D {D}")
    if S > 0x7fffffff:
        raise ValueError(f"S_cap {S} does not fit 32 bits")
    params = (B, H, S, D // block_size, 2)
    _is(s, sn, params, _F16, index)
    return shape, D, params


def _fits(n: int, name: str) -> int:
    if not -0x80000000 <= n <= 0x7fffffff:
        raise ValueError(f"{name} {n} does not fit 32 bits")
    return n


def _starts(t0: Union[int, torch.Tensor], B: int, index: int):
    """(address of the per-sequence first rows or None, first row of all)."""
    if isinstance(t0, torch.Tensor):
        return _is(t0, "t0", (B,), torch.int32, index), 0
    return None, _fits(t0, "t0")


def kv_compress_int4(x: torch.Tensor, block_size: int, xq: Optional[torch.Tensor] = None,
                     scales: Optional[torch.Tensor] = None, stream=None):
    """fp16 or bf16 [B, H, S, D] -> (codes uint8 [B, H, S, D // 2], scales fp16
    [B, H, S, D // block_size, 2])."""
    index = _device(x, "x")
    if stream is not None:
        return _elsewhere(kv_compress_int4, index, stream, x, block_size, xq, scales)
    if x.dim() != 4:
        raise ValueError("x must be [B, H, S, D]")
    B, H, S, D = x.shape
    if block_size <= 0 or D % block_size or D % 2:
        raise ValueError(f"block_size {block_size} does not divide D {D}")
    if xq is None:
        xq = torch.empty((B, H, S, D // 2), dtype=torch.uint8, device=x.device)
    if scales is None:
        scales = torch.empty((B, H, S, D // block_size, 2), dtype=_F16, device=x.device)
    if xq.dim() != 4 or xq.shape[2] != S:
        raise ValueError(f"xq {tuple(xq.shape)} does not have x's {S} rows")
    kv_append_int4(x, xq, scales, 0, block_size)
    return xq, scales


def kv_append_int4(x: torch.Tensor, cache_q: torch.Tensor, cache_s: torch.Tensor,
                   t0: Union[int, torch.Tensor], block_size: int, stream=None) -> None:
    """Quantise T tokens per head, x [B, H, T, D], into rows [t0, t0 + T) of a 4-bit cache."""
    index = _device(x, "x")
    if stream is not None or _current_device() != index:
        return _elsewhere(kv_append_int4, index, stream, x, cache_q, cache_s, t0, block_size)
    dt = _dtype(x, "x")
    (Bx, Hx, T, Dx), strides = _rows(x, "x", x.dtype, index)
    (B, H, S_cap, _), D, _ = _cache(cache_q, cache_s, "cache_q", "cache_s", block_size, index)
    if B != Bx or H != Hx or D != Dx or T > S_cap:
        raise ValueError(f"cache_q {tuple(cache_q.shape)} does not match x {tuple(x.shape)}")
    starts, first = _starts(t0, B, index)
    status = load().tqkv_kv_append_int4(
        x.data_ptr(), _L3(*strides), cache_q.data_ptr(), cache_s.data_ptr(), starts, first, B, H, T,
        D, block_size, S_cap, dt, _current_stream(index))
    if status:
        raise TqkvError("tqkv_kv_append_int4", status)


def kv_reconstruct_int4(xq: torch.Tensor, scales: torch.Tensor, block_size: int,
                        y: Optional[torch.Tensor] = None, t0: Union[int, torch.Tensor] = 0,
                        T: Optional[int] = None, dtype: torch.dtype = torch.float16,
                        stream=None) -> torch.Tensor:
    """The values of rows [t0, t0 + T) of a 4-bit cache (all of them by default): [B, H, T, D] in
    `dtype`, or in y's."""
    index = _device(xq, "xq")
    if stream is not None or _current_device() != index:
        return _elsewhere(kv_reconstruct_int4, index, stream, xq, scales, block_size, y, t0, T, dtype)
    (B, H, S_cap, _), D, _ = _cache(xq, scales, "xq", "scales", block_size, index)
    starts, first = _starts(t0, B, index)
    if T is None:
        if starts is not None:
            raise ValueError("T is required with a tensor t0")
        T = S_cap - first
    _fits(T, "T")
    if y is None:
        # scales is fp16 on the right device: the cheapest way to a tensor like it
        y = scales.new_empty((B, H, T if T > 0 else 0, D)) if dtype is _F16 else \
            scales.new_empty((B, H, T if T > 0 else 0, D), dtype=dtype)
        dt = _dtype(y, "dtype")
    else:
        dt = _dtype(y, "y")
        _is(y, "y", (B, H, T, D), y.dtype, index)
    status = load().tqkv_kv_reconstruct_int4(
        xq.data_ptr(), scales.data_ptr(), y.data_ptr(), starts, first, B, H, T, D, block_size,
        S_cap, dt, _current_stream(index))
    if status:
        raise TqkvError("tqkv_kv_reconstruct_int4", status)
    return y


_default_ws: dict = {}
_ws_bytes: dict = {}


def _workspace(ws: Optional[Workspace], index: int, handle: int, key):
    """(address, bytes) of the scratch for a decode of sizes `key`.  Without a Workspace of the
    caller's, every stream has its own; a call that is being captured gets its own buffer from the
    graph's memory, zeroed by the graph, so that graphs may replay side by side."""
    need = _ws_bytes.get((index, key))
    if need is None:
        need = int(load().tqkv_decode_int4_workspace_bytes(*key))
        if len(_ws_bytes) < 4096:
            _ws_bytes[(index, key)] = need
    if need == 0:
        return None, 0
    if ws is not None:
        ws.check_device(index)
        buf = ws.buf
        if buf is not None and buf.numel() >= need:
            return buf.data_ptr(), buf.numel()
    if torch.cuda.is_current_stream_capturing():
        if ws is not None:
            raise ValueError("a Workspace cannot grow while a graph is captured: call once before "
                             "the capture, or leave the workspace to the call")
        buf = torch.empty(need, dtype=torch.uint8, device=torch.device("cuda", index))
        # only the counters in front (4 bytes a CTA) have to be zero: no INT8 call uses this buffer
        check("tqkv_workspace_init",
              load().tqkv_workspace_init(buf.data_ptr(), min(need, 16384), handle))
        return buf.data_ptr(), need
    if ws is None:
        ws = _default_ws.get((index, handle))
        if ws is None:
            ws = _default_ws.setdefault((index, handle), Workspace(torch.device("cuda", index)))
    return ws.get(need)


def decode_int4(q: torch.Tensor, kq: torch.Tensor, ks: torch.Tensor, vq: torch.Tensor,
                vs: torch.Tensor, block_size: int, S: Optional[int] = None,
                lengths: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                workspace: Optional[Workspace] = None, stream=None) -> torch.Tensor:
    """Decode attention over a 4-bit cache -> O [B, H_q, D] in q's type.

    q [B, H_q, D]; caches with H_kv heads, H_q a multiple of H_kv.  Sequence b attends over its
    first lengths[b] rows (int32 [B] on the device, taken into [0, S]), or over S rows; S defaults
    to the cache's.  A sequence without rows gives zeros."""
    index = _device(q, "q")
    if stream is not None or _current_device() != index:
        return _elsewhere(decode_int4, index, stream, q, kq, ks, vq, vs, block_size, S, lengths, out,
                          workspace)
    dt = _dtype(q, "q")
    shape, D, params = _cache(kq, ks, "kq", "ks", block_size, index)
    B, H_kv, S_cap, _ = shape
    v_ptr = _is(vq, "vq", shape, _U8, index)
    vs_ptr = _is(vs, "vs", params, _F16, index)
    if q.dim() != 3:
        raise ValueError("q must be [B, H_q, D]")
    H_q = q.shape[1]
    q_ptr = _is(q, "q", (B, H_q, D), q.dtype, index)
    if S is None:
        S = S_cap
    else:
        _fits(S, "S")
    if H_kv == 0 or H_q % H_kv:
        raise ValueError(f"H_q {H_q} is not a multiple of H_kv {H_kv}")
    n = None if lengths is None else _is(lengths, "lengths", (B,), torch.int32, index)
    if out is None:
        out = torch.empty_like(q)
    else:
        _is(out, "out", (B, H_q, D), q.dtype, index)
    handle = _current_stream(index)
    ptr, size = _workspace(workspace, index, handle, (B, H_q, H_kv, S, D))
    status = load().tqkv_decode_int4(
        q_ptr, kq.data_ptr(), ks.data_ptr(), v_ptr, vs_ptr, n, out.data_ptr(), B, H_q, H_kv, S,
        S_cap, D, block_size, dt, ptr, size, handle)
    if status:
        raise TqkvError("tqkv_decode_int4", status)
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


_NO_CACHE = (0, 0, 0), 0, 0, 0, 0, 0, 0, 0, 0, 0   # v's strides, v, caches, starts, t0, block, S_cap


def _pack(index, q, k, positions, table, q_weight, k_weight, eps, interleaved, sections, q_out, k_out,
          append=_NO_CACHE) -> bytes:
    """tqkv_norm_rope_args (include/tqkv.h) after the checks that both forms share."""
    dt = _dtype(q, "q")
    dtype = q.dtype
    (B, H_q, T, D), qs = _rows(q, "q", dtype, index)
    (Bk, H_kv, Tk, Dk), kst = _rows(k, "k", dtype, index)
    if Bk != B or Tk != T or Dk != D:
        raise ValueError(f"k {tuple(k.shape)} does not match q {tuple(q.shape)}")
    if table.dim() != 3:
        raise ValueError("table must be float32 [max_pos, rot_dim // 2, 2]")
    max_pos, pairs, _ = table.shape
    if max_pos > 0x7fffffff:
        raise ValueError(f"max_pos {max_pos} does not fit 32 bits")
    t_ptr = _is(table, "table", (max_pos, pairs, 2), torch.float32, index)
    if sections is None:
        axes, counts = 1, (0, 0, 0, 0)
        pos = _is(positions, "positions", (B, T), torch.int32, index)
    else:
        axes = len(sections)
        if not 1 <= axes <= 4 or sum(sections) != pairs or min(sections) < 0:
            raise ValueError(f"sections {tuple(sections)}: 1 to 4 counts that sum to {pairs}")
        counts = (*sections, 0, 0, 0)[:4]
        pos = _is(positions, "positions", (axes, B, T), torch.int32, index)
    qw = 0 if q_weight is None else _is(q_weight, "q_weight", (D,), dtype, index)
    kw = 0 if k_weight is None else _is(k_weight, "k_weight", (D,), dtype, index)
    vst, v, kq, vq, ks, vs, starts, t0, block_size, S_cap = append
    return NORM_ROPE_PACK.pack(
        q.data_ptr(), k.data_ptr(), v, *qs, *kst, *vst, qw, kw, t_ptr, pos, q_out, k_out, kq, vq, ks,
        vs, starts, eps, t0, B, H_q, H_kv, T, D, block_size, S_cap, dt, 2 * pairs, max_pos,
        1 if interleaved else 0, axes, *counts)


def _new_rows(t: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor of t's shape, type and device."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


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
    NaN.  Outputs must not overlap the inputs."""
    index = _device(q, "q")
    if stream is not None or _current_device() != index:
        return _elsewhere(qk_norm_rope, index, stream, q, k, positions, table, q_weight, k_weight,
                          eps, interleaved, sections, q_out, k_out)
    if q_out is None:
        q_out = _new_rows(q)
    else:
        _is(q_out, "q_out", q.shape, q.dtype, index)
    if k_out is None:
        k_out = _new_rows(k)
    else:
        _is(k_out, "k_out", k.shape, q.dtype, index)
    args = _pack(index, q, k, positions, table, q_weight, k_weight, eps, interleaved, sections,
                 q_out.data_ptr(), k_out.data_ptr())
    status = load().tqkv_qk_norm_rope(args, _current_stream(index))
    if status:
        raise TqkvError("tqkv_qk_norm_rope", status)
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
    index = _device(q, "q")
    if stream is not None or _current_device() != index:
        return _elsewhere(qk_norm_rope_append_int4, index, stream, q, k, v, positions, table, kq, ks,
                          vq, vs, t0, block_size, q_weight, k_weight, eps, interleaved, sections,
                          q_out)
    v_shape, vst = _rows(v, "v", q.dtype, index)
    if v_shape != k.shape:
        raise ValueError(f"v {tuple(v_shape)} does not match k {tuple(k.shape)}")
    shape, D, params = _cache(kq, ks, "kq", "ks", block_size, index)
    B, H_kv, S_cap, _ = shape
    if B != v_shape[0] or H_kv != v_shape[1] or D != v_shape[3]:
        raise ValueError(f"kq {tuple(shape)} does not match k {tuple(k.shape)}")
    vq_ptr = _is(vq, "vq", shape, _U8, index)
    vs_ptr = _is(vs, "vs", params, _F16, index)
    starts, first = _starts(t0, B, index)
    if q_out is None:
        q_out = _new_rows(q)
    else:
        _is(q_out, "q_out", q.shape, q.dtype, index)
    args = _pack(index, q, k, positions, table, q_weight, k_weight, eps, interleaved, sections,
                 q_out.data_ptr(), 0, (vst, v.data_ptr(), kq.data_ptr(), vq_ptr, ks.data_ptr(), vs_ptr,
                                       starts or 0, first, block_size, S_cap))
    status = load().tqkv_qk_norm_rope_append_int4(args, _current_stream(index))
    if status:
        raise TqkvError("tqkv_qk_norm_rope_append_int4", status)
    return q_out
