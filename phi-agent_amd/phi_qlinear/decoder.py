"""The operators between a decoder layer's int8 linears (include/phi_decoder.h).

``rms_norm_quant`` turns the residual stream into the int8 operand of the
linear that follows, ``kv_cache_write`` / ``kv_cache_read`` keep keys and
values in an int8 paged cache, ``paged_attention`` attends over it.
"""
from __future__ import annotations

import ctypes
from operator import itemgetter

import torch

from . import (_DTYPES, F32, ROUND_HALF_AWAY, KvCacheDesc, _check, _dt, _ptr, _require_device, _stream, _ws, load)


def _empty(shape, dtype, like: torch.Tensor, stream) -> torch.Tensor:
    """A new tensor beside `like`, from the memory of the stream that will write it.
    (The sizes one by one: as a tuple they cost 0.8 us more.)"""
    if stream is None:
        return torch.empty(*shape, dtype=dtype, device=like.device)
    with torch.cuda.stream(stream):
        return torch.empty(*shape, dtype=dtype, device=like.device)


def _row_pitch(name: str, t: torch.Tensor, shape) -> int:
    """The pitch of a [rows, K] tensor with contiguous rows (of one row: any from K on)."""
    if t.shape == shape and t.is_contiguous():
        return shape[1]
    if t.shape != shape:
        raise ValueError(f"rms_norm_quant: {name} is {tuple(t.shape)}, not {tuple(shape)}")
    pitch, step = t.stride()
    if step != 1 and shape[1] > 1 and shape[0] > 0:
        raise ValueError(f"rms_norm_quant: {name}'s last dimension must be contiguous")
    return pitch if shape[0] > 1 else max(pitch, shape[1])


def rms_norm_quant(x: torch.Tensor, weight: torch.Tensor | None, eps: float, *, residual: torch.Tensor | None = None,
                   residual_out: torch.Tensor | None = None, shift: torch.Tensor | None = None, rotate: bool = True,
                   qmax: float = 127.0, round_mode: int = ROUND_HALF_AWAY, y: torch.Tensor | None = None,
                   q: torch.Tensor | None = None, s: torch.Tensor | None = None, stream=None):
    """Root-mean-square norm of the rows of x [rows, K] (f32/bf16), rotated and
    quantised (phi_hip_rms_norm_quant): r = x + residual, written to
    residual_out (which may be residual); y = r / sqrt(mean(r^2) + eps) *
    weight + shift, written to y if that is given; returns (q int8 [rows, K],
    s f32 [rows]), the operand of i8_gemm."""
    _require_device(x, weight, residual, residual_out, shift, y, q, s)
    shape = x.shape
    rows, K = shape
    ldx = _row_pitch("x", x, shape)
    if q is None:
        q, ldq = _empty(shape, torch.int8, x, stream), K
    else:
        ldq = _row_pitch("q", q, shape)
    if s is None:
        s = _empty((rows,), torch.float32, x, stream)
    elif s.shape != shape[:1] or (rows > 1 and s.stride(0) != 1):
        raise ValueError(f"rms_norm_quant: s is {tuple(s.shape)}, not contiguous {(rows,)}")
    ldr, rdt = (0, F32) if residual is None else (_row_pitch("residual", residual, shape), _dt(residual))
    if residual is not None and residual_out is not None and (
            _row_pitch("residual_out", residual_out, shape) != ldr or residual_out.dtype != residual.dtype):
        raise ValueError("rms_norm_quant: residual and residual_out differ in dtype or pitch")
    w = weight if weight is not None else shift
    for t in (weight, shift):
        if t is not None and (t.shape != shape[1:] or (K > 1 and t.stride(0) != 1) or t.dtype != w.dtype):
            raise ValueError(f"rms_norm_quant: weight and shift must be contiguous {(K,)} of one dtype")
    ldy, ydt = (0, F32) if y is None else (_row_pitch("y", y, shape), _dt(y))
    if q.dtype != torch.int8 or s.dtype != torch.float32:
        raise ValueError("rms_norm_quant: q is int8, s f32")
    _check(load().phi_hip_rms_norm_quant(
        _stream(stream), x.data_ptr(), _dt(x), ldx, _ptr(residual), _ptr(residual_out), rdt, ldr, _ptr(weight),
        _ptr(shift), F32 if w is None else _dt(w), eps, rows, K, _ptr(y), ydt, ldy, q.data_ptr(), ldq, s.data_ptr(),
        qmax, round_mode, 1 if rotate else 0))
    return q, s


class KvCache(tuple):
    """An int8 paged cache (k, v, k_scale, v_scale): codes k, v int8 [blocks,
    heads, page, dim] and their scales f32 [blocks, heads, page].  Any strides
    with a contiguous dim (a permuted [blocks, page, heads, dim] fits); k and v
    alike, the scales alike."""

    def __new__(cls, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor):
        shape, kst, sst = k.shape, k.stride(), k_scale.stride()
        if (k.dtype != torch.int8 or v.dtype != torch.int8 or k_scale.dtype != torch.float32
                or v_scale.dtype != torch.float32 or v.shape != shape or len(shape) != 4 or k_scale.shape != shape[:3]
                or v_scale.shape != shape[:3]):
            raise ValueError("KvCache: k and v are int8 [blocks, heads, page, dim], their scales f32 [blocks, heads, page]")
        if kst != v.stride() or sst != v_scale.stride() or kst[3] != 1:
            raise ValueError("KvCache: k and v (and their scales) must have the same strides, dim contiguous")
        _require_device(k, v, k_scale, v_scale)
        self = tuple.__new__(cls, (k, v, k_scale, v_scale))
        self._heads, self._dim = shape[1], shape[3]
        self._desc = ctypes.byref(KvCacheDesc(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), *shape,
                                              kst[0], kst[1], kst[2], *sst))
        return self

    k = property(itemgetter(0))
    v = property(itemgetter(1))
    k_scale = property(itemgetter(2))
    v_scale = property(itemgetter(3))


def kv_cache_empty(blocks: int, page: int, heads: int, dim: int, device) -> KvCache:
    """A cache with nothing written yet."""
    codes = [torch.empty((blocks, heads, page, dim), dtype=torch.int8, device=device) for _ in range(2)]
    scales = [torch.empty((blocks, heads, page), dtype=torch.float32, device=device) for _ in range(2)]
    return KvCache(*codes, *scales)


def _vectors(who: str, name: str, t: torch.Tensor, shape):
    """The token and head strides of [tokens, heads, dim] vectors."""
    st = t.stride()
    if t.shape != shape or st[2] != 1:
        raise ValueError(f"{who}: {name} is {tuple(t.shape)}, not {tuple(shape)} with its last dimension contiguous")
    return st[0], st[1]


def _kv_tokens(who: str, cache: KvCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, shape):
    _require_device(k, v, slots)
    if k.dtype != v.dtype or slots.dtype != torch.int64 or not slots.is_contiguous():
        raise ValueError(f"{who}: k and v of one dtype, slots contiguous int64")
    return (*_vectors(who, "k", k, shape), *_vectors(who, "v", v, shape))


def kv_cache_write(cache: KvCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, *, stream=None) -> None:
    """Quantise k, v [tokens, heads, dim] (f32/bf16, any token and head strides)
    into the cache at slots [tokens] int64 (block * page + place, each once;
    negative: the token is skipped), one scale a token and head
    (phi_hip_kv_cache_write)."""
    n = slots.numel()
    kt, kh, vt, vh = _kv_tokens("kv_cache_write", cache, k, v, slots, (n, cache._heads, cache._dim))
    _check(load().phi_hip_kv_cache_write(_stream(stream), cache._desc, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, _dt(k),
                                         slots.data_ptr(), n))


def kv_cache_read(cache: KvCache, slots: torch.Tensor, *, out_dtype=torch.bfloat16, k: torch.Tensor | None = None,
                  v: torch.Tensor | None = None, stream=None):
    """The values at slots [tokens] int64 as k, v [tokens, heads, dim] (zeros for
    a negative slot; phi_hip_kv_cache_read).  k and v share no memory."""
    n = slots.numel()
    shape = (n, cache._heads, cache._dim)
    if k is None:
        k = _empty(shape, out_dtype, slots, stream)
    if v is None:
        v = _empty(shape, k.dtype, slots, stream)
    kt, kh, vt, vh = _kv_tokens("kv_cache_read", cache, k, v, slots, shape)
    _check(load().phi_hip_kv_cache_read(_stream(stream), cache._desc, slots.data_ptr(), n, k.data_ptr(), kt, kh,
                                        v.data_ptr(), vt, vh, _dt(k)))
    return k, v


def paged_attention_workspace(tokens: int, q_heads: int, kv_heads: int, dim: int, batch: int, max_q: int, max_kv: int,
                              dtype: torch.dtype, device) -> torch.Tensor | None:
    """A buffer of phi_hip_paged_attention_workspace_bytes bytes (None when 0)."""
    n = load().phi_hip_paged_attention_workspace_bytes(tokens, q_heads, kv_heads, dim, batch, max_q, max_kv, _DTYPES[dtype])
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


def paged_attention(q: torch.Tensor, cache: KvCache, block_table: torch.Tensor, q_start: torch.Tensor,
                    kv_len: torch.Tensor, *, max_q: int, max_kv: int, scale: float | None = None, causal: bool = True,
                    window: int = 0, out: torch.Tensor | None = None, workspace: torch.Tensor | None = None,
                    stream=None) -> torch.Tensor:
    """Attention of new tokens q [tokens, q_heads, dim] (bf16/f32) over the
    cache (phi_hip_paged_attention).  Sequence b's new tokens are rows
    q_start[b] .. q_start[b + 1] - 1, the last of its kv_len[b] tokens, which
    lie in blocks block_table[b] (int32, as q_start [batch + 1] and kv_len
    [batch]); max_q and max_kv bound the new tokens and the length of any
    sequence.  scale: dim ** -0.5 if not given.  A row that sees no token gives
    zeros; rows of no sequence are left as they are.  out may be columns of the
    tensor that q is in."""
    _require_device(q, block_table, q_start, kv_len, out, workspace)
    shape = q.shape
    T, Hq, D = shape
    B = kv_len.numel()
    if D != cache._dim:
        raise ValueError(f"paged_attention: q is {tuple(shape)}, the cache's vectors have {cache._dim} elements")
    qt, qh = _vectors("paged_attention", "q", q, shape)
    i32 = torch.int32
    if (block_table.dtype != i32 or q_start.dtype != i32 or kv_len.dtype != i32 or block_table.dim() != 2
            or block_table.shape[0] != B or q_start.numel() != B + 1 or not q_start.is_contiguous()
            or not kv_len.is_contiguous()):
        raise ValueError("paged_attention: block_table [batch, width], q_start [batch + 1], kv_len [batch], int32, contiguous")
    width, (pitch, step) = block_table.shape[1], block_table.stride()
    if step != 1 and width > 1:
        raise ValueError("paged_attention: block_table's rows must be contiguous")
    if out is None:
        out, ot, oh = _empty(shape, q.dtype, q, stream), Hq * D, D
    else:
        ot, oh = _vectors("paged_attention", "out", out, shape)
        if out.dtype != q.dtype:
            raise ValueError("paged_attention: out and q differ in dtype")
    L, dt = load(), _dt(q)
    if workspace is None:
        wn = L.phi_hip_paged_attention_workspace_bytes(T, Hq, cache._heads, D, B, max_q, max_kv, dt)
        if wn:
            workspace = _empty((wn,), torch.uint8, q, stream)
    wp, wn = _ws(workspace)
    _check(L.phi_hip_paged_attention(_stream(stream), q.data_ptr(), dt, qt, qh, T, Hq, cache._desc, block_table.data_ptr(),
                                     width, pitch if B > 1 else width, q_start.data_ptr(), kv_len.data_ptr(), B, max_q, max_kv,
                                     D ** -0.5 if scale is None else scale, 1 if causal else 0, window, out.data_ptr(),
                                     ot, oh, wp, wn))
    return out
