"""The operators between a decoder layer's int8 linears (include/phi_decoder.h).

``rms_norm_quant`` turns the residual stream into the int8 operand of the
linear that follows, ``kv_cache_write`` / ``kv_cache_read`` keep keys and
values in an int8 paged cache, ``paged_attention`` attends over it.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import (F32, ROUND_HALF_AWAY, KvCacheDesc, _check, _dt, _ptr, _require_device, _stream, _ws, load)


def _empty(shape, dtype, like: torch.Tensor, stream) -> torch.Tensor:
    """A new tensor beside `like`, from the memory of the stream that will write it."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=like.device)
    with torch.cuda.stream(stream):
        return torch.empty(shape, dtype=dtype, device=like.device)


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
    rows, K = x.shape
    if q is None:
        q = _empty((rows, K), torch.int8, x, stream)
    if s is None:
        s = _empty((rows,), torch.float32, x, stream)
    for name, t, shape in (("residual", residual, (rows, K)), ("residual_out", residual_out, (rows, K)),
                           ("weight", weight, (K,)), ("shift", shift, (K,)), ("y", y, (rows, K)), ("q", q, (rows, K)),
                           ("s", s, (rows,))):
        if t is not None and tuple(t.shape) != shape:
            raise ValueError(f"rms_norm_quant: {name} is {tuple(t.shape)}, not {shape}")
        if t is not None and K > 1 and rows > 0 and t.stride(-1) != 1 and t.numel() > 1:
            raise ValueError(f"rms_norm_quant: {name}'s last dimension must be contiguous")
    if x.stride(1) != 1 and K > 1:
        raise ValueError("rms_norm_quant: x's last dimension must be contiguous")
    if residual is not None and residual_out is not None and (
            residual.dtype != residual_out.dtype or (rows > 1 and residual.stride(0) != residual_out.stride(0))):
        raise ValueError("rms_norm_quant: residual and residual_out differ in dtype or pitch")
    if weight is not None and shift is not None and weight.dtype != shift.dtype:
        raise ValueError("rms_norm_quant: weight and shift differ in dtype")
    w = weight if weight is not None else shift
    pitch = lambda t: max(t.stride(0), K)  # noqa: E731  (one row's pitch is any number)
    _check(load().phi_hip_rms_norm_quant(
        _stream(stream), _ptr(x), _dt(x), pitch(x), _ptr(residual), _ptr(residual_out),
        F32 if residual is None else _dt(residual), 0 if residual is None else pitch(residual), _ptr(weight),
        _ptr(shift), F32 if w is None else _dt(w), float(eps), rows, K, _ptr(y), F32 if y is None else _dt(y),
        0 if y is None else pitch(y), _ptr(q), pitch(q), _ptr(s), float(qmax), round_mode, 1 if rotate else 0))
    return q, s


class KvCache(NamedTuple):
    """An int8 paged cache: codes k, v int8 [blocks, heads, page, dim] and their
    scales f32 [blocks, heads, page].  Any strides with a contiguous dim (a
    permuted [blocks, page, heads, dim] fits); k and v alike, the scales alike."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


def kv_cache_empty(blocks: int, page: int, heads: int, dim: int, device) -> KvCache:
    """A cache with nothing written yet."""
    codes = [torch.empty((blocks, heads, page, dim), dtype=torch.int8, device=device) for _ in range(2)]
    scales = [torch.empty((blocks, heads, page), dtype=torch.float32, device=device) for _ in range(2)]
    return KvCache(*codes, *scales)


def _desc(c: KvCache):
    k, v, ks, vs = c
    _require_device(k, v, ks, vs)
    kst, sst = k.stride(), ks.stride()
    if (k.dtype != torch.int8 or v.dtype != torch.int8 or ks.dtype != torch.float32 or vs.dtype != torch.float32
            or k.shape != v.shape or k.dim() != 4 or ks.shape != k.shape[:3] or vs.shape != k.shape[:3]):
        raise ValueError("KvCache: k and v are int8 [blocks, heads, page, dim], their scales f32 [blocks, heads, page]")
    if kst != v.stride() or sst != vs.stride() or kst[3] != 1:
        raise ValueError("KvCache: k and v (and their scales) must have the same strides, dim contiguous")
    return ctypes.byref(KvCacheDesc(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), *k.shape, kst[0], kst[1],
                                    kst[2], *sst))


def _vectors(who: str, name: str, t: torch.Tensor, shape) -> None:
    if tuple(t.shape) != shape or t.stride(2) != 1:
        raise ValueError(f"{who}: {name} is {tuple(t.shape)}, not {shape} with its last dimension contiguous")


def kv_cache_write(cache: KvCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, *, stream=None) -> None:
    """Quantise k, v [tokens, heads, dim] (f32/bf16, any token and head strides)
    into the cache at slots [tokens] int64 (block * page + place; negative: the
    token is skipped), one scale a token and head (phi_hip_kv_cache_write)."""
    _require_device(k, v, slots)
    shape = (slots.numel(), cache.k.shape[1], cache.k.shape[3])
    _vectors("kv_cache_write", "k", k, shape)
    _vectors("kv_cache_write", "v", v, shape)
    if k.dtype != v.dtype or slots.dtype != torch.int64 or not slots.is_contiguous():
        raise ValueError("kv_cache_write: k and v of one dtype, slots contiguous int64")
    _check(load().phi_hip_kv_cache_write(_stream(stream), _desc(cache), _ptr(k), k.stride(0), k.stride(1), _ptr(v),
                                         v.stride(0), v.stride(1), _dt(k), _ptr(slots), shape[0]))


def kv_cache_read(cache: KvCache, slots: torch.Tensor, *, out_dtype=torch.bfloat16, k: torch.Tensor | None = None,
                  v: torch.Tensor | None = None, stream=None):
    """The values at slots [tokens] int64 as k, v [tokens, heads, dim] (zeros for
    a negative slot; phi_hip_kv_cache_read)."""
    shape = (slots.numel(), cache.k.shape[1], cache.k.shape[3])
    if k is None:
        k = _empty(shape, out_dtype, slots, stream)
    if v is None:
        v = _empty(shape, k.dtype, slots, stream)
    _require_device(k, v, slots)
    _vectors("kv_cache_read", "k", k, shape)
    _vectors("kv_cache_read", "v", v, shape)
    if k.dtype != v.dtype or slots.dtype != torch.int64 or not slots.is_contiguous():
        raise ValueError("kv_cache_read: k and v of one dtype, slots contiguous int64")
    _check(load().phi_hip_kv_cache_read(_stream(stream), _desc(cache), _ptr(slots), shape[0], _ptr(k), k.stride(0),
                                        k.stride(1), _ptr(v), v.stride(0), v.stride(1), _dt(k)))
    return k, v


def paged_attention_workspace(tokens: int, q_heads: int, kv_heads: int, dim: int, batch: int, max_q: int, max_kv: int,
                              dtype: torch.dtype, device) -> torch.Tensor | None:
    """A buffer of phi_hip_paged_attention_workspace_bytes bytes (None when 0)."""
    from . import _DTYPES
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
    zeros."""
    _require_device(q, block_table, q_start, kv_len, out, workspace)
    T, Hq, D = q.shape
    B = kv_len.numel()
    if D != cache.k.shape[3] or q.stride(2) != 1:
        raise ValueError(f"paged_attention: q is {tuple(q.shape)}, the cache's vectors have {cache.k.shape[3]} elements")
    if (block_table.dtype != torch.int32 or q_start.dtype != torch.int32 or kv_len.dtype != torch.int32
            or block_table.dim() != 2 or block_table.shape[0] != B or q_start.numel() != B + 1
            or not q_start.is_contiguous() or not kv_len.is_contiguous()
            or (block_table.shape[1] > 1 and block_table.stride(1) != 1)):
        raise ValueError("paged_attention: block_table [batch, width], q_start [batch + 1], kv_len [batch], int32, contiguous")
    if out is None:
        out = _empty((T, Hq, D), q.dtype, q, stream)
    _vectors("paged_attention", "out", out, (T, Hq, D))
    if out.dtype != q.dtype:
        raise ValueError("paged_attention: out and q differ in dtype")
    L, desc, dt = load(), _desc(cache), _dt(q)
    if workspace is None:
        n = L.phi_hip_paged_attention_workspace_bytes(T, Hq, cache.k.shape[1], D, B, max_q, max_kv, dt)
        if n:
            workspace = _empty((n,), torch.uint8, q, stream)
    wp, wn = _ws(workspace)
    _check(L.phi_hip_paged_attention(_stream(stream), _ptr(q), dt, q.stride(0), q.stride(1), T, Hq, desc,
                                     _ptr(block_table), block_table.shape[1], max(block_table.stride(0), block_table.shape[1]),
                                     _ptr(q_start), _ptr(kv_len), B, max_q, max_kv, D ** -0.5 if scale is None else scale,
                                     1 if causal else 0, window, _ptr(out), out.stride(0), out.stride(1), wp, wn))
    return out
