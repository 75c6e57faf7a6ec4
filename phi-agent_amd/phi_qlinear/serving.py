"""What a server of many requests runs beside the decoder layer's operators
(include/phi_serving.h).

``rotary`` turns vectors by their positions, ``rotary_cache_write`` does so on
a projection's way into the paged cache, ``kv_cache_copy`` copies pages of it,
as ``KvPages`` says when sequences fork or pages move together,
``paged_attention_shared`` attends over prefixes that sequences share and their own tokens,
``lora_batched`` adds each request's own adapter to a linear's output.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _DTYPES, _check, _dt, _ptr, _stream, _ws, load
from .decoder import KvCache, _empty, _vectors


def _here(who: str, stream, *tensors) -> None:
    """Device tensors, all of the device that the call runs on."""
    at = {t.get_device() for t in tensors if t is not None}
    if -1 in at:
        raise ValueError("phi_qlinear operates on device tensors")
    dev = torch._C._cuda_getDevice() if stream is None else stream.device.index
    if at != {dev}:
        raise ValueError(f"{who}: tensors of device {sorted(at)} in a call on device {dev}")


def rotary_frequencies(rot: int, base: float = 10000.0, *, scaling: str | None = None, factor: float = 1.0,
                       length: int = 8192, slow: float = 1.0, fast: float = 32.0, device="cuda") -> torch.Tensor:
    """Radians a position of `rot` elements' pairs, fp64 [rot / 2]: base^(-2 j / rot),
    for a context of `factor` times the trained `length` by one of these rules:

      linear  all of them 1 / factor
      ntk     another base, base * factor^(rot / (rot - 2)): the last pair's 1 / factor
      parts   pairs of more than `fast` turns in `length` positions as they are, those
              of fewer than `slow` turns 1 / factor, between them a mean weighted by
              the turns
      ramp    the same, weighted by the pair's number j between those that have `fast`
              and `slow` turns (rounded to whole pairs)
    """
    if rot < 2 or rot % 2:
        raise ValueError(f"rotary_frequencies: {rot} is no even number from 2 on")
    j = torch.arange(rot // 2, dtype=torch.float64)
    if scaling == "ntk":
        if rot < 4:
            raise ValueError("rotary_frequencies: ntk needs two pairs")
        base = base * factor ** (rot / (rot - 2))
    f = base ** (-2.0 * j / rot)
    if scaling in (None, "ntk"):
        return f.to(device)
    if scaling == "linear":
        keep = torch.zeros_like(f)
    elif scaling == "parts":
        keep = ((length * f / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
    elif scaling == "ramp":
        pair = lambda turns: rot * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        first, last = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), rot - 1)
        keep = 1 - ((j - first) / max(last - first, 1e-3)).clamp(0, 1)
    else:
        raise ValueError(f"rotary_frequencies: no rule {scaling!r}")
    return (f * (keep + (1 - keep) / factor)).to(device)


def _turns(who: str, positions: torch.Tensor, freq: torch.Tensor, tokens: int) -> None:
    if (positions.dtype != torch.int64 or positions.shape != (tokens,) or not positions.is_contiguous()
            or freq.dtype != torch.float64 or freq.dim() != 1 or not freq.is_contiguous()):
        raise ValueError(f"{who}: positions [tokens] int64 and freq [rot / 2] float64, contiguous")


def rotary(x: torch.Tensor, positions: torch.Tensor, freq: torch.Tensor, *, interleaved: bool = False,
           scale: float = 1.0, out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """Rotary positions of x [tokens, heads, dim] (f32/bf16, any strides with a
    contiguous dim; phi_hip_rotary): the pairs of each vector's first 2 len(freq)
    elements, (j, j + len(freq)) or, interleaved, (2 j, 2 j + 1), turned by
    positions [tokens] int64 times freq [rot / 2] float64 and scaled; the rest
    copied.  out may be x."""
    _here("rotary", stream, x, positions, freq, out)
    shape = x.shape
    T, H, D = shape
    xt, xh = _vectors("rotary", "x", x, shape)
    _turns("rotary", positions, freq, T)
    if out is None:
        out, ot, oh = _empty(shape, x.dtype, x, stream), H * D, D
    else:
        ot, oh = _vectors("rotary", "out", out, shape)
        if out.dtype != x.dtype:
            raise ValueError("rotary: out and x differ in dtype")
    _check(load().phi_hip_rotary(_stream(stream), x.data_ptr(), _dt(x), xt, xh, T, H, D, positions.data_ptr(),
                                 freq.data_ptr(), 2 * freq.shape[0], 1 if interleaved else 0, scale, out.data_ptr(), ot, oh))
    return out


def rotary_cache_write(cache: KvCache, q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor,
                       positions: torch.Tensor, freq: torch.Tensor, slots: torch.Tensor, *, interleaved: bool = False,
                       scale: float = 1.0, out: torch.Tensor | None = None, stream=None) -> torch.Tensor | None:
    """A projection's output on its way to attention (phi_hip_rotary_cache_write):
    q [tokens, q_heads, dim] rotated as by `rotary` and returned (out may be q; q
    None: there is none), k [tokens, heads, dim] rotated and v as it is into the
    cache at slots [tokens], as by `kv_cache_write`.  q, k and v of one dtype
    (f32/bf16), vectors 16-byte aligned."""
    who = "rotary_cache_write"
    _here(who, stream, cache.k, q, k, v, positions, freq, slots, out)
    n = slots.numel()
    shape = (n, cache._heads, cache._dim)
    if k.dtype != v.dtype or (q is not None and q.dtype != k.dtype) or slots.dtype != torch.int64 or not slots.is_contiguous():
        raise ValueError(f"{who}: q, k and v of one dtype, slots contiguous int64")
    kt, kh = _vectors(who, "k", k, shape)
    vt, vh = _vectors(who, "v", v, shape)
    _turns(who, positions, freq, n)
    qp = op = None
    qt = qh = ot = oh = heads = 0
    if q is not None:
        heads = q.shape[1]
        qt, qh = _vectors(who, "q", q, (n, heads, cache._dim))
        if out is None:
            out, ot, oh = _empty(q.shape, q.dtype, q, stream), heads * cache._dim, cache._dim
        else:
            ot, oh = _vectors(who, "out", out, q.shape)
            if out.dtype != q.dtype:
                raise ValueError(f"{who}: out and q differ in dtype")
        qp, op = q.data_ptr(), out.data_ptr()
    elif out is not None:
        raise ValueError(f"{who}: out without q")
    _check(load().phi_hip_rotary_cache_write(
        _stream(stream), cache._desc, qp, qt, qh, heads, op, ot, oh, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, _dt(k),
        positions.data_ptr(), freq.data_ptr(), 2 * freq.shape[0], 1 if interleaved else 0, scale, slots.data_ptr(), n))
    return out


def kv_cache_copy(source: KvCache, target: KvCache, from_blocks: torch.Tensor, to_blocks: torch.Tensor, *,
                  tokens: torch.Tensor | None = None, stream=None) -> None:
    """Blocks from_blocks[i] of a cache to blocks to_blocks[i] of another, or of
    the same (phi_hip_kv_cache_copy): all tokens, or the first tokens[i].  int32,
    of one length.  A block that is written is written once and not read in the
    same call; a pair with a block that its cache does not have is skipped."""
    _here("kv_cache_copy", stream, source.k, target.k, from_blocks, to_blocks, tokens)
    n = from_blocks.numel()
    for t in (from_blocks, to_blocks, tokens):
        if t is not None and (t.dtype != torch.int32 or t.shape != (n,) or not t.is_contiguous()):
            raise ValueError("kv_cache_copy: from_blocks, to_blocks and tokens are contiguous int32 of one length")
    _check(load().phi_hip_kv_cache_copy(_stream(stream), source._desc, target._desc, from_blocks.data_ptr(),
                                        to_blocks.data_ptr(), _ptr(tokens), n))


class KvPages:
    """Who has which pages of a paged cache: pages handed out as sequences grow,
    shared when they fork, taken back when their last sequence ends, and moved
    together.  Host side only: `copies` holds what the device has yet to copy,
    (from, to, tokens), for `flush` to do before the next write or attention.

    A sequence's pages are append-only, so a forked one shares its parent's whole
    pages and gets a copy of the last where that is not full: the parent's tokens are
    written before the flush that makes it.  Slots hold until pages move (`compact`);
    those that were not written by then are not valid after it."""

    def __init__(self, blocks: int, page: int):
        self.page, self.of, self.length, self.copies = page, {}, {}, []
        self.users = [0] * blocks
        self.free = list(range(blocks))[::-1]  # the lowest is handed out first

    def _take(self, n: int) -> list[int]:
        if n > len(self.free):
            raise RuntimeError("the cache is full")
        got = [self.free.pop() for _ in range(n)]
        for b in got:
            self.users[b] = 1
        return got

    def grow(self, seq, tokens: int) -> list[int]:
        """Room for `tokens` more of a sequence (a new one, if it is not known):
        their slots.  All or nothing: RuntimeError where there are too few pages."""
        if tokens < 0:
            raise ValueError(f"KvPages: {tokens} tokens")
        at, mine = self.length.get(seq, 0), self.of.get(seq, [])
        new = self._take(max(0, -(-(at + tokens) // self.page) - len(mine)))
        self.of[seq] = mine = mine + new
        self.length[seq] = at + tokens
        return [mine[t // self.page] * self.page + t % self.page for t in range(at, at + tokens)]

    def fork(self, parent, child) -> None:
        """A sequence `child` with the parent's tokens."""
        if child in self.of:
            raise ValueError(f"KvPages: {child!r} is there already")
        n, pages = self.length[parent], self.of[parent]
        whole, rest = divmod(n, self.page)
        last = self._take(1) if rest else []
        for b in pages[:whole]:
            self.users[b] += 1
        if rest:
            self.copies.append((pages[whole], last[0], rest))
        self.of[child], self.length[child] = pages[:whole] + last, n

    def end(self, seq) -> None:
        """A sequence's pages back, but for those that others share."""
        for b in self.of.pop(seq, []):
            self.users[b] -= 1
            if not self.users[b]:
                self.free.append(b)
        self.length.pop(seq, None)
        self.free.sort(reverse=True)

    def shared(self, seqs) -> int:
        """How many leading pages all of `seqs` share."""
        rows = [self.of[s] for s in seqs]
        n = min(self.length[s] // self.page for s in seqs)
        return next((i for i in range(n) if any(r[i] != rows[0][i] for r in rows)), n)

    def compact(self) -> int:
        """Move pages so that those in use are the lowest; the number of them."""
        used = [b for b, n in enumerate(self.users) if n]
        high = [b for b in used if b >= len(used)]
        low = [b for b in range(len(used)) if not self.users[b]]
        move = dict(zip(high, low))
        for a, b in move.items():
            self.users[a], self.users[b] = 0, self.users[a]
            self.copies.append((a, b, self.page))
        self.of = {s: [move.get(b, b) for b in pages] for s, pages in self.of.items()}
        self.free = list(range(len(used), len(self.users)))[::-1]
        return len(used)

    def flush(self, cache: KvCache, stream=None) -> None:
        """Have the device do the copies, in as few calls as leave no block in one that
        is written there and read, or written twice.  Those of a call that raises, and
        all after it, are kept."""
        if stream is not None:
            with torch.cuda.stream(stream):
                return self.flush(cache)
        while self.copies:
            read, written, now, later = set(), set(), [], []
            for c in self.copies:
                meets = c[0] in written or c[1] in written or c[1] in read
                (later if later or meets else now).append(c)
                read.add(c[0]), written.add(c[1])
            part = torch.tensor(now, dtype=torch.int32).t().contiguous().to(cache.k.device)
            kv_cache_copy(cache, cache, part[0], part[1], tokens=part[2])
            self.copies = later


def paged_attention_shared_workspace(tokens: int, q_heads: int, kv_heads: int, dim: int, groups: int, batch: int, max_prefix: int,
                                     max_q: int, max_kv: int, dtype: torch.dtype, device) -> torch.Tensor:
    """A buffer of phi_hip_paged_attention_shared_workspace_bytes bytes."""
    n = load().phi_hip_paged_attention_shared_workspace_bytes(tokens, q_heads, kv_heads, dim, groups, batch, max_prefix, max_q,
                                                              max_kv, _DTYPES[dtype])
    return torch.empty(n, dtype=torch.uint8, device=device)


def _table(name: str, t: torch.Tensor, rows: int) -> int:
    """The pitch of a table [rows, width] int32 with contiguous rows."""
    pitch, step = t.stride()
    if t.dtype != torch.int32 or t.shape[0] != rows or (step != 1 and t.shape[1] > 1):
        raise ValueError(f"paged_attention_shared: {name} is [{rows}, width] int32 with contiguous rows")
    return pitch if rows > 1 else t.shape[1]


def paged_attention_shared(q: torch.Tensor, cache: KvCache, prefix_table: torch.Tensor, prefix_len: torch.Tensor,
                           group_start: torch.Tensor, block_table: torch.Tensor, q_start: torch.Tensor,
                           kv_len: torch.Tensor, *, max_prefix: int, max_q: int, max_kv: int, scale: float | None = None,
                           out: torch.Tensor | None = None, workspace: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """Causal attention of new tokens q [tokens, q_heads, dim] (bf16/f32) over
    prefixes that sequences share and their own tokens
    (phi_hip_paged_attention_shared; for a few new tokens each).  Sequences group_start[g] ..
    group_start[g + 1] - 1 see prefix_len[g] tokens in blocks prefix_table[g],
    then their own as by `paged_attention`: kv_len[b] in blocks block_table[b],
    the last of them rows q_start[b] .. q_start[b + 1] - 1 of q.  All int32;
    max_prefix, max_q and max_kv bound a prefix, the new tokens and the own tokens
    of any sequence.  scale: dim ** -0.5 if not given."""
    who = "paged_attention_shared"
    _here(who, stream, q, cache.k, prefix_table, prefix_len, group_start, block_table, q_start, kv_len, out, workspace)
    shape = q.shape
    T, Hq, D = shape
    G, B, i32 = prefix_len.numel(), kv_len.numel(), torch.int32
    if D != cache._dim:
        raise ValueError(f"{who}: q is {tuple(shape)}, the cache's vectors have {cache._dim} elements")
    qt, qh = _vectors(who, "q", q, shape)
    for name, t, n in (("prefix_len", prefix_len, G), ("group_start", group_start, G + 1), ("q_start", q_start, B + 1), ("kv_len", kv_len, B)):
        if t.dtype != i32 or t.shape != (n,) or not t.is_contiguous():
            raise ValueError(f"{who}: {name} is contiguous int32 [{n}]")
    prefix_pitch, pitch = _table("prefix_table", prefix_table, G), _table("block_table", block_table, B)
    if out is None:
        out, ot, oh = _empty(shape, q.dtype, q, stream), Hq * D, D
    else:
        ot, oh = _vectors(who, "out", out, shape)
        if out.dtype != q.dtype:
            raise ValueError(f"{who}: out and q differ in dtype")
    L, dt = load(), _dt(q)
    if workspace is None:
        wn = L.phi_hip_paged_attention_shared_workspace_bytes(T, Hq, cache._heads, D, G, B, max_prefix, max_q, max_kv, dt)
        workspace = _empty((wn,), torch.uint8, q, stream)
    wp, wn = _ws(workspace)
    _check(L.phi_hip_paged_attention_shared(
        _stream(stream), q.data_ptr(), dt, qt, qh, T, Hq, cache._desc, prefix_table.data_ptr(), prefix_table.shape[1], prefix_pitch,
        prefix_len.data_ptr(), group_start.data_ptr(), G, max_prefix, block_table.data_ptr(), block_table.shape[1], pitch,
        q_start.data_ptr(), kv_len.data_ptr(), B, max_q, max_kv, D ** -0.5 if scale is None else scale, out.data_ptr(), ot, oh, wp, wn))
    return out


def lora_batched_workspace(rows: int, K: int, R: int, device) -> torch.Tensor:
    """A buffer of phi_hip_lora_batched_workspace_bytes bytes."""
    return torch.empty(load().phi_hip_lora_batched_workspace_bytes(rows, K, R), dtype=torch.uint8, device=device)


def _pitch(name: str, t: torch.Tensor, shape) -> int:
    """The pitch of a [rows, columns] tensor with contiguous rows (of one row: any from the columns on)."""
    if t.shape != shape or (t.stride(1) != 1 and shape[1] > 1):
        raise ValueError(f"lora_batched: {name} is {tuple(t.shape)}, not {tuple(shape)} with contiguous rows")
    return t.stride(0) if shape[0] > 1 else max(t.stride(0), shape[1])


def lora_batched(x: torch.Tensor, A: torch.Tensor, B: torch.Tensor, adapter: torch.Tensor, *,
                 scale: torch.Tensor | None = None, base: torch.Tensor | None = None, out: torch.Tensor | None = None,
                 out_dtype=None, workspace: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """base + scale[a] B[a] (A[a] x) for rows of x [rows, K], a the row's adapter
    [rows] int32 (below 0 or not below the adapters: none; phi_hip_lora_batched).
    A [adapters, R, K] and B [adapters, N, R] of one dtype, scale [adapters] f32
    (None: 1), base [rows, N] the linear's output (None: 0); out may be base.  out
    has base's dtype, or out_dtype (x's if neither is given).  All f32/bf16."""
    _here("lora_batched", stream, x, A, B, adapter, scale, base, out, workspace)
    M, K = x.shape
    if A.dim() != 3 or B.dim() != 3 or A.dtype != B.dtype:
        raise ValueError("lora_batched: A is [adapters, R, K] and B [adapters, N, R], of one dtype")
    n, R, N = A.shape[0], A.shape[1], B.shape[1]
    ast, bst = A.stride(), B.stride()
    if A.shape[2] != K or B.shape[0] != n or B.shape[2] != R or (K > 1 and ast[2] != 1) or (R > 1 and bst[2] != 1):
        raise ValueError(f"lora_batched: factors of {tuple(A.shape)} and {tuple(B.shape)} for rows of {K}, last dimension contiguous")
    if adapter.dtype != torch.int32 or adapter.shape != (M,) or not adapter.is_contiguous():
        raise ValueError("lora_batched: adapter is contiguous int32 [rows]")
    if scale is not None and (scale.dtype != torch.float32 or scale.shape != (n,) or not scale.is_contiguous()):
        raise ValueError("lora_batched: scale is contiguous f32 [adapters]")
    shape = (M, N)
    if out is None:
        out = _empty(shape, out_dtype or (x if base is None else base).dtype, x, stream)
    if (base is not None and base.dtype != out.dtype) or (out_dtype is not None and out.dtype != out_dtype):
        raise ValueError("lora_batched: base and out differ in dtype")
    L = load()
    if workspace is None:
        workspace = _empty((L.phi_hip_lora_batched_workspace_bytes(M, K, R),), torch.uint8, x, stream)
    wp, wn = _ws(workspace)
    _check(L.phi_hip_lora_batched(
        _stream(stream), x.data_ptr(), _dt(x), _pitch("x", x, (M, K)), M, K, A.data_ptr(), ast[0], ast[1] if R > 1 else max(ast[1], K),
        B.data_ptr(), bst[0], bst[1] if N > 1 else max(bst[1], R), _dt(A), n, R, N, adapter.data_ptr(), _ptr(scale), _ptr(base),
        0 if base is None else _pitch("base", base, shape), out.data_ptr(), _dt(out), _pitch("out", out, shape), wp, wn))
    return out
