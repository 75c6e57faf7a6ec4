"""Plain 64-bit forms of the decoder layer's operators, on the CPU, and the
errors that their kernels' arithmetic may add."""
import math

import torch


def hadamard() -> torch.Tensor:
    """The linear's 256-wide rotation (J - 2R)^(x4) / 16, rows and columns alike."""
    j = torch.ones((4, 4), dtype=torch.float64) - 2 * torch.eye(4, dtype=torch.float64).flip(0)
    h = torch.kron(torch.kron(j, j), torch.kron(j, j))
    return h / 16


def norm(x, weight, shift, residual, eps, rotate):
    """(r, y, z) in 64 bits: the sum, the normalised row, the row that is quantised."""
    r = x.double() if residual is None else x.double() + residual.double()
    y = r / torch.sqrt((r * r).mean(dim=1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.double()
    if shift is not None:
        y = y + shift.double()
    z = (y.reshape(-1, 256) @ hadamard()).reshape(y.shape) if rotate else y
    return r, y, z


def quantise_f32(x):
    """(codes, scale) of the last axis in the kernels' own fp32 steps, finite x:
    amax / 127, its reciprocal, ties away from zero."""
    x = x.float()
    amax = x.abs().amax(dim=-1)
    s = torch.where(amax > 1e-30, amax / 127.0, torch.ones_like(amax))
    d = x * (1.0 / s)[..., None]
    t = torch.trunc(d)  # d - t is exact
    q = t + torch.where((d - t).abs() >= 0.5, torch.copysign(torch.ones_like(d), d), torch.zeros_like(d))
    return q.clamp(-127, 127).to(torch.int8), s


def attention(q, k, v, ks, vs, table, q_start, kv_len, *, scale, causal=True, window=0):
    """out [tokens, heads, dim] in 64 bits and, beside each value, how far a
    kernel may be from it (bound); rows of no sequence give NaN (nothing writes them)."""
    T, Hq, D = q.shape
    blocks, H, page, _ = k.shape
    G = Hq // H
    out = torch.full((T, Hq, D), math.nan, dtype=torch.float64)
    bound = torch.full((T, Hq, D), math.nan, dtype=torch.float64)
    f32 = q.dtype == torch.float32
    steps = 8355711.0 if f32 else 32639.0  # the largest integer that holds |q| / its row's largest
    p_bits = 2.0 ** -21 if f32 else 2.0 ** -11
    for b in range(len(kv_len)):
        s0, n, kv = q_start[b], q_start[b + 1] - q_start[b], kv_len[b]
        t = torch.arange(kv)
        block = table[b][t // page] if kv else torch.zeros(0, dtype=torch.int64)
        live = (block >= 0) & (block < blocks)
        bl, at = block.clamp(0, blocks - 1).long(), t % page
        for i in range(n):
            pos = kv - n + i
            seen = live.clone()
            if causal:
                seen &= t <= pos
            if window:
                seen &= t > pos - window
            if not bool(seen.any()):
                out[s0 + i], bound[s0 + i] = 0.0, 0.0
                continue
            for h in range(Hq):
                g = h // G
                kd = k[bl[seen], g, at[seen]].double() * ks[bl[seen], g, at[seen]].double()[:, None]
                vd = v[bl[seen], g, at[seen]].double() * vs[bl[seen], g, at[seen]].double()[:, None]
                qd = q[s0 + i, h].double()
                logit = (kd @ qd) * scale
                p = torch.softmax(logit, dim=0)
                o = p @ vd
                # Half a step of q a product, and the logit's own fp32 roundings
                # (five of them, on values up to the largest logit in base 2).
                e = abs(scale) * 0.5 / steps * float(qd.abs().max()) * float(kd.abs().sum(dim=1).max())
                e += 5 * 2.0 ** -24 * 1.4427 * float(logit.abs().max()) + 2.0 ** -22
                # Softmax with each logit off by e: every weight by 2e; then p's
                # bits, the sums in fp32, and the output's own rounding.
                weight = p @ vd.abs()
                out[s0 + i, h] = o
                bound[s0 + i, h] = (2.0 * e + p_bits + 2.0 ** -20) * weight + (2.0 ** -23 if f32 else 2.0 ** -8) * o.abs()
    return out, bound


def make_case(lens, *, Hq, H, D, page, dtype, seed, blocks_extra=2, token_major=False, spare=0.0):
    """CPU tensors of a batch: lens is [(new tokens, tokens in the cache)].  What
    no sequence has written holds NaN scales; spare entries of the table are -1."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-kv // page) for _, kv in lens]
    blocks = sum(need) + blocks_extra
    order = torch.randperm(blocks, generator=g).tolist()
    width = max(need + [1]) + 1
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    k = torch.randint(-127, 128, (blocks, H, page, D), generator=g, dtype=torch.int8)
    v = torch.randint(-127, 128, (blocks, H, page, D), generator=g, dtype=torch.int8)
    ks, vs = (torch.full((blocks, H, page), math.nan) for _ in range(2))
    for b, (_, kv) in enumerate(lens):
        for j in range(need[b]):
            table[b, j] = blk = order.pop()
            m = min(page, kv - j * page)
            ks[blk, :, :m] = torch.rand((H, m), generator=g) * 0.02 + 0.002
            vs[blk, :, :m] = torch.rand((H, m), generator=g) * 0.05 + 0.002
    starts = [0]
    for n, _ in lens:
        starts.append(starts[-1] + n)
    q = (torch.randn((starts[-1], Hq, D), generator=g)).to(dtype)
    if token_major:  # the same cache with the heads inside a block's tokens
        k, v = (x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for x in (k, v))
        ks, vs = (x.permute(0, 2, 1).contiguous().permute(0, 2, 1) for x in (ks, vs))
    return dict(q=q, k=k, v=v, ks=ks, vs=vs, table=table, starts=starts, kv_len=[kv for _, kv in lens])
