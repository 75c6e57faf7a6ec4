"""Plain 64-bit forms of the serving operators, on the CPU."""
import torch


def rotated(x, positions, freq, interleaved, scale):
    """x [tokens, heads, dim] turned, in 64 bits, and beside each value the sum of
    its terms' magnitudes (of what was only copied: 0)."""
    half = freq.numel()
    x = x.double()
    angle = positions.double()[:, None] * freq
    cos, sin = torch.cos(angle)[:, None] * scale, torch.sin(angle)[:, None] * scale
    j = torch.arange(half)
    i, k = (2 * j, 2 * j + 1) if interleaved else (j, j + half)
    a, b = x[..., i], x[..., k]
    y, mag = x.clone(), torch.zeros_like(x)
    y[..., i], y[..., k] = a * cos - b * sin, b * cos + a * sin
    mag[..., i] = mag[..., k] = abs(scale) * (a.abs() + b.abs())
    return y, mag


def adapted(x, A, B, adapter, scale, base):
    """base + scale B (A x) of each row's adapter in 64 bits and, beside each value,
    the sum of its terms' magnitudes through both products (0: none)."""
    n, R, K = A.shape
    M, N = x.shape[0], B.shape[1]
    y = torch.zeros((M, N), dtype=torch.float64) if base is None else base.double()
    mag = torch.zeros((M, N), dtype=torch.float64)
    for a in range(n):
        mine = adapter == a
        s = 1.0 if scale is None else scale[a].double()
        xa, Aa, Ba = x[mine].double(), A[a].double(), B[a].double()
        y[mine] += (xa @ Aa.t()) @ Ba.t() * s
        mag[mine] = (xa.abs() @ Aa.abs().t()) @ Ba.abs().t() * abs(s)
    return y, mag


def shared_case(groups, free, *, Hq, H, D, page, dtype, seed, blocks_extra=2, token_major=False):
    """CPU tensors of a batch with shared prefixes: groups [(prefix length, [(new
    tokens, own tokens)])], free [(new, own)] sequences of no group, first[0] before the
    groups where free is a pair of lists.  What nothing has written holds NaN scales; spare
    entries of the tables are -1."""
    g = torch.Generator().manual_seed(seed)
    before, after = free if isinstance(free, tuple) else ([], free)
    seqs = before + [m for _, members in groups for m in members] + after
    lens = [p for p, _ in groups] + [kv for _, kv in seqs]
    need = [-(-n // page) for n in lens]
    blocks = sum(need) + blocks_extra
    order = torch.randperm(blocks, generator=g).tolist()
    k = torch.randint(-127, 128, (blocks, H, page, D), generator=g, dtype=torch.int8)
    v = torch.randint(-127, 128, (blocks, H, page, D), generator=g, dtype=torch.int8)
    ks, vs = (torch.full((blocks, H, page), float("nan")) for _ in range(2))
    widths = [max(need[:len(groups)] + [1]) + 1, max(need[len(groups):] + [1]) + 1]
    tables = [torch.full((len(groups), widths[0]), -1, dtype=torch.int32), torch.full((len(seqs), widths[1]), -1, dtype=torch.int32)]
    for i, n in enumerate(lens):
        table, row = (tables[0], i) if i < len(groups) else (tables[1], i - len(groups))
        for j in range(need[i]):
            table[row, j] = blk = order.pop()
            m = min(page, n - j * page)
            ks[blk, :, :m] = torch.rand((H, m), generator=g) * 0.02 + 0.002
            vs[blk, :, :m] = torch.rand((H, m), generator=g) * 0.05 + 0.002
    starts, firsts = [0], [len(before)]
    for n, _ in seqs:
        starts.append(starts[-1] + n)
    for _, members in groups:
        firsts.append(firsts[-1] + len(members))
    q = torch.randn((starts[-1], Hq, D), generator=g).to(dtype)
    if token_major:
        k, v = (x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for x in (k, v))
        ks, vs = (x.permute(0, 2, 1).contiguous().permute(0, 2, 1) for x in (ks, vs))
    return dict(q=q, k=k, v=v, ks=ks, vs=vs, prefix_table=tables[0], table=tables[1], prefix_len=[p for p, _ in groups],
                group_start=firsts, starts=starts, kv_len=[kv for _, kv in seqs])


def shared_attention(c, scale):
    """out [tokens, heads, dim] in 64 bits (rows of no sequence NaN) and how far a kernel may be from it.

    A logit's error is half a step of q's 16 bits (bf16; or 24) a product, 2^-11 of k's elements (of
    a chunk; fp32 queries: none) and fp32 roundings, five of them on values up to the largest logit in base 2;
    a weight is off by twice that, and by p's, v's and its scale's 2^-11 each (fp32 queries: 2^-21) and
    sums in fp32, 2^-20, of two parts and their join.  The least bits of v's and p's units, 2^-29 of the
    largest |v| seen, and the output's own rounding."""
    q, k, v, ks, vs = (c[x] for x in ("q", "k", "v", "ks", "vs"))
    T, Hq, D = q.shape
    blocks, H, page, _ = k.shape
    f32 = q.dtype == torch.float32
    out, bound = (torch.full((T, Hq, D), float("nan"), dtype=torch.float64) for _ in range(2))

    def tokens(table, n):
        t = torch.arange(n)
        blk = table[t // page].long() if n else t
        live = (blk >= 0) & (blk < blocks)
        return torch.where(live, blk, 0), t % page, live

    for b, kv in enumerate(c["kv_len"]):
        s0, n = c["starts"][b], c["starts"][b + 1] - c["starts"][b]
        if n <= 0:
            continue
        blk, at, live = tokens(c["table"][b], kv)
        seen = live & (torch.arange(kv) <= kv - n + torch.arange(n)[:, None])
        for g in range(len(c["prefix_len"])):
            if c["group_start"][g] <= b < c["group_start"][g + 1]:
                pb, pa, pl = tokens(c["prefix_table"][g], c["prefix_len"][g])
                blk, at, seen = torch.cat([pb, blk]), torch.cat([pa, at]), torch.cat([pl.expand(n, -1), seen], dim=1)
        some = seen.any(1)
        for h in range(Hq):
            g = h // (Hq // H)
            there = seen.any(0)
            kd = torch.where(there[:, None], k[blk, g, at].double() * ks[blk, g, at].double()[:, None], 0.0)
            vd = torch.where(there[:, None], v[blk, g, at].double() * vs[blk, g, at].double()[:, None], 0.0)
            qd = q[s0:s0 + n, h].double()
            logit = (qd @ kd.t()) * scale
            p = torch.softmax(logit.masked_fill(~seen, -float("inf")), dim=1)
            p = torch.where(seen, p, 0.0)
            o = p @ vd
            e = abs(scale) * 0.5 / (8355711.0 if f32 else 32639.0) * qd.abs().amax(1) * (kd.abs().sum(1).max() if len(kd) else 0.0)
            if len(kd):
                e = e + (0.0 if f32 else 2.0 ** -11) * abs(scale) * (qd.abs() @ kd.abs().t()).amax(1)
                e = e + 5 * 2.0 ** -24 * 1.4427 * torch.where(seen, logit, 0.0).abs().amax(1) + 2.0 ** -22
            weight = p @ vd.abs()
            least = (vd.abs().max() if len(vd) else 0.0) * 2.0 ** -29
            rel = 2 * e[:, None] + (2.0 ** -20 if f32 else 3 * 2.0 ** -11) + 2.0 ** -20
            out[s0:s0 + n, h] = torch.where(some[:, None], o, 0.0)
            bound[s0:s0 + n, h] = torch.where(some[:, None], rel * weight + least + (2.0 ** -23 if f32 else 2.0 ** -8) * o.abs(), 0.0)
    return out, bound
