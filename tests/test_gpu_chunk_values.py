"""Paged attention of chunks (bf16 sequences of more than 128 rows) on values at the
ends of their ranges.

The oracle is a plain softmax in 64 bits, a sequence and head at a time.  Beside each
value stands how far the kernel's arithmetic may be from it:
  k   fp16, in a unit in which 16 tokens' largest scale is 2^7 to 2^8: 2^-11 of an
      element, or half a subnormal's step, 2^-25 of 2^7 at least: 2^-32 of that scale
  v   fp16 of its scale's fp16 (2^-11 each), in a unit in which 16 tokens' largest scale
      is 2^5 to 2^6: 2^-30 of that scale from v's step and 2^-32 from a scale's own
  q   exact, but half a subnormal's step (2^-25 where the row's largest is 2^7 or more)
  p   fp16 in 2^14 at the row's largest: 2^-11 of it, or 2^-25 / 2^14 = 2^-39 of the
      largest p, for a v of up to 128 times the largest scale of the 16 tokens that it
      sees some of
  sums in fp32 (2^-20 of the sum of magnitudes), the logit's own roundings (five, in
  units of 2^-24) and exp2's, 2^-22; the output's bf16."""
import math

import pytest
import torch

import decoder_ref as R
import phi_qlinear as Q

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def groups_top(scales, codes, live):
    """Of [tokens] scales: the largest |scale| among a token's 16, of those that are live
    and have a nonzero code."""
    s = torch.where(live & codes.ne(0).any(dim=1), scales.double().abs(), 0.0)
    pad = -len(s) % 16
    top = torch.cat([s, torch.zeros(pad, dtype=s.dtype)]).view(-1, 16).max(dim=1)[0]
    return top.repeat_interleave(16)[:len(s)]


def rows_top(seen, top):
    """Of [rows, tokens] seen and groups_top: the largest of the 16 tokens that a row sees some of."""
    pad = -len(top) % 16
    seen = torch.nn.functional.pad(seen, (0, pad)).view(len(seen), -1, 16).any(2)
    return torch.where(seen, torch.nn.functional.pad(top, (0, pad)).view(-1, 16).max(1)[0], 0.0).max(1)[0]


def oracle(c, *, scale, causal=True, window=0):
    """(out, bound) in 64 bits; NaN for rows of no sequence and rows that see a scale of NaN."""
    q, k, v, ks, vs, table = (c[x] for x in ("q", "k", "v", "ks", "vs", "table"))
    T, Hq, D = q.shape
    blocks, H, page, _ = k.shape
    G = Hq // H
    out, bound = (torch.full((T, Hq, D), math.nan, dtype=torch.float64) for _ in range(2))
    for b, kv in enumerate(c["kv_len"]):
        s0, n = c["starts"][b], c["starts"][b + 1] - c["starts"][b]
        t = torch.arange(kv)
        blk = table[b][t // page].long() if kv else t
        live = (blk >= 0) & (blk < blocks)
        pos = kv - n + torch.arange(n)[:, None]
        seen = live[None, :].expand(n, -1)
        if causal:
            seen = seen & (t <= pos)
        if window:
            seen = seen & (t > pos - window)
        some = seen.any(0)
        blk, at = blk.clamp(0, blocks - 1), t % page
        for h in range(Hq):
            g = h // G
            if not bool(some.any()):
                out[s0:s0 + n, h], bound[s0:s0 + n, h] = 0.0, 0.0
                continue
            (kd, k_top), (vd, v_top) = (
                (torch.where(some[:, None], x[blk, g, at].double() * s[blk, g, at].double()[:, None], 0.0),
                 groups_top(s[blk, g, at], x[blk, g, at], some)) for x, s in ((k, ks), (v, vs)))
            qd = q[s0:s0 + n, h].double()
            logit = qd @ kd.T * scale
            p = torch.where(seen, torch.exp(logit - torch.where(seen, logit, -math.inf).max(1, keepdim=True)[0].clamp(min=-1e300)), 0.0)
            p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
            e = 2.0 ** -11 * (qd.abs() @ kd.abs().T) + 2.0 ** -32 * (qd.abs().sum(1)[:, None] * k_top + qd.abs().max(1)[0][:, None] * kd.abs().sum(1))
            # A weight is off by the factor of its own logit's error, their sum by the mean of
            # these; where that is past a half, every weight by the largest error twice.
            e = torch.where(seen, abs(scale) * e + 5 * 2.0 ** -24 * 1.4427 * logit.abs(), 0.0) + 2.0 ** -22
            twice, e = torch.expm1(2 * e.max(1)[0].clamp(max=100.0))[:, None], p * torch.expm1(e.clamp(max=100.0))
            weight, off = p @ vd.abs(), e.sum(1)[:, None]
            soft = torch.where(off < 0.5, (e @ vd.abs() + off * weight) / (1 - off).clamp(min=0.5), twice * weight)
            least = 2.0 ** -29 * (p @ v_top)[:, None] + 2.0 ** -39 * 256 * (rows_top(seen, v_top) * p.max(1)[0] * seen.sum(1))[:, None]
            o = p @ vd
            out[s0:s0 + n, h] = o
            bound[s0:s0 + n, h] = soft + (3 * 2.0 ** -11 + 2.0 ** -20) * weight + least + 2.0 ** -8 * o.abs()
    return out, bound


def run(dev, c, *, max_q=None, **kw):
    to = lambda t: torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=dev).copy_(t)  # noqa: E731
    cache = Q.KvCache(*(to(c[x]) for x in ("k", "v", "ks", "vs")))
    starts, lens = (torch.tensor(c[x], dtype=torch.int32, device=dev) for x in ("starts", "kv_len"))
    n = max(b - a for a, b in zip(c["starts"], c["starts"][1:]))
    got = Q.paged_attention(to(c["q"]), cache, c["table"].to(dev), starts, lens, max_q=max_q or n, max_kv=max(c["kv_len"]), **kw)
    return got.cpu()


def check(dev, c, *, max_q=None, out=None, **kw):
    assert (c["starts"][1] - c["starts"][0]) * (c["q"].shape[1] // c["k"].shape[1]) > 128
    kw.setdefault("scale", c["q"].shape[2] ** -0.5)
    got = run(dev, c, max_q=max_q, out=out, **kw)
    want, bound = oracle(c, **kw)
    err = (got.double() - want).abs()
    nan = want.isnan()
    assert torch.equal(got.isnan(), nan), f"{int(got.isnan().sum())} values are NaN, {int(nan.sum())} should be"
    worst = float((err / bound.clamp(min=1e-300))[~nan].max())
    assert worst <= 1.0, f"{worst:.3g} times the bound"
    return got


def case(lens, D=128, page=16, Hq=1, H=1, seed=1, **kw):
    return R.make_case(lens, Hq=Hq, H=H, D=D, page=page, dtype=BF16, seed=seed, **kw)


def place(c, b, t):
    """Token t of sequence b in the cache: an index of ks and vs (head 0)."""
    page = c["k"].shape[2]
    return int(c["table"][b, t // page]), 0, t % page


# ------------------------------------------------------------------ scales of v
@pytest.mark.parametrize("D,page", [(128, 16), (64, 8), (80, 24), (256, 64)])
@pytest.mark.parametrize("bits", [6, 10, 12, 14, 16, 20, 24])
def test_small_values_beside_large_ones(dev, D, page, bits):
    """One token of every 16 has values 2^bits of the others' and no weight to speak of."""
    c = case([(150, 500)], D=D, page=page, seed=bits)
    c["q"][:, 0, 0] = 16
    c["k"][..., 0] = 0
    c["vs"] = c["vs"].clamp(min=0.03) * 2.0 ** -bits
    for t in range(5, 500, 16):
        at = place(c, 0, t)
        c["k"][at] = 0
        c["k"][at][0], c["ks"][at], c["vs"][at] = -127, 0.5, 0.05
    check(dev, c)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("top", [2.0 ** 117, 2.0 ** 118, 1e36, 2.0 ** -100, 1e-31])
def test_largest_and_smallest_value_scales(dev, D, top):
    """Scales to 2^119.6, whose values to 2^126.6 fp32 holds, and down to 4e-33."""
    c = case([(140, 333)], D=D, seed=D)
    c["vs"] *= top / 0.052
    check(dev, c)


# ------------------------------------------------------------------ query rows of nothing
@pytest.mark.parametrize("D,page", [(64, 16), (128, 16), (128, 24), (80, 32), (256, 16), (192, 7)])
@pytest.mark.parametrize("n,kv", [(140, 228), (150, 150), (200, 1301), (130, 47)])
def test_zero_and_tiny_query_rows(dev, D, page, n, kv):
    """Equal weights for all that a row of zeros sees, wherever the last tile of 64 ends."""
    c = case([(n, kv)], D=D, page=page, seed=D + kv)
    for i, x in enumerate((0.0, 1e-8, 1e-12, 1e-20, 1e-30, 1e-38, -0.0)):
        c["q"][i::11] *= x
    check(dev, c)
    check(dev, c, causal=False)
    check(dev, c, window=33)


@pytest.mark.parametrize("page", [16, 8])
def test_zero_query_rows_over_holes(dev, page):
    """Whole groups of 16 tokens that are not there, at the ends of tiles and within them."""
    c = case([(160, 700), (140, 333)], page=page)
    c["q"][::2], c["q"][1::4] = 0, c["q"][1::4] * 1e-13
    c["table"][0, 32 // page:64 // page], c["table"][0, 400 // page], c["table"][1, 0:16 // page] = -1, 1 << 20, -5
    check(dev, c)


@pytest.mark.parametrize("q,k", [(1e-20, 1e-20), (1e-30, 1e30), (1e25, 1e-25), (1.0, 1e-33), (1e-12, 1e8)])
def test_units_of_q_and_k_apart(dev, q, k):
    """Rows and keys of sizes whose product is 1, or all but nothing, beside groups that are not there."""
    c = case([(140, 420)], page=8, seed=7)
    c["q"][::3] *= q
    c["ks"] *= k
    c["q"][1::3] *= min(1.0, 1.0 / k)
    c["q"][2::3] = 0
    c["table"][0, 4:10], c["table"][0, 30] = -1, -1
    check(dev, c)


# ------------------------------------------------------------------ vectors of zeros
@pytest.mark.parametrize("D,page", [(128, 16), (64, 8), (80, 24), (256, 16), (192, 7)])
@pytest.mark.parametrize("bits", [12, 16, 20, 30, 40, 90])
def test_zero_values_beside_small_ones(dev, D, page, bits):
    """A vector of zeros has the scale 1, whatever its neighbours have."""
    c = case([(150, 500)], D=D, page=page, seed=bits)
    c["vs"] *= 2.0 ** -bits
    for t in (*range(3, 500, 16), *range(200, 250)):
        at = place(c, 0, t)
        c["v"][at], c["vs"][at] = 0, 1.0
    check(dev, c)
    check(dev, c, window=100)


@pytest.mark.parametrize("size", [1.0, 1e-4, 1e-8, 1e-20])
def test_written_zero_vectors(dev, size):
    """As the cache's own quantiser writes them, keys of zeros among them too."""
    H, D, page, kv, n = 2, 128, 16, 400, 150
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn((kv, H, D), generator=g) for _ in range(2))
    v *= size
    for x in (k, v):
        x[torch.rand((kv, H), generator=g) < 0.1] = 0
    v[-70:-60] = 0
    cache = Q.kv_cache_empty(kv // page, page, H, D, dev)
    Q.kv_cache_write(cache, k.to(BF16).to(dev), v.to(BF16).to(dev), torch.arange(kv, device=dev))
    c = dict(q=torch.randn((n, 2 * H, D), generator=g).to(BF16), table=torch.arange(kv // page, dtype=torch.int32)[None],
             starts=[0, n], kv_len=[kv], **{x: t.cpu() for x, t in zip(("k", "v", "ks", "vs"), cache)})
    check(dev, c)


# ------------------------------------------------------------------ places that no row sees
@pytest.mark.parametrize("D,page", [(128, 16), (64, 8), (80, 24), (256, 16)])
@pytest.mark.parametrize("junk", [1e30, -1e30, 3e38, math.inf, math.nan])
def test_junk_below_the_window(dev, D, page, junk):
    """What lies before the first row's window, in its tile or far before it, may hold anything."""
    n, kv, window = 150, 700, 90
    c = case([(n, kv)], D=D, page=page, seed=D)
    for t in range(kv - n + 1 - window):
        c["ks"][place(c, 0, t)] = c["vs"][place(c, 0, t)] = junk
    check(dev, c, window=window)


@pytest.mark.parametrize("junk", [1e30, math.inf, math.nan])
def test_junk_past_the_end_and_in_other_blocks(dev, junk):
    c = case([(150, 300), (140, 190)], page=24, seed=3, blocks_extra=4)
    for x in ("ks", "vs"):
        c[x] = torch.where(c[x].isnan(), torch.full_like(c[x], junk), c[x])
    c["table"][0, 3] = -1
    check(dev, c)


# ------------------------------------------------------------------ far ends
@pytest.mark.parametrize("e", [126, 127])
def test_largest_query_rows(dev, e):
    """Rows whose largest element has bf16's largest exponents keep their logits' size."""
    c = case([(140, 333)], seed=e)
    scale = 2.0 ** -e
    c["q"][::2] = (c["q"][::2].float().clamp(-1.9, 1.9) * 2.0 ** e).to(BF16)
    c["q"][::2, 0, 0] = 1.5 * 2.0 ** e
    c["q"][1::2] = (c["q"][1::2].float() * 2.0 ** (e - 3)).to(BF16)
    check(dev, c, scale=scale)


# ------------------------------------------------------------------ a lone sequence of few rows
@pytest.mark.parametrize("n", [1, 5, 64, 128, 129, 0])
@pytest.mark.parametrize("kv", [300, 2500])
def test_lone_sequence_shorter_than_its_bound(dev, n, kv):
    """A buffer of 200 tokens of which q_start says that n are there: a prompt's last
    chunk.  One captured call serves all n; rows of no sequence are left as they are."""
    D, T = 128, 200
    c = case([(T, kv)], D=D, seed=n)
    to = lambda t: t.to(dev)  # noqa: E731
    cache = Q.KvCache(*(to(c[x]) for x in ("k", "v", "ks", "vs")))
    q, table, lens = to(c["q"]), to(c["table"]), torch.tensor([kv], dtype=torch.int32, device=dev)
    starts, out = torch.tensor([0, T], dtype=torch.int32, device=dev), torch.empty_like(q)
    ws = Q.paged_attention_workspace(T, 1, 1, D, 1, T, kv, BF16, dev)
    call = lambda: Q.paged_attention(q, cache, table, starts, lens, max_q=T, max_kv=kv, out=out, workspace=ws)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    c["starts"] = [0, n]
    want, bound = oracle(dict(c, q=c["q"][:n]), scale=D ** -0.5)
    for run_it in (call, graph.replay, call, graph.replay):
        starts.copy_(torch.tensor([0, n], dtype=torch.int32))
        out.fill_(7.0)
        run_it()
        got = out.cpu()
        assert bool(((got[:n].double() - want).abs() <= bound).all()) and bool((got[n:] == 7).all())
        starts[1] = T
        graph.replay()  # the whole buffer between


# ------------------------------------------------------------------ scales, strides, values that are not finite
@pytest.mark.parametrize("scale", [-0.3, 0.0, -0.0, 2.5, 40.0, 1e-30])
def test_scales(dev, scale):
    check(dev, case([(60, 200), (50, 70)], Hq=6, H=2, D=64, seed=2), scale=scale)


@pytest.mark.parametrize("lens", [[(140, 200)], [(150, 1500), (140, 150), (3, 2000)]])
def test_queries_and_output_in_wider_tensors(dev, lens):
    """Columns of wider tensors, q's and out's of different widths; what lies beside out stays."""
    c = case(lens, Hq=4, H=2, D=64, seed=2)
    T = c["starts"][-1]
    wide = torch.randn((T, 9, 64), generator=torch.Generator().manual_seed(1)).to(BF16)
    wide[:, 3:7] = c["q"]
    c["q"] = wide[:, 3:7]
    big = torch.full((T, 7, 72), 3.0, dtype=BF16, device=dev)
    check(dev, c, out=big[:, 1:5, :64])
    assert bool((big[:, 0] == 3).all()) and bool((big[:, 5:] == 3).all()) and bool((big[..., 64:] == 3).all())


@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_query_rows_that_are_not_finite(dev, page, bad):
    """Such a row is NaN, and no other."""
    c = case([(150, 420)], Hq=2, page=page, seed=6)
    c["q"][7, 1, 3] = c["q"][149, 0, 127] = bad
    got = run(dev, c, scale=0.1)
    want = torch.zeros((150, 2), dtype=torch.bool)
    want[7, 1] = want[149, 0] = True
    assert torch.equal(got.isnan(), want[:, :, None].expand_as(got))


@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("name", ["ks", "vs"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("window", [0, 40])
def test_cache_scales_that_are_not_finite(dev, page, name, bad, window):
    """The rows that see such a token are NaN, and only they."""
    n, kv, t = 200, 330, 201
    c = case([(n, kv)], page=page, seed=6)
    c[name][place(c, 0, t)] = bad
    got = run(dev, c, scale=0.1, window=window)
    pos = kv - n + torch.arange(n)
    want = (pos >= t) & ((pos - window < t) if window else True)
    assert torch.equal(got.isnan(), want[:, None, None].expand_as(got))


@pytest.mark.parametrize("D,page", [(64, 16), (128, 24), (256, 16)])
def test_peaks_and_wide_ranges(dev, D, page):
    """One token far above the rest (a sink), logits of thousands, v scales 30 powers of ten apart."""
    c = case([(200, 700)], D=D, page=page, seed=16)
    c["ks"][place(c, 0, 0)] = 0.25
    check(dev, c)
    check(dev, c, scale=40.0)
    for t in range(0, 700, 5):
        c["vs"][place(c, 0, t)] *= 10.0 ** -(t % 31)
    check(dev, c)
    c["vs"] *= 1e30
    check(dev, c)
    check(dev, c, causal=False)


@pytest.mark.parametrize("at,bits", [(333, 8), (333, 16), (333, 22), (256, 22), (256, 30), (256, 40), (256, 90)])
def test_small_values_before_large_ones(dev, at, bits):
    """Rows that see tokens of small v scales only, beside later tokens of large ones."""
    c = case([(400, 500)], seed=bits)
    for t in range(at):
        c["vs"][place(c, 0, t)] *= 2.0 ** -bits
    got = check(dev, c)
    # Against the same batch without the later tokens.
    n = at - 100
    alone = run(dev, dict(c, q=c["q"][:n], starts=[0, n], kv_len=[at]), scale=128 ** -0.5)
    want, bound = (x[:n] for x in oracle(c, scale=128 ** -0.5))
    assert bool(((alone.double() - want).abs() <= bound).all() and ((got[:n].double() - alone.double()).abs() <= 2 * bound).all())


@pytest.mark.parametrize("D", [64, 128, 256])
def test_large_values_that_windows_leave_behind(dev, D):
    """Windows of rows in one block that see large values, some, and none."""
    c = case([(300, 900)], D=D, seed=D)
    for t in range(900):
        c["vs"][place(c, 0, t)] *= 2.0 ** -(40 * (t // 16 % 20 != 0))
    check(dev, c, window=70)
    check(dev, c, window=200)
