"""GPU: the operators between a decoder layer's int8 linears
(phi_hip_rms_norm_quant, phi_hip_kv_cache_write / _read,
phi_hip_paged_attention) against plain 64-bit forms.

Tolerances.  Norm: the stored residual is one rounded sum (exact).  The row's
factor 1/sqrt(mean) is a fp32 sum of up to 32768 squares by lanes and a tree
(under 2^-18 of it, so 2^-19 of the factor); a rotated value adds four passes of
four roundings on partial sums of at most 16 times the row's largest rotated
value: 16 x 16 x 2^-24 = 1.6e-5 of it.  So the scale is within 2e-5 of its
64-bit value, a code within 0.5 + 127 x 4e-5 < 0.51 of the 64-bit quotient.  Against
the library's own quantiser on the norm's fp32 output the codes and scales
are exact.  Cache: exact.  Attention: decoder_ref.attention derives a bound
for each value from the arithmetic that the header states."""
import math

import pytest
import torch

import decoder_ref as R
import phi_qlinear as Q

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def randn(shape, seed, dtype=F32, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def same_bits(a, b):
    t = {2: torch.int16, 4: torch.int32, 1: torch.int8}[a.element_size()]
    return a.dtype == b.dtype and torch.equal(a.cpu().contiguous().view(t), b.cpu().contiguous().view(t))


# ------------------------------------------------------------------ norm
NORMS = [  # rows, K, x, residual, weight, shift, rotate
    (1, 256, BF16, None, F32, False, True),
    (1, 4096, BF16, BF16, BF16, False, True),
    (3, 1, F32, F32, F32, True, False),
    (2, 17, BF16, F32, None, True, False),
    (5, 255, F32, BF16, F32, False, False),
    (7, 512, F32, F32, BF16, True, True),
    (4, 768, BF16, F32, None, False, True),
    (9, 1023, BF16, BF16, F32, True, False),
    (67, 1280, F32, None, None, False, True),
    (6, 5003, F32, F32, F32, True, False),
    (5, 5120, BF16, F32, F32, False, True),
    (130, 4352, F32, BF16, F32, True, True),
    (3, 8192, BF16, F32, BF16, True, True),
    (2, 16384, F32, F32, F32, False, True),
    (3, 17000, BF16, BF16, F32, False, False),
    (2, 24832, BF16, F32, F32, True, True),
    (2, 32767, F32, F32, F32, True, False),
    (2, 32768, BF16, BF16, BF16, False, True),
]


def norm_inputs(rows, K, xd, rd, wd, shift, seed, pad=0):
    x = randn((rows, K + pad), seed, xd)[:, :K]
    x[:, ::61] *= 8
    res = None if rd is None else randn((rows, K + pad), seed + 1, rd, 3.0)[:, :K]
    w = None if wd is None else (1 + randn((K,), seed + 2, F32, 0.2)).to(wd)
    sh = randn((K,), seed + 3, wd or F32, 0.3) if shift else None
    return x, res, w, sh


def run_norm(dev, x, w, res, sh, eps=1e-6, **kw):
    to = lambda t: None if t is None else torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=dev).copy_(t)  # noqa: E731
    x, w, res, sh = to(x), to(w), to(res), to(sh)
    out = None if res is None else torch.empty_strided(res.shape, res.stride(), dtype=res.dtype, device=dev)
    q, s = Q.rms_norm_quant(x, w, eps, residual=res, residual_out=out, shift=sh, **kw)
    torch.cuda.synchronize()
    return q.cpu(), s.cpu(), None if out is None else out.cpu()


@pytest.mark.parametrize("rows,K,xd,rd,wd,shift,rotate", NORMS)
def test_norm_against_64_bits(dev, rows, K, xd, rd, wd, shift, rotate):
    x, res, w, sh = norm_inputs(rows, K, xd, rd, wd, shift, seed=K)
    y = torch.full((rows, K), math.nan, dtype=F32, device=dev)
    q, s, out = run_norm(dev, x, w, res, sh, rotate=rotate, y=y)
    r64, y64, z = R.norm(x, w, sh, res, 1e-6, rotate)
    if res is not None:
        assert same_bits(out, (x.float() + res.float()).to(rd))
    # y: the factor's 2^-19 and four roundings of its own.
    mag = (y64 - (0 if sh is None else sh.double())).abs() + (0 if sh is None else sh.double().abs())
    assert bool(((y.cpu().double() - y64).abs() <= mag * 2.0 ** -18 + 1e-30).all())
    s64 = z.abs().amax(dim=1) / 127
    assert bool(((s.double() - s64).abs() <= 2e-5 * s64).all())
    assert bool(((q.double() - z / s64[:, None]).abs() <= 0.51).all())
    if K % 256 == 0 and K <= 24576:
        q2, s2 = Q.quant_rotate(y, rotate=rotate)
        assert same_bits(q, q2) and same_bits(s, s2)


@pytest.mark.parametrize("K,rotate", [(512, True), (1280, True), (1000, False), (777, False)])
@pytest.mark.parametrize("pad", [0, 1, 8])
def test_norm_pitches_outputs_and_rounding(dev, K, rotate, pad):
    """Odd pitches (rows that start at any element), a bf16 y, in place, qmax 7
    and ties to even, codes at an odd pitch."""
    rows = 11
    x, res, w, sh = norm_inputs(rows, K, BF16, F32, F32, True, seed=K + pad, pad=pad)
    _, _, z = R.norm(x, w, sh, res, 1e-5, rotate)
    qb = torch.full((rows, K + 3), 99, dtype=torch.int8, device=dev)
    y = torch.empty((rows, K + pad), dtype=BF16, device=dev)[:, :K]
    y32 = torch.empty((rows, K), dtype=F32, device=dev)
    dx, dr, dw, ds = x.to(dev), torch.empty((rows, K + pad), device=dev)[:, :K].copy_(res), w.to(dev), sh.to(dev)
    dx = torch.empty((rows, K + pad), dtype=BF16, device=dev)[:, :K].copy_(x)
    q, s = Q.rms_norm_quant(dx, dw, 1e-5, residual=dr, shift=ds, rotate=rotate, qmax=7.0,
                            round_mode=Q.ROUND_HALF_EVEN, q=qb[:, :K], y=y)
    _, _ = Q.rms_norm_quant(dx, dw, 1e-5, residual=dr, residual_out=dr, shift=ds, rotate=rotate, y=y32)
    torch.cuda.synchronize()
    assert same_bits(dr, x.float() + res)  # in place, once
    assert same_bits(y, y32.to(BF16))
    s64 = z.abs().amax(dim=1) / 7
    assert bool(((s.cpu().double() - s64).abs() <= 2e-5 * s64).all())
    assert bool(((q.cpu().double() - z / s64[:, None]).abs() <= 0.501).all())
    assert bool((qb[:, K:] == 99).all())


@pytest.mark.parametrize("K,rotate", [(512, True), (4096, True), (1000, False), (20480, True)])
def test_norm_odd_rows(dev, K, rotate):
    """A row of zeros (with and without eps), rows with an infinity or a NaN, tiny and huge rows."""
    x = randn((8, K), 5)
    x[1] = 0
    x[2, K // 2] = math.inf
    x[3, K - 1] = math.nan
    x[4] *= 1e-25
    x[5] *= 1e17
    x[6] *= 3e18  # its squares sum to 1e37 K, past fp32 from K = 35
    q, s, _ = run_norm(dev, x, None, None, None, rotate=rotate)
    assert math.isnan(s[2]) and math.isnan(s[3]) and not q[2].any() and not q[3].any()
    assert s[1] == 1 and not q[1].any()
    _, _, z = R.norm(x, None, None, None, 1e-6, rotate)
    for i in (0, 5, 7):
        s64 = z[i].abs().max() / 127
        assert abs(s[i].double() - s64) <= 2e-5 * s64
        assert bool(((q[i].double() - z[i] / s64).abs() <= 0.51).all())
    s64 = z[4].abs().max() / 127  # 1e-22: far under eps, over the quantiser's 1e-30
    assert abs(s[4].double() - s64) <= 2e-5 * s64
    assert math.isnan(s[6]) or abs(s[6].double() - z[6].abs().max() / 127) <= 2e-5 * z[6].abs().max() / 127
    q, s, _ = run_norm(dev, x[1:2], None, None, None, eps=0.0, rotate=rotate)
    assert math.isnan(s[0])  # 0 / 0


def test_norm_same_on_another_stream_and_twice(dev):
    x, res, w, _ = norm_inputs(64, 2048, BF16, F32, F32, False, seed=1)
    x, res, w = x.to(dev), res.to(dev), w.to(dev)
    a = Q.rms_norm_quant(x, w, 1e-6, residual=res)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    b = Q.rms_norm_quant(x, w, 1e-6, residual=res, stream=st)
    torch.cuda.synchronize()
    assert same_bits(a[0], b[0]) and same_bits(a[1], b[1])
    empty = Q.rms_norm_quant(x[:0], w, 1e-6)
    assert empty[0].shape == (0, 2048)


# ------------------------------------------------------------------ cache
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T,H,D,page,major", [(1, 1, 16, 1, False), (5, 3, 64, 8, False), (33, 2, 80, 24, True),
                                             (17, 8, 128, 16, False), (300, 4, 96, 32, True), (9, 1, 256, 7, False),
                                             (129, 5, 176, 64, False)])
def test_cache_write_and_read(dev, T, H, D, page, major, dtype):
    """Codes, scales and values to the bit, from columns of a wider tensor, into a
    cache of either order, some tokens without a slot; nothing else is written."""
    g = torch.Generator().manual_seed(T * D)
    blocks = T // page + 3
    qkv = (torch.randn((T, 4 * H, D), generator=g) * torch.rand((T, 4 * H, 1), generator=g) * 4).to(dtype)
    qkv[T // 2, :, :] = 0
    k, v = qkv[:, H:2 * H], qkv[:, 3 * H:]
    slots = torch.randperm(blocks * page, generator=g)[:T].clone()
    if T > 4:
        slots[3], slots[4] = -1, blocks * page  # neither has a place
    kc, vc = (torch.full((blocks, H, page, D), 77, dtype=torch.int8, device=dev) for _ in range(2))
    ks, vs = (torch.full((blocks, H, page), -5.0, device=dev) for _ in range(2))
    if major:
        kc, vc = (torch.full((blocks, page, H, D), 77, dtype=torch.int8, device=dev).permute(0, 2, 1, 3) for _ in range(2))
        ks, vs = (torch.full((blocks, page, H), -5.0, device=dev).permute(0, 2, 1) for _ in range(2))
    cache = Q.KvCache(kc, vc, ks, vs)
    d = qkv.to(dev)
    Q.kv_cache_write(cache, d[:, H:2 * H], d[:, 3 * H:], slots.to(dev))
    rk, rv = Q.kv_cache_read(cache, slots.to(dev), out_dtype=dtype)
    torch.cuda.synchronize()
    live = (slots >= 0) & (slots < blocks * page)
    for x, codes, scales, back in ((k, kc, ks, rk), (v, vc, vs, rv)):
        c, s = R.quantise_f32(x)
        want_c = torch.full((blocks, H, page, D), 77, dtype=torch.int8)
        want_s = torch.full((blocks, H, page), -5.0)
        want_c[slots[live] // page, :, slots[live] % page] = c[live]
        want_s[slots[live] // page, :, slots[live] % page] = s[live]
        assert torch.equal(codes.cpu(), want_c) and torch.equal(scales.cpu(), want_s)
        val = torch.where(live[:, None, None], c.float() * s[..., None], torch.zeros(()))
        assert torch.equal(back.cpu(), val.to(dtype))


def test_cache_not_finite_and_empty(dev):
    H, D, page = 2, 64, 16
    cache = Q.kv_cache_empty(2, page, H, D, dev)
    x = randn((4, H, D), 3, BF16)
    x[1, 0, 5], x[2, 1, 9] = math.inf, math.nan
    slots = torch.arange(4)
    Q.kv_cache_write(cache, x.to(dev), x.to(dev), slots.to(dev))
    k, v = Q.kv_cache_read(cache, slots.to(dev))
    k, v = k.cpu(), v.cpu()
    assert bool(k[1, 0].isnan().all()) and bool(k[2, 1].isnan().all()) and not bool(k[1, 1].isnan().any())
    assert not cache.k[0, 0, 1].any() and same_bits(k, v)
    Q.kv_cache_write(cache, x[:0].to(dev), x[:0].to(dev), slots[:0].to(dev))
    assert Q.kv_cache_read(cache, slots[:0].to(dev))[0].shape == (0, H, D)


# ------------------------------------------------------------------ attention
def run_attention(dev, c, *, max_q=None, max_kv=None, scale=None, out=None, stream=None, **kw):
    D = c["q"].shape[2]
    n = [b - a for a, b in zip(c["starts"], c["starts"][1:])]
    to = lambda t: torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=dev).copy_(t)  # noqa: E731
    cache = Q.KvCache(*(to(c[x]) for x in ("k", "v", "ks", "vs")))
    q, table = to(c["q"]), c["table"].to(dev)
    starts, lens = (torch.tensor(c[x], dtype=torch.int32, device=dev) for x in ("starts", "kv_len"))
    torch.cuda.synchronize()
    got = Q.paged_attention(q, cache, table, starts, lens, max_q=max_q or max(n),
                            max_kv=max(c["kv_len"]) if max_kv is None else max_kv,
                            scale=D ** -0.5 if scale is None else scale, out=out, stream=stream, **kw)
    torch.cuda.synchronize()
    return got


def check_attention(dev, c, *, scale=None, causal=True, window=0, **kw):
    D = c["q"].shape[2]
    got = run_attention(dev, c, scale=scale, causal=causal, window=window, **kw)
    want, bound = R.attention(c["q"], c["k"], c["v"], c["ks"], c["vs"], c["table"], c["starts"], c["kv_len"],
                              scale=D ** -0.5 if scale is None else scale, causal=causal, window=window)
    err = (got.cpu().double() - want).abs()
    worst = float((err / bound.clamp(min=1e-300)).max())
    assert bool((err <= bound).all()), f"{worst:.3g} times the bound"
    return got


ATTENTION = [  # lens, Hq, H, D, page, window
    ([(1, 1)], 1, 1, 16, 1, 0),
    ([(1, 63)], 4, 4, 64, 16, 0),
    ([(1, 64), (1, 65), (1, 0), (1, 200)], 8, 2, 128, 16, 0),
    ([(1, 777)], 32, 8, 128, 16, 0),
    ([(1, 300), (1, 129), (1, 31), (1, 1)], 7, 1, 80, 24, 0),
    ([(1, 1500), (1, 700)], 16, 1, 256, 64, 100),
    ([(1, 259)], 40, 2, 96, 7, 0),
    ([(1, 500), (1, 33)], 12, 4, 192, 128, 0),
    ([(2, 3), (3, 90), (1, 17)], 6, 2, 64, 8, 0),
    ([(5, 70), (4, 4)], 10, 2, 128, 16, 33),
    ([(16, 16), (9, 140), (33, 40)], 4, 2, 112, 32, 0),
    ([(40, 300), (1, 77), (64, 64)], 8, 2, 128, 16, 0),
    ([(130, 257)], 3, 3, 80, 24, 50),
    ([(150, 150), (7, 333)], 4, 1, 256, 16, 0),
    ([(70, 71)], 16, 1, 48, 256, 0),
    ([(3, 2), (4, 0), (2, 2)], 2, 1, 64, 16, 0),  # more new tokens than the cache holds: empty rows
]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lens,Hq,H,D,page,window", ATTENTION)
def test_attention_against_64_bits(dev, lens, Hq, H, D, page, window, dtype):
    c = R.make_case(lens, Hq=Hq, H=H, D=D, page=page, dtype=dtype, seed=D + Hq, token_major=D % 64 != 0)
    check_attention(dev, c, window=window)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lens", [[(1, 90), (1, 5)], [(20, 90), (3, 3)], [(140, 200)]])
def test_attention_without_the_causal_mask(dev, lens, dtype):
    c = R.make_case(lens, Hq=4, H=2, D=64, page=16, dtype=dtype, seed=9)
    check_attention(dev, c, causal=False)


@pytest.mark.parametrize("lens", [[(1, 9000)], [(1, 4097), (1, 100), (1, 0)], [(17, 3000)], [(2, 2500), (1, 2499)]])
def test_attention_long_axis(dev, lens):
    """Lengths at which the tokens are split over blocks and joined."""
    c = R.make_case(lens, Hq=4, H=2, D=64, page=16, dtype=BF16, seed=4)
    check_attention(dev, c)
    c = R.make_case(lens, Hq=2, H=1, D=128, page=64, dtype=F32, seed=5)
    check_attention(dev, c, max_kv=c["table"].shape[1] * 64)


def test_attention_holes_and_bad_table_entries(dev):
    """Entries that are no block of the cache are tokens that are not there."""
    for lens in ([(1, 200), (1, 40)], [(30, 200), (9, 40)]):
        c = R.make_case(lens, Hq=4, H=1, D=128, page=16, dtype=BF16, seed=8)
        c["table"][0, 2], c["table"][0, 5], c["table"][1, :] = -1, 1 << 30, c["k"].shape[0]
        got = check_attention(dev, c)
        assert not bool(got[lens[0][0]:].any())  # the second sequence has no token left


def test_attention_strides_scale_and_untouched_rows(dev):
    """q and out as columns of wider tensors, a negative and a zero scale, rows of no sequence left alone."""
    lens = [(3, 50), (1, 33), (20, 60)]
    for scale in (-0.3, 0.0, 2.5):
        c = R.make_case(lens, Hq=6, H=2, D=64, page=16, dtype=BF16, seed=2)
        wide = torch.randn((24, 10, 64), generator=torch.Generator().manual_seed(1)).to(BF16)
        wide[:, 2:8] = c["q"]
        c["q"] = wide[:, 2:8]
        big = torch.full((24, 9, 64), 3.0, dtype=BF16, device=dev)
        check_attention(dev, c, scale=scale, out=big[:, 1:7])
        assert bool((big[:, 0] == 3).all()) and bool((big[:, 7:] == 3).all())
    c = R.make_case(lens, Hq=2, H=1, D=64, page=16, dtype=BF16, seed=3)
    q = torch.cat([c["q"], torch.ones((2, 2, 64), dtype=BF16)])
    out = torch.full(q.shape, 5.0, dtype=BF16, device=dev)
    c["q"] = q
    check = run_attention(dev, c, out=out)
    assert bool((check[24:] == 5).all())


@pytest.mark.parametrize("n,kv", [(1, 70), (40, 70)])
def test_attention_not_finite(dev, n, kv):
    """A NaN row of q is a NaN row of out and no other; a NaN or infinite scale of a
    token shows in the rows that see it, and only there."""
    c = R.make_case([(n, kv)], Hq=2, H=1, D=64, page=16, dtype=BF16, seed=6)
    c["q"][0, 1, 3] = math.nan
    got = run_attention(dev, c).cpu()
    assert bool(got[0, 1].isnan().all()) and not bool(got[0, 0].isnan().any()) and not bool(got[1:].isnan().any())
    if n > 1:
        for name in ("ks", "vs"):
            c = R.make_case([(n, kv)], Hq=2, H=1, D=64, page=16, dtype=BF16, seed=6)
            t = kv - n + 5  # seen from row 5 on
            c[name][c["table"][0, t // 16], 0, t % 16] = math.nan
            got = run_attention(dev, c).cpu()
            assert not bool(got[:5].isnan().any()) and bool(got[5:].isnan().any(dim=2).all())


@pytest.mark.parametrize("n,kv", [(1, 3000), (64, 700)])
def test_attention_peaks_and_large_logits(dev, n, kv):
    """One token far above the rest (a sink): the rest still count; logits of
    thousands; v scales from 1e-30 to 1e30."""
    c = R.make_case([(n, kv)], Hq=2, H=1, D=64, page=16, dtype=BF16, seed=16)
    c["ks"][c["table"][0, 0], 0, 0] = 0.25
    check_attention(dev, c)
    check_attention(dev, c, scale=40.0)
    c["vs"][c["table"][0, 0], 0, 0] = 1e-30
    check_attention(dev, c)
    c["vs"] *= 1e30
    check_attention(dev, c)


def test_attention_repeats_to_the_bit(dev):
    for lens in ([(1, 5000), (1, 300)], [(64, 2000), (1, 900)]):
        c = R.make_case(lens, Hq=8, H=2, D=128, page=16, dtype=BF16, seed=12)
        a = run_attention(dev, c)
        assert same_bits(a, run_attention(dev, c))
        assert same_bits(a, run_attention(dev, c, stream=torch.cuda.Stream()))


def test_attention_nothing_to_do(dev):
    c = R.make_case([(2, 20)], Hq=2, H=1, D=64, page=16, dtype=BF16, seed=1)
    c["kv_len"] = [0]
    assert not bool(run_attention(dev, c, max_kv=0).any())
    cache = Q.KvCache(*(c[x].to(dev) for x in ("k", "v", "ks", "vs")))
    z = torch.zeros(1, dtype=torch.int32, device=dev)
    assert Q.paged_attention(c["q"][:0].to(dev), cache, c["table"][:0].to(dev), z, z[:0], max_q=0, max_kv=0).shape[0] == 0


# ------------------------------------------------------------------ together
def test_write_then_attend_matches_attention_on_the_values(dev):
    """Chunks and single tokens of two sequences written as they come and attended to."""
    H, G, D, page = 2, 3, 128, 16
    cache = Q.kv_cache_empty(20, page, H, D, dev)
    for t in cache[2:]:
        t.fill_(math.nan)
    table = torch.randperm(20, generator=torch.Generator().manual_seed(0))[:16].reshape(2, 8).to(torch.int32)
    dt, lens = table.to(dev), [0, 0]
    ks, vs = [[], []], [[], []]
    for step, new in enumerate([(40, 7), (1, 1), (1, 20), (1, 1)]):
        T = sum(new)
        qkv = randn((T, (G + 2) * H, D), 100 + step, BF16)
        slots, row = [], 0
        for b in range(2):
            for i in range(new[b]):
                t = lens[b] + i
                slots.append(int(table[b, t // page]) * page + t % page)
            c, s = R.quantise_f32(qkv[row:row + new[b], G * H:(G + 1) * H])
            ks[b].append(c.double() * s.double()[..., None])
            c, s = R.quantise_f32(qkv[row:row + new[b], (G + 1) * H:])
            vs[b].append(c.double() * s.double()[..., None])
            lens[b] += new[b]
            row += new[b]
        d = qkv.to(dev)
        Q.kv_cache_write(cache, d[:, G * H:(G + 1) * H], d[:, (G + 1) * H:], torch.tensor(slots, device=dev))
        got = Q.paged_attention(d[:, :G * H], cache, dt, torch.tensor([0, new[0], T], dtype=torch.int32, device=dev),
                                torch.tensor(lens, dtype=torch.int32, device=dev), max_q=max(new), max_kv=128).cpu()
        row = 0
        for b in range(2):
            k, v = torch.cat(ks[b]), torch.cat(vs[b])
            for i in range(new[b]):
                n = lens[b] - new[b] + i + 1
                for h in range(G * H):
                    p = torch.softmax((k[:n, h // G] @ qkv[row, h].double()) * D ** -0.5, dim=0)
                    want = p @ v[:n, h // G]
                    # bf16 out, p at 11 bits, the logits' error under 2^-10 at these sizes
                    bound = 2.0 ** -8 * want.abs() + (2.0 ** -9 + 2.0 ** -11) * (p @ v[:n, h // G].abs())
                    assert bool(((got[row, h].double() - want).abs() <= bound).all())
                row += 1
