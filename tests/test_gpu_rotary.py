"""GPU: rotary positions, alone and with the cache write, and copies of pages.

Tolerances.  A pair's cosine and sine are within 2^-22 (the angle's 32-bit
fraction of a turn, its conversion and product to fp32, and the series' roundings
are each under 2^-24); times the scale, one rounding, and a product, an fma: four of 2^-24
more on terms of at most scale (|a| + |b|).  So a turned element is within 2^-21 of
that magnitude, then its own rounding: 2^-24 or 2^-8 of the value.  What is quantised
is not rounded before: its scale is within 2^-20 of its 64-bit value and a code within
0.5 + 127 x 2^-19 < 0.501 of the quotient."""
import math

import pytest
import torch

import phi_qlinear as Q
import serving_ref as R

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
ROUND = {BF16: 2.0 ** -8, F32: 2.0 ** -24}


def randn(shape, seed, dtype=F32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def bits(t):
    return t.cpu().contiguous().view({2: torch.int16, 4: torch.int32, 1: torch.int8}[t.element_size()])


def same_bits(a, b):
    return a.dtype == b.dtype and torch.equal(bits(a), bits(b))


def positions_of(T, seed, far=1 << 20):
    g = torch.Generator().manual_seed(seed)
    p = torch.randint(-far, far, (T,), generator=g)
    p[0] = 0
    return p


CASES = [  # tokens, heads, dim, rot, dtype, far
    (1, 1, 2, 2, F32, 1000),
    (1, 32, 128, 128, BF16, 131072),
    (3, 5, 64, 64, BF16, 1 << 24),
    (17, 20, 80, 64, F32, 4352),
    (9, 3, 80, 40, BF16, 4096),
    (33, 7, 96, 96, F32, 1 << 30),
    (65, 4, 128, 32, BF16, 100000),
    (5, 2, 192, 192, BF16, 100000),
    (7, 3, 256, 256, F32, 100000),
    (4, 3, 576, 64, BF16, 100000),
    (2, 2, 1024, 1024, F32, 100000),
    (3, 2, 1023, 1000, BF16, 5000),
    (11, 3, 97, 20, BF16, 5000),
    (6, 2, 9, 8, F32, 5000),
    (8, 1, 1, None, F32, 1),
    (260, 1, 16, 16, BF16, 5000),
    (700, 40, 128, 128, BF16, 40000),
]


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("T,H,D,rot,dtype,far", CASES)
def test_rotary_against_64_bits(dev, T, H, D, rot, dtype, far, inter):
    if rot is None:
        with pytest.raises(Q.QLinearError, match="rotated"):
            Q.rotary(torch.zeros((T, H, D), device=dev), torch.zeros(T, dtype=torch.int64, device=dev),
                     torch.ones(1, dtype=torch.float64, device=dev))
        return
    x, pos, freq = randn((T, H, D), T + D, dtype), positions_of(T, D, far), Q.rotary_frequencies(rot, device="cpu")
    want, mag = R.rotated(x, pos, freq, inter, 1.25)
    got = Q.rotary(x.to(dev), pos.to(dev), freq.to(dev), interleaved=inter, scale=1.25)
    err = (got.cpu().double() - want).abs()
    assert bool((err <= 2.0 ** -21 * mag + ROUND[dtype] * want.abs() * (mag > 0)).all()), float((err - 2.0 ** -21 * mag).max())
    assert same_bits(got[..., rot:], x[..., rot:])


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("D,rot,dtype", [(128, 128, BF16), (128, 64, F32), (80, 40, BF16), (64, 20, F32), (50, 50, BF16)])
def test_rotary_strides_and_places(dev, D, rot, dtype, inter):
    """Columns of a wide buffer, heads outside, every offset, in place: the same bits as contiguous ones."""
    T, H = 37, 6
    x, pos, freq = randn((T, H, D), 3, dtype), positions_of(T, 4).to(dev), Q.rotary_frequencies(rot, device=dev)
    call = lambda x, **kw: Q.rotary(x, pos, freq, interleaved=inter, **kw)  # noqa: E731
    want = call(x.to(dev))
    for off in (0, 1, 2, 4, 8):
        wide = torch.full((T, (H + 2) * D + 8), 7.0, dtype=dtype, device=dev)
        part = wide[:, off:off + H * D].unflatten(1, (H, D))
        part.copy_(x)
        assert same_bits(call(part), want)
        assert call(part, out=part) is part and same_bits(part, want)
        assert bool((wide[:, :off] == 7).all()) and bool((wide[:, off + H * D:] == 7).all())
        assert same_bits(call(x.to(dev), out=part), want)
    outside = x.to(dev).transpose(0, 1).contiguous().transpose(0, 1)
    assert same_bits(call(outside), want) and same_bits(call(outside, out=outside), want)
    one = x[:, :1].to(dev).expand(T, H, D)  # one vector a token under all heads
    assert same_bits(call(one), call(x[:, :1].to(dev)).expand(T, H, D))
    # Columns of out beside x.
    both = torch.empty((T, H, 2 * D), dtype=dtype, device=dev)
    both[..., :D] = x.to(dev)
    assert same_bits(call(both[..., :D], out=both[..., D:]), want) and same_bits(both[..., :D], x)


def test_rotary_of_values_that_are_not_finite(dev):
    """They reach their own pair only."""
    x = randn((4, 2, 64), 1)
    x[1, 0, 3], x[2, 1, 40], x[3, 0, 60] = math.inf, math.nan, math.nan
    pos = torch.arange(4, device=dev)
    got = Q.rotary(x.to(dev), pos, Q.rotary_frequencies(48, device=dev)).cpu()
    bad = ~got.isfinite()
    want = torch.zeros_like(bad)
    want[1, 0, [3, 27]] = want[2, 1, [16, 40]] = want[3, 0, 60] = True
    assert torch.equal(bad, want)


def test_rotary_of_no_tokens(dev):
    e = torch.empty((0, 4, 64), dtype=BF16, device=dev)
    z = torch.empty(0, dtype=torch.int64, device=dev)
    f = Q.rotary_frequencies(64, device=dev)
    assert Q.rotary(e, z, f).shape == (0, 4, 64)
    c = Q.kv_cache_empty(4, 16, 2, 64, dev)
    assert Q.rotary_cache_write(c, e, e[:, :2], e[:, 2:], z, f, z).shape == (0, 4, 64)


def test_rotary_of_more_tokens_than_a_launch_has(dev):
    """2^24 + 50 tokens, a block each: the last of the first launch, and the second's."""
    T, D = (1 << 24) + 50, 513
    row = randn((1, 1, D), 4, BF16)
    pos, f = torch.arange(T, device=dev), Q.rotary_frequencies(512, device=dev)
    out = torch.full((T, 1, D), 7, dtype=BF16, device=dev)
    Q.rotary(row.to(dev).expand(T, 1, D), pos, f, out=out)
    for a, b in ((0, 3), ((1 << 24) - 30, T)):
        want = Q.rotary(row.to(dev).expand(b - a, 1, D).contiguous(), pos[a:b], f)
        assert same_bits(out[a:b], want)


def test_rotary_python_refusals(dev):
    x = torch.zeros((4, 2, 64), device=dev)
    pos, f = torch.arange(4, device=dev), Q.rotary_frequencies(64, device=dev)
    for kw in (dict(positions=pos.int()), dict(positions=pos[:3]), dict(freq=f.float()), dict(freq=f.cpu()),
               dict(x=x.transpose(1, 2)), dict(out=x.bfloat16()), dict(out=x[:3]), dict(positions=pos.repeat(2)[::2])):
        with pytest.raises(ValueError):
            Q.rotary(**{**dict(x=x, positions=pos, freq=f), **kw})
    with pytest.raises(Q.QLinearError):
        Q.rotary(x, pos, torch.ones(33, dtype=torch.float64, device=dev))


# ------------------------------------------------------------------ with the cache write
WRITES = [  # tokens, q heads, heads, dim, rot, page, dtype
    (1, 32, 8, 128, 128, 16, BF16),
    (64, 4, 2, 64, 64, 16, BF16),
    (77, 5, 1, 80, 80, 24, F32),
    (33, 6, 3, 96, 20, 7, BF16),
    (19, 8, 8, 256, 64, 1, F32),
    (50, 0, 2, 16, 16, 32, BF16),
    (9, 3, 3, 192, 192, 64, BF16),
    (40, 10, 2, 48, 24, 16, F32),
    (700, 40, 8, 128, 128, 64, BF16),
]


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("token_major", [False, True])
@pytest.mark.parametrize("T,Hq,H,D,rot,page,dtype", WRITES)
def test_cache_write_is_rotary_and_write(dev, T, Hq, H, D, rot, page, dtype, token_major, inter):
    """Bit for bit what rotary on fp32 and kv_cache_write make, and those against 64 bits."""
    blocks = -(-T // page) + 3
    qkv = randn((T, Hq + 2 * H, D), T, dtype)
    qkv[:, :, ::61] *= 6
    qkv = qkv.to(dev)
    q, k, v = qkv.split([Hq, H, H], dim=1)
    pos, freq = positions_of(T, 5).to(dev), Q.rotary_frequencies(rot, device=dev)
    slots = torch.randperm(blocks * page, generator=torch.Generator().manual_seed(T))[:T]
    slots[2::5] = -1
    if T > 8:
        slots[8] = blocks * page
    slots = slots.to(dev)

    def fresh():
        c = Q.kv_cache_empty(blocks, page, H, D, dev)
        if token_major:
            c = Q.KvCache(*(x.transpose(1, 2).contiguous().transpose(1, 2) for x in c))
        for x in c:
            x.fill_(77)
        return c

    a, b = fresh(), fresh()
    got = Q.rotary_cache_write(a, q if Hq else None, k, v, pos, freq, slots, interleaved=inter, scale=1.1)
    turned = Q.rotary(k.float(), pos, freq, interleaved=inter, scale=1.1)
    Q.kv_cache_write(b, turned, v.float(), slots)
    for x, y in zip(a, b):
        assert same_bits(x, y)
    if Hq:
        assert same_bits(got, Q.rotary(q, pos, freq, interleaved=inter, scale=1.1))
        assert Q.rotary_cache_write(a, q, k, v, pos, freq, slots, interleaved=inter, scale=1.1, out=q) is q and same_bits(q, got)
    else:
        assert got is None
    want, _ = R.rotated(k.cpu(), pos.cpu(), freq.cpu(), inter, 1.1)
    kept = (slots >= 0) & (slots < blocks * page)
    block, at = slots[kept].cpu() // page, slots[kept].cpu() % page
    codes, scales = a.k.cpu()[block, :, at].double(), a.k_scale.cpu()[block, :, at].double()
    s64 = want[kept.cpu()].abs().amax(-1) / 127
    assert bool(((scales - s64).abs() <= 2.0 ** -20 * s64).all())
    assert bool(((codes - want[kept.cpu()] / s64[..., None]).abs() <= 0.501).all())


def test_cache_write_of_values_that_are_not_finite(dev):
    """A vector with one has the scale NaN and codes 0, v's as k's, and its neighbours nothing of it."""
    x = randn((6, 2, 64), 8)
    x[1, 0, 5], x[2, 1, 63], x[4, 0, 0] = math.inf, math.nan, -math.inf
    c = Q.kv_cache_empty(1, 8, 2, 64, dev)
    pos, f = torch.arange(6, device=dev), Q.rotary_frequencies(32, device=dev)
    Q.rotary_cache_write(c, None, x.to(dev), x.to(dev), pos, f, pos)
    for s, codes in ((c.k_scale, c.k), (c.v_scale, c.v)):
        bad = s[0, :, :6].cpu().isnan()
        assert bad.nonzero().tolist() == [[0, 1], [0, 4], [1, 2]]
        assert not codes[0, :, :6].cpu()[bad].any() and bool((codes[0, :, :6].cpu()[~bad].abs().amax(-1) == 127).all())


# ------------------------------------------------------------------ copies
COPIES = [  # heads, page, dim, pairs
    (8, 16, 128, 16),
    (1, 1, 16, 5),
    (3, 24, 80, 7),
    (2, 7, 256, 9),
    (5, 64, 48, 3),
    (16, 256, 64, 2),
    (8, 64, 128, 40),
]


def random_cache(blocks, H, page, D, dev, seed, token_major=False):
    g = torch.Generator().manual_seed(seed)
    c = [torch.randint(-128, 128, (blocks, H, page, D), generator=g, dtype=torch.int8) for _ in range(2)]
    c += [torch.randn((blocks, H, page), generator=g) for _ in range(2)]
    if token_major:
        c = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in c]
    return Q.KvCache(*(torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device=dev).copy_(x) for x in c))


@pytest.mark.parametrize("part", [False, True])
@pytest.mark.parametrize("majors", [(False, False), (True, True), (False, True), (True, False)])
@pytest.mark.parametrize("H,page,D,n", COPIES)
def test_copy_between_caches(dev, H, page, D, n, majors, part):
    """Into another cache of another layout, and within one."""
    g = torch.Generator().manual_seed(n + page)
    a, b = (random_cache(2 * n + 3 + i, H, page, D, dev, i, majors[i]) for i in (0, 1))
    order = torch.randperm(2 * n + 3, generator=g)
    frm, to = order[:n].int(), order[n:2 * n].int()
    tokens = torch.randint(-1, page + 2, (n,), generator=g).int() if part else None
    if n > 4:
        frm[1], to[2], frm[3], to[4] = -1, 2 * n + 4, 2 * n + 3, -7
    for target in (b, a):
        want = [x.clone() for x in target]
        for i in range(n):
            m = page if tokens is None else max(0, min(page, int(tokens[i])))
            if 0 <= frm[i] < a.k.shape[0] and 0 <= to[i] < target.k.shape[0]:
                for x, y in zip(a, want):
                    y[to[i], :, :m] = x[frm[i], :, :m]
        Q.kv_cache_copy(a, target, frm.to(dev), to.to(dev), tokens=None if tokens is None else tokens.to(dev))
        for x, y in zip(target, want):
            assert same_bits(x, y)


def test_copy_of_more_pages_than_a_launch_has(dev):
    n = 5_700_000  # three blocks a page
    a, b = (Q.kv_cache_empty(n, 1, 1, 16, dev) for _ in range(2))
    for x in a:
        x.copy_(torch.arange(x.numel(), device=dev).view(x.shape) % 127)
    to = torch.arange(n, device=dev, dtype=torch.int32)
    Q.kv_cache_copy(a, b, to.flip(0), to, tokens=(to % 7 > 0).int())
    for x, y in zip(a, b):
        assert bool((x.flip(0) == y)[to % 7 > 0].all())


def test_copy_of_a_part_of_a_wider_cache(dev):
    """Heads of a wider cache: strides that no contiguous one has."""
    wide, a = random_cache(9, 6, 16, 64, dev, 1), random_cache(9, 2, 16, 64, dev, 2)
    part = Q.KvCache(*(x[:, 2:4] for x in wide))
    before = [x.clone() for x in wide]
    frm, to = torch.tensor([0, 5], dtype=torch.int32, device=dev), torch.tensor([8, 1], dtype=torch.int32, device=dev)
    Q.kv_cache_copy(a, part, frm, to)
    for x, y, z in zip(wide, before, a):
        y[[8, 1], 2:4] = z[[0, 5]]
        assert same_bits(x, y)


def test_copy_refusals(dev):
    a, b = random_cache(3, 2, 16, 64, dev, 1), random_cache(3, 2, 16, 48, dev, 1)
    i = torch.zeros(1, dtype=torch.int32, device=dev)
    with pytest.raises(Q.QLinearError, match="heads, page, dim"):
        Q.kv_cache_copy(a, b, i, i + 1)
    for kw in (dict(from_blocks=i.long()), dict(to_blocks=i.cpu()), dict(to_blocks=i.repeat(2)), dict(tokens=i.repeat(2))):
        with pytest.raises(ValueError):
            Q.kv_cache_copy(a, a, **{**dict(from_blocks=i, to_blocks=i + 1), **kw})


def test_pages_moved_together_keep_their_tokens(dev):
    """Forks, ends and a compaction on the device."""
    page, H, D = 8, 2, 32
    pages, c = Q.KvPages(24, page), Q.kv_cache_empty(24, page, H, D, dev)
    kept = {}

    def grow(seq, n, seed):
        x = randn((n, 2, H, D), seed).to(dev)
        slots = torch.tensor(pages.grow(seq, n), device=dev)
        pages.flush(c)
        Q.kv_cache_write(c, x[:, 0], x[:, 1], slots)
        kept.setdefault(seq, []).append([y.clone() for y in Q.kv_cache_read(c, slots)])

    def check():
        pages.flush(c)
        for seq, want in kept.items():
            slots = [pages.of[seq][t // page] * page + t % page for t in range(pages.length[seq])]
            got = Q.kv_cache_read(c, torch.tensor(slots, device=dev))
            for i in range(2):
                assert same_bits(got[i], torch.cat([w[i] for w in want]))

    grow("a", 19, 1), grow("b", 40, 2)
    for child in "cd":
        pages.fork("a", child)
        kept[child] = list(kept["a"])
    grow("c", 9, 3), grow("a", 1, 4), grow("d", 30, 5)
    check()
    pages.end("b"), kept.pop("b")
    pages.fork("d", "e")
    kept["e"] = list(kept["d"])
    pages.compact()
    grow("e", 3, 6)
    check()


# ------------------------------------------------------------------ streams and graphs
def test_calls_on_a_stream_and_in_a_graph(dev):
    """Replayed after its inputs changed in place, and on a stream of its own: the eager bits."""
    T, Hq, H, D, page = 40, 8, 2, 64, 16
    qkv, pos = randn((T, Hq + 2 * H, D), 1, BF16).to(dev), positions_of(T, 2).to(dev)
    q, k, v = qkv.split([Hq, H, H], dim=1)
    freq, slots = Q.rotary_frequencies(D, device=dev), torch.arange(T, device=dev)
    cache, want_cache = (random_cache(8, H, page, D, dev, 3) for _ in range(2))
    frm, to = torch.tensor([0, 1], dtype=torch.int32, device=dev), torch.tensor([5, 6], dtype=torch.int32, device=dev)
    out, turned = torch.empty((T, Hq, D), dtype=BF16, device=dev), torch.empty((T, H, D), dtype=BF16, device=dev)

    def step(cache, out, turned, stream=None):
        Q.rotary_cache_write(cache, q, k, v, pos, freq, slots, out=out, stream=stream)
        Q.rotary(k, pos, freq, interleaved=True, out=turned, stream=stream)
        Q.kv_cache_copy(cache, cache, frm, to, stream=stream)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    step(cache, out, turned, side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(cache, out, turned)
    for i in range(3):
        qkv.copy_(randn((T, Hq + 2 * H, D), 10 + i, BF16))
        pos.add_(977)
        want = torch.empty_like(out), torch.empty_like(turned)
        step(want_cache, *want)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert same_bits(out, want[0]) and same_bits(turned, want[1])
        for x, y in zip(cache, want_cache):
            assert same_bits(x, y)
