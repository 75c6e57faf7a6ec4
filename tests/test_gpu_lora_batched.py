"""GPU: the adapters of many requests (phi_hip_lora_batched) against 64 bits.

Tolerance.  A sum of n fp32 terms in any order is within n 2^-24 of its terms'
magnitudes; a matrix instruction may drop bits where terms of one step meet, at most
one 2^-23 of the step's largest a term.  So h is within (2 K + 16) 2^-24, the
second product within (6 R + 16) 2^-24 (three terms of h), of the sum of magnitudes
through both, which is taken whole here; the scale and base add 2^-23 of the result's parts,
the output's rounding 2^-24 or 2^-8 of the value."""
import math

import pytest
import torch

import phi_qlinear as Q
import serving_ref as R

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
ROUND = {BF16: 2.0 ** -8, F32: 2.0 ** -24}


def randn(shape, seed, dtype=F32, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def bits(t):
    return t.cpu().contiguous().view({2: torch.int16, 4: torch.int32}[t.element_size()])


def same_bits(a, b):
    return a.dtype == b.dtype and torch.equal(bits(a), bits(b))


def inputs(M, K, N, rank, n, xd, wd, od, seed=0, mixed=True):
    x, base = randn((M, K), seed, xd), randn((M, N), seed + 1, od)
    A, B = randn((n, rank, K), seed + 2, wd, K ** -0.5), randn((n, N, rank), seed + 3, wd, rank ** -0.5)
    g = torch.Generator().manual_seed(seed + 4)
    adapter = torch.randint(-2, n + 1, (M,), generator=g) if mixed else torch.arange(M) * n // M
    return x, A, B, adapter.int(), torch.rand(n, generator=g) + 0.5, base


def near(got, want, mag, base, K, rank):
    part = 0 if base is None else base.double().abs()
    tol = mag * (2 * K + 6 * rank + 32) * 2.0 ** -24 + (mag + part) * 2.0 ** -23 + ROUND[got.dtype] * want.abs()
    err = (got.cpu().double() - want).abs()
    return bool((err <= tol).all()), float((err - tol).max())


SIZES = [  # rows, K, N, ranks, adapters, mixed
    (1, 64, 64, 16, 1, True),
    (1, 4096, 512, 16, 40, False),
    (64, 512, 256, 16, 32, True),
    (64, 512, 272, 8, 100, True),
    (65, 256, 1000, 32, 3, True),
    (130, 264, 96, 33, 2, False),
    (33, 100, 77, 5, 4, True),
    (200, 31, 33, 1, 1, True),
    (31, 1, 1, 1, 2, True),
    (300, 1024, 640, 64, 5, False),
    (70, 640, 528, 128, 9, True),
    (50, 96, 300, 256, 3, True),
    (40, 333, 160, 200, 70, True),
    (1000, 512, 1536, 64, 8, False),
    (640, 777, 333, 16, 3, False),
    (515, 1030, 100, 40, 90, True),
    (900, 600, 1300, 7, 2, True),
    (512, 544, 96, 256, 4, False),
    (600, 511, 200, 16, 5, False),
    (2100, 520, 60, 32, 1, False),
    (1100, 520, 333, 40, 5, True),
    (1030, 777, 200, 256, 3, False),
    (1025, 512, 96, 200, 90, True),
    (1500, 1030, 700, 33, 6, False),
    (1024, 512, 64, 64, 1, False),
]


@pytest.mark.parametrize("xd,wd,od", [(BF16, BF16, BF16), (F32, F32, F32), (BF16, F32, BF16), (F32, BF16, F32), (BF16, BF16, F32),
                                      (F32, F32, BF16)])
@pytest.mark.parametrize("M,K,N,rank,n,mixed", SIZES)
def test_against_64_bits(dev, M, K, N, rank, n, mixed, xd, wd, od):
    x, A, B, adapter, scale, base = inputs(M, K, N, rank, n, xd, wd, od, seed=M + K, mixed=mixed)
    to = lambda t: t.to(dev)  # noqa: E731
    for s, b in ((scale, base), (None, None)):
        want, mag = R.adapted(x, A, B, adapter, s, b)
        got = Q.lora_batched(to(x), to(A), to(B), to(adapter), scale=None if s is None else to(s), base=None if b is None else to(b), out_dtype=od)
        assert got.dtype == od
        fine, by = near(got, want, mag, b, K, rank)
        assert fine, by
        none = (adapter < 0) | (adapter >= n)
        if bool(none.any()):
            assert same_bits(got[none.to(dev)], torch.zeros_like(got[none.to(dev)]) if b is None else b[none])


@pytest.mark.parametrize("wd", [BF16, F32])
def test_rows_do_not_depend_on_their_neighbours(dev, wd):
    """The same row under other mixtures of adapters, and beside rows and factors that are not finite."""
    x, A, B, adapter, scale, base = (t.to(dev) for t in inputs(128, 512, 256, 16, 6, BF16, wd, BF16, mixed=True))
    adapter.clamp_(0, 5)
    want = Q.lora_batched(x, A, B, adapter, scale=scale, base=base)
    for a in range(6):
        alone = torch.where(adapter == a, adapter, torch.full_like(adapter, -1))
        got = Q.lora_batched(x, A, B, alone, scale=scale, base=base)
        mine = adapter == a
        assert same_bits(got[mine], want[mine]) and same_bits(got[~mine], base[~mine])
    x2, A2, B2 = x.clone(), A.clone(), B.clone()
    x2[5], A2[3], B2[4] = math.nan, math.inf, math.nan
    keep = (adapter != 3) & (adapter != 4)
    keep[5] = False
    got = Q.lora_batched(x2, A2, B2, adapter, scale=scale, base=base)
    assert same_bits(got[keep], want[keep])
    assert bool(got[5].isnan().all()) and bool(got[(adapter == 4) & (torch.arange(128, device=dev) != 5)].isnan().all())


@pytest.mark.parametrize("wd", [BF16, F32])
def test_values_that_pass_fp32(dev, wd):
    """An infinite A x meets B as such: infinities of B's signs, NaN at its zeros."""
    x = torch.full((2, 64), 2.0 ** 120, dtype=BF16, device=dev)
    A = torch.full((1, 8, 64), 2.0 ** 10, dtype=wd, device=dev)
    A[:, 1:] = 0
    B = torch.zeros((1, 32, 8), dtype=wd, device=dev)
    B[0, 1, 0], B[0, 2, 0] = 1.0, -1.0
    got = Q.lora_batched(x, A, B, torch.tensor([0, -1], dtype=torch.int32, device=dev), out_dtype=F32)
    assert got[0, 1] == math.inf and got[0, 2] == -math.inf and bool(got[0, 3:].isnan().all()) and not got[1].any()


@pytest.mark.parametrize("off", [1, 8])
@pytest.mark.parametrize("wd,od", [(BF16, BF16), (F32, F32)])
def test_strides_and_places(dev, off, wd, od):
    """Columns of wider buffers, factors with pitches, base updated in place, neighbours left alone."""
    M, K, N, rank, n = 70, 264, 336, 24, 4
    x, A, B, adapter, scale, base = (t.to(dev) for t in inputs(M, K, N, rank, n, BF16, wd, od))
    want = Q.lora_batched(x, A, B, adapter, scale=scale, base=base)

    def within(t, extra):
        wide = torch.full((*t.shape[:-1], t.shape[-1] + off + extra), 9.0, dtype=t.dtype, device=dev)
        part = wide[..., off:off + t.shape[-1]]
        part.copy_(t)
        return wide, part

    (_, xs), (_, As), (_, Bs), (wide, bs) = within(x, 3), within(A, 8), within(B, 5), within(base, 7)
    assert same_bits(Q.lora_batched(xs, As, Bs, adapter, scale=scale, base=bs), want)
    assert Q.lora_batched(xs, As, Bs, adapter, scale=scale, base=bs, out=bs) is bs and same_bits(bs, want)
    assert bool((wide[:, :off] == 9).all()) and bool((wide[:, off + N:] == 9).all())
    # One set of factors for all adapters, and adapters inside out.
    one = Q.lora_batched(x, A[:1].expand(n, -1, -1), B[:1].expand(n, -1, -1), adapter, scale=scale, base=base)
    assert same_bits(one, Q.lora_batched(x, A[:1].repeat(n, 1, 1), B[:1].repeat(n, 1, 1), adapter, scale=scale, base=base))
    turned = A.transpose(0, 1).contiguous().transpose(0, 1), B.transpose(0, 1).contiguous().transpose(0, 1)
    assert same_bits(Q.lora_batched(x, *turned, adapter, scale=scale, base=base), want)


def test_agrees_with_the_tail(dev):
    """One adapter for all rows: lora_tail's result but for the order of sums."""
    M, K, N, rank = 100, 512, 384, 16
    x, A, B, _, _, base = (t.to(dev) for t in inputs(M, K, N, rank, 1, F32, F32, F32))
    got = Q.lora_batched(x, A, B, torch.zeros(M, dtype=torch.int32, device=dev), base=base)
    tail = Q.lora_tail(x, A[0], B[0], base.clone())
    _, mag = R.adapted(x.cpu(), A.cpu(), B.cpu(), torch.zeros(M, dtype=torch.int32), None, None)
    assert bool(((got - tail).cpu().double().abs() <= mag * (4 * K + 12 * rank) * 2.0 ** -24 + base.cpu().abs() * 2.0 ** -22).all())


def test_of_no_rows_and_refusals(dev):
    x, A, B, adapter, scale, base = (t.to(dev) for t in inputs(4, 64, 32, 8, 2, BF16, BF16, BF16))
    assert Q.lora_batched(x[:0], A, B, adapter[:0]).shape == (0, 32)
    args = dict(x=x, A=A, B=B, adapter=adapter, scale=scale, base=base)
    for kw in (dict(A=A.float()), dict(A=A[0]), dict(B=B[:1]), dict(adapter=adapter.long()), dict(adapter=adapter[:3]), dict(scale=scale.double()),
               dict(base=base[:3]), dict(out_dtype=F32), dict(A=A.transpose(1, 2)), dict(x=x.t()), dict(scale=scale.cpu()), dict(out=base.float())):
        with pytest.raises(ValueError):
            Q.lora_batched(**{**args, **kw})
    with pytest.raises(Q.QLinearError, match="overlap"):
        Q.lora_batched(x, A, B, adapter, base=x[:, :32], out=x[:, 16:48])
    with pytest.raises(Q.QLinearError, match="workspace"):
        Q.lora_batched(**args, workspace=torch.empty(16, dtype=torch.uint8, device=dev))
    with pytest.raises(Q.QLinearError, match="exceeds"):
        Q.lora_batched(x, A.repeat(1, 33, 1), B.repeat(1, 1, 33), adapter)


def test_on_a_stream_and_in_graphs(dev):
    """Two captured calls that share a workspace, replayed on changed inputs, and a call on a stream of its own."""
    M, K, N, rank, n = 48, 1024, 512, 16, 7
    x, A, B, adapter, scale, base = (t.to(dev) for t in inputs(M, K, N, rank, n, BF16, BF16, BF16))
    ws = Q.lora_batched_workspace(M, K, rank, dev)
    outs = [torch.empty_like(base) for _ in range(2)]

    flipped = A.flip(0)
    call = lambda i, out, **kw: Q.lora_batched(x, (A, flipped)[i], B, adapter, scale=scale, base=base, out=out, **kw)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    call(0, outs[0], stream=side)
    torch.cuda.synchronize()
    assert same_bits(outs[0], call(0, torch.empty_like(base)))
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(i, outs[i], workspace=ws)
        graphs.append(g)
    for k in range(3):
        x.copy_(randn((M, K), 50 + k, BF16))
        adapter.copy_(torch.randint(-1, n, (M,), generator=torch.Generator().manual_seed(k)).int())
        want = [call(i, torch.empty_like(base)) for i in range(2)]
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(same_bits(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("M,K,rank", [(130, 48, 4), (600, 512, 4), (1100, 512, 40)])
def test_adapters_of_one_place_in_the_table(dev, M, K, rank):
    """Numbers that agree in their low bits, in every tile, few rows and many."""
    n = 4200
    x, A, B, _, scale, base = inputs(M, K, 40, rank, n, BF16, BF16, BF16)
    i = torch.arange(M)
    adapter = ((i * 7 % 5) * 1024 + i % 3 - 1).int()  # -1 to 4097
    got = Q.lora_batched(*(t.to(dev) for t in (x, A, B, adapter)), scale=scale.to(dev), base=base.to(dev))
    want, mag = R.adapted(x, A, B, adapter, scale, base)
    fine, by = near(got, want, mag, base, K, rank)
    assert fine, by


@pytest.mark.parametrize("off", [1, 8])
@pytest.mark.parametrize("wd,od,rank", [(BF16, BF16, 24), (BF16, BF16, 72), (F32, F32, 40), (BF16, F32, 256), (F32, BF16, 200)])
def test_many_rows_in_place_and_strided(dev, off, wd, od, rank):
    M, K, N, n = 1100, 520, 333, 5
    x, A, B, adapter, scale, base = (t.to(dev) for t in inputs(M, K, N, rank, n, BF16, wd, od))
    want = Q.lora_batched(x, A, B, adapter, scale=scale, base=base)
    exact, mag = R.adapted(*(t.cpu() for t in (x, A, B, adapter, scale, base)))
    fine, by = near(want, exact, mag, base.cpu(), K, rank)
    assert fine, by

    def within(t):
        wide = torch.full((*t.shape[:-1], t.shape[-1] + off + 3), 9.0, dtype=t.dtype, device=dev)
        part = wide[..., off:off + t.shape[-1]]
        part.copy_(t)
        return wide, part

    (_, xs), (_, As), (_, Bs), (wide, bs) = within(x), within(A), within(B), within(base)
    assert Q.lora_batched(xs, As, Bs, adapter, scale=scale, base=bs, out=bs) is bs and same_bits(bs, want)
    assert bool((wide[:, :off] == 9).all()) and bool((wide[:, off + N:] == 9).all())


def test_many_rows_do_not_depend_on_their_neighbours(dev):
    x, A, B, adapter, scale, base = (t.to(dev) for t in inputs(1050, 576, 300, 48, 6, BF16, BF16, BF16))
    adapter.clamp_(0, 5)
    want = Q.lora_batched(x, A, B, adapter, scale=scale, base=base)
    for a in range(6):
        mine = adapter == a
        got = Q.lora_batched(x, A, B, torch.where(mine, adapter, torch.full_like(adapter, 6)), scale=scale, base=base)
        assert same_bits(got[mine], want[mine]) and same_bits(got[~mine], base[~mine])
    x2, A2 = x.clone(), A.clone()
    x2[7], A2[2] = math.nan, math.inf
    keep = adapter != 2
    keep[7] = False
    assert same_bits(Q.lora_batched(x2, A2, B, adapter, scale=scale, base=base)[keep], want[keep])


def test_many_rows_in_a_graph(dev):
    """Captured in place, replayed on other adapters and activations, eager work between."""
    M, K, N, rank, n = 1040, 512, 384, 64, 3
    x, A, B, adapter, scale, base = (t.to(dev) for t in inputs(M, K, N, rank, n, BF16, BF16, BF16))
    ws, out = Q.lora_batched_workspace(M, K, rank, dev), base.clone()
    call = lambda o: Q.lora_batched(x, A, B, adapter, scale=scale, base=o, out=o, workspace=ws)  # noqa: E731
    call(out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(out)
    for k in range(3):
        x.copy_(randn((M, K), 70 + k, BF16))
        adapter.copy_(torch.randint(-1, n + 1, (M,), generator=torch.Generator().manual_seed(k)).int())
        want = call(base.clone())
        out.copy_(base)
        g.replay()
        torch.cuda.synchronize()
        assert same_bits(out, want)
