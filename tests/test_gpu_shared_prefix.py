"""GPU: attention of sequences that share prefixes (phi_hip_paged_attention_shared)
against a plain softmax in 64 bits; serving_ref.shared_attention derives each value's
bound from the arithmetic that the headers state."""
import math

import pytest
import torch

import phi_qlinear as Q
import serving_ref as R

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def same_bits(a, b):
    t = {2: torch.int16, 4: torch.int32}[a.element_size()]
    return a.dtype == b.dtype and torch.equal(a.cpu().contiguous().view(t), b.cpu().contiguous().view(t))


def arguments(dev, c, **kw):
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    to = lambda t: torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=dev).copy_(t)  # noqa: E731
    new = [b - a for a, b in zip(c["starts"], c["starts"][1:])]
    got = dict(q=to(c["q"]), cache=Q.KvCache(*(to(c[x]) for x in ("k", "v", "ks", "vs"))), prefix_table=c["prefix_table"].to(dev),
               prefix_len=i32(c["prefix_len"]), group_start=i32(c["group_start"]), block_table=c["table"].to(dev), q_start=i32(c["starts"]),
               kv_len=i32(c["kv_len"]), max_prefix=max(c["prefix_len"]), max_q=max(new), max_kv=max(c["kv_len"]))
    return {**got, **kw}


def check(dev, c, scale=None, **kw):
    scale = c["q"].shape[2] ** -0.5 if scale is None else scale
    got = Q.paged_attention_shared(**arguments(dev, c, scale=scale, **kw))
    want, bound = R.shared_attention(c, scale)
    err = (got.cpu().double() - want).abs()
    there = ~want.isnan().any(-1).any(-1)
    assert bool((err[there] <= bound[there]).all()), f"{float((err / bound.clamp(min=1e-300))[there].max()):.3g} times the bound"
    return got


CASES = [  # groups, free, Hq, H, D, page
    ([(1, [(1, 1)])], [], 1, 1, 16, 1),
    ([(40, [(1, 5), (1, 20)])], [], 4, 2, 64, 16),
    ([(777, [(1, 30)] * 4)], [], 8, 2, 128, 16),
    ([(200, [(1, 0)] * 3)], [(1, 9)], 4, 1, 64, 16),
    ([(0, [(1, 7), (2, 40)]), (65, [(3, 3)])], [], 4, 2, 80, 24),
    ([(300, [(1, i) for i in range(1, 41)])], [(1, 0), (1, 50)], 8, 2, 64, 16),
    ([(1000, [(1, 17)] * 70), (30, [(2, 90)] * 3)], [], 4, 1, 128, 64),
    ([(64, [(5, 5), (33, 40)]), (129, [(1, 1)]), (7, [(2, 300), (70, 70)])], ([(2, 8)], [(3, 64)]), 10, 2, 96, 32),
    ([(500, [(150, 200), (1, 3)])], [], 4, 2, 128, 16),
    ([(90, [(140, 140)])], [(1, 700)], 2, 1, 256, 16),
    ([(3000, [(1, 2000), (1, 10), (4, 500)])], [], 6, 2, 192, 128),
    ([(100, [(3, 2), (4, 0)])], [(3, 1)], 2, 1, 64, 16),  # more new tokens than the own part holds
    ([(50, []), (60, [(1, 4)]), (70, [])], [], 4, 4, 48, 8),  # groups of nobody
]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("groups,free,Hq,H,D,page", CASES)
def test_against_64_bits(dev, groups, free, Hq, H, D, page, dtype):
    c = R.shared_case(groups, free, Hq=Hq, H=H, D=D, page=page, dtype=dtype, seed=D + Hq, token_major=D % 64 != 0)
    check(dev, c)


@pytest.mark.parametrize("rows", [16, 128, 129, 256, 257, 600])
def test_at_the_kernels_borders(dev, rows):
    """Groups of as many rows as one tile, one kernel, or one more has."""
    c = R.shared_case([(321, [(1, 33)] * rows)], [(1, 5)], Hq=1, H=1, D=64, page=16, dtype=BF16, seed=rows)
    check(dev, c)


@pytest.mark.parametrize("prefix", [9000, 40000])
def test_long_prefixes(dev, prefix):
    """Lengths at which both parts are split over many blocks."""
    c = R.shared_case([(prefix, [(1, 700), (1, 1), (1, 3)] * 15), (prefix // 3, [(1, 5000)])], [], Hq=4, H=1, D=64, page=64, dtype=BF16, seed=2)
    check(dev, c)
    c = R.shared_case([(prefix, [(1, 300), (2, 40)])], [], Hq=4, H=2, D=128, page=16, dtype=F32, seed=3)
    check(dev, c)


def test_is_attention_over_both_tables_joined(dev):
    """Beside paged_attention of the same sequences with the prefix' blocks first in their
    tables, and groups that pages of forked sequences give."""
    H, D, page, G = 2, 128, 16, 4
    pages, cache = Q.KvPages(400, page), Q.kv_cache_empty(400, page, H, D, dev)
    slots = pages.grow(0, 1000)
    gen = torch.Generator().manual_seed(1)
    rand = lambda *s: torch.randn(s, generator=gen).to(BF16).to(dev)  # noqa: E731
    Q.kv_cache_write(cache, rand(1000, H, D), rand(1000, H, D), torch.tensor(slots, device=dev))
    for s in range(1, 50):
        pages.fork(0, s)
    pages.flush(cache)
    seqs = list(range(50))
    new = torch.tensor([pages.grow(s, 1 + s % 3) [-1] for s in seqs], device=dev)
    lens = [pages.length[s] for s in seqs]
    for s in seqs:  # the tokens before the last of each are written too
        at = torch.tensor([pages.of[s][t // page] * page + t % page for t in range(1000, lens[s])], device=dev)
        Q.kv_cache_write(cache, rand(len(at), H, D), rand(len(at), H, D), at)
    assert new.numel() == 50
    q = rand(50, H * G, D)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    width = max(len(pages.of[s]) for s in seqs)
    table = i32([pages.of[s] + [-1] * (width - len(pages.of[s])) for s in seqs])
    starts = i32(list(range(51)))
    want = Q.paged_attention(q, cache, table, starts, i32(lens), max_q=1, max_kv=max(lens)).float()
    n = pages.shared(seqs)
    assert n == 1000 // page
    got = Q.paged_attention_shared(q, cache, table[:1, :n], i32([n * page]), i32([0, 50]), table[:, n:], starts, i32([x - n * page for x in lens]),
                                   max_prefix=n * page, max_q=1, max_kv=max(lens) - n * page).float()
    # Both within their bounds of the same values: bf16's rounding and 2^-9 of the weights (|v| to 5) each.
    assert float((got - want).abs().max()) <= 2 * (2.0 ** -8 * float(want.abs().max()) + 2.0 ** -9 * 5)
    assert float((got - want).norm() / want.norm()) < 2.0 ** -8


def test_holes_scales_and_rows_left_alone(dev):
    for rows in (2, 150):
        c = R.shared_case([(200, [(1, 40)] * rows)], [], Hq=4, H=2, D=64, page=16, dtype=BF16, seed=8)
        c["prefix_table"][0, 2], c["prefix_table"][0, 5], c["table"][0, 0], c["table"][1, :] = -1, 1 << 30, c["k"].shape[0], -5
        for scale in (-0.3, 0.0, 2.5):
            check(dev, c, scale=scale)
        c["prefix_table"][:] = -1
        assert not bool(check(dev, c)[1].any())
    # max_q below a sequence's rows, rows past the last sequence, columns of wider tensors, a wider table.
    c = R.shared_case([(70, [(3, 20), (6, 31)])], [(1, 5)], Hq=4, H=2, D=64, page=16, dtype=BF16, seed=4)
    want = check(dev, c)
    wide = torch.full((12, 8, 64), 5.0, dtype=BF16, device=dev)
    qw = torch.zeros((12, 6, 64), dtype=BF16, device=dev)
    qw[:10, 1:5] = c["q"].to(dev)
    got = Q.paged_attention_shared(**arguments(dev, c, q=qw[:, 1:5], out=wide[:, 2:6], max_q=4))
    assert got.data_ptr() == wide[:, 2:6].data_ptr()
    assert same_bits(got[:7], want[:7]) and bool((got[7:9] == 5).all()) and same_bits(got[9], want[9]) and bool((got[10:] == 5).all())
    assert bool((wide[:, :2] == 5).all()) and bool((wide[:, 6:] == 5).all())
    # max_prefix below the length: tokens past it are not seen.
    short = Q.paged_attention_shared(**arguments(dev, c, max_prefix=33)).cpu().double()
    want, bound = R.shared_attention(dict(c, prefix_len=[33]), 0.125)
    assert bool(((short - want).abs() <= bound).all())


@pytest.mark.parametrize("rows", [3, 140])
def test_not_finite(dev, rows):
    """NaN in q is NaN of its own row; a NaN scale in a prefix is NaN of its group's rows, in
    own tokens of that sequence's."""
    c = R.shared_case([(100, [(1, 20)] * rows), (40, [(1, 20)] * 2)], [], Hq=2, H=1, D=64, page=16, dtype=BF16, seed=6)
    c["q"][0, 1, 3] = math.nan
    got = Q.paged_attention_shared(**arguments(dev, c)).cpu()
    assert bool(got[0, 1].isnan().all()) and int(got.isnan().any(-1).sum()) == 1
    for name in ("ks", "vs"):
        for prefix in (True, False):
            c = R.shared_case([(100, [(1, 20)] * rows), (40, [(1, 20)] * 2)], [], Hq=2, H=1, D=64, page=16, dtype=BF16, seed=6)
            block = c["prefix_table"][0, 1] if prefix else c["table"][1, 0]
            c[name][block, 0, 5] = math.nan
            bad = Q.paged_attention_shared(**arguments(dev, c)).cpu().isnan().any(-1).all(-1)
            want = torch.zeros(rows + 2, dtype=torch.bool)
            want[(slice(0, rows) if prefix else 1)] = True
            assert torch.equal(bad, want)


def test_repeats_to_the_bit(dev):
    c = R.shared_case([(2500, [(1, 300)] * 40), (600, [(5, 77)] * 3)], [(1, 800)], Hq=8, H=2, D=128, page=16, dtype=BF16, seed=12)
    a = Q.paged_attention_shared(**arguments(dev, c))
    assert same_bits(a, Q.paged_attention_shared(**arguments(dev, c)))
    args = arguments(dev, c)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    b = Q.paged_attention_shared(**args, stream=side)
    side.synchronize()
    assert same_bits(a, b)


def test_one_workspace_after_other_calls(dev):
    """What an earlier call left in the workspace means nothing to a later one."""
    big = R.shared_case([(500, [(1, 300)] * 40), (60, [(5, 77)] * 3)], [(1, 80)], Hq=4, H=1, D=64, page=16, dtype=BF16, seed=1)
    small = R.shared_case([(50, [(1, 3)])], [(1, 8), (1, 0), (2, 9)], Hq=4, H=1, D=64, page=16, dtype=BF16, seed=2)
    n = Q.load().phi_hip_paged_attention_shared_workspace_bytes(56, 4, 1, 64, 2, 44, 500, 5, 300, Q.BF16)
    for fill in (0, 0xff, 0x01):
        ws = torch.full((n,), fill, dtype=torch.uint8, device=dev)
        for c in (big, small, big):
            want = Q.paged_attention_shared(**arguments(dev, c))
            assert same_bits(Q.paged_attention_shared(**arguments(dev, c, workspace=ws)), want)
    # Rows behind the last sequence keep what they held, whatever was left for them.
    args = arguments(dev, big)
    out = torch.full(big["q"].shape, 4.0, dtype=BF16, device=dev)
    Q.paged_attention_shared(**{**args, "q_start": args["q_start"].clamp(max=30)}, out=out, workspace=ws)
    assert bool((out[30:] == 4).all()) and not bool((out[:30] == 4).all(-1).any())


def test_captured_with_growing_sequences(dev):
    """Two graphs that share a workspace, replayed with other lengths, tables and groups, each
    against the eager call."""
    cases = [R.shared_case([(300 + 50 * i, [(1, 20 + i)] * (35 + i)), (40, [(1, 9 + i)] * (5 - i))], [], Hq=4, H=1, D=64, page=16, dtype=BF16,
                           seed=20 + i) for i in range(3)]
    blocks = max(c["k"].shape[0] for c in cases)
    widths = [max(c[t].shape[1] for c in cases) for t in ("prefix_table", "table")]
    for c in cases:
        for name in ("k", "v", "ks", "vs"):
            c[name] = torch.cat([c[name], c[name][:1].expand(blocks - c[name].shape[0], *c[name].shape[1:])])
        for name, w in zip(("prefix_table", "table"), widths):
            c[name] = torch.nn.functional.pad(c[name], (0, w - c[name].shape[1]), value=-1)
    bounds = dict(max_prefix=400, max_q=1, max_kv=32)
    state = arguments(dev, cases[0], **bounds)
    n = Q.load().phi_hip_paged_attention_shared_workspace_bytes(40, 4, 1, 64, 2, 40, 400, 1, 32, Q.BF16)
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    outs = [torch.empty_like(state["q"]) for _ in range(2)]
    for out, s in zip(outs, (0.125, 0.25)):
        Q.paged_attention_shared(**state, out=out, workspace=ws, scale=s)
    torch.cuda.synchronize()
    graphs = []
    for out, s in zip(outs, (0.125, 0.25)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            Q.paged_attention_shared(**state, out=out, workspace=ws, scale=s)
        graphs.append(g)
    for c in (*cases, cases[0]):
        fresh = arguments(dev, c, **bounds)
        for name in ("q", "prefix_table", "prefix_len", "group_start", "block_table", "q_start", "kv_len"):
            state[name].copy_(fresh[name])
        for x, y in zip(state["cache"], fresh["cache"]):
            x.copy_(y)
        want = [Q.paged_attention_shared(**fresh, scale=s) for s in (0.125, 0.25)]
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(same_bits(a, b) for a, b in zip(outs, want))


def test_nothing_to_do_and_refusals(dev):
    c = R.shared_case([(40, [(1, 5), (1, 20)])], [], Hq=4, H=2, D=64, page=16, dtype=BF16, seed=1)
    args = arguments(dev, c)
    z = torch.zeros(1, dtype=torch.int32, device=dev)
    assert Q.paged_attention_shared(**{**args, "q": args["q"][:0], "block_table": args["block_table"][:0], "q_start": z, "kv_len": z[:0], "max_q": 0}).shape[0] == 0
    empty = arguments(dev, dict(c, prefix_len=[0], kv_len=[0, 0]))
    assert not bool(Q.paged_attention_shared(**empty).any())
    for kw in (dict(prefix_len=args["prefix_len"].long()), dict(group_start=args["group_start"][:1]), dict(kv_len=args["kv_len"].cpu()),
               dict(prefix_table=args["prefix_table"].repeat(2, 1)), dict(block_table=args["block_table"].t()), dict(q=args["q"][..., :32]),
               dict(out=args["q"].float())):
        with pytest.raises(ValueError):
            Q.paged_attention_shared(**{**args, **kw})
    for kw, text in ((dict(max_prefix=1000), "prefix table"), (dict(max_kv=1000), "block table"), (dict(max_q=3), "out of range"),
                     (dict(scale=math.inf), "scale"), (dict(out=args["q"]), "overlap"), (dict(workspace=torch.empty(64, dtype=torch.uint8, device=dev)), "workspace")):
        with pytest.raises(Q.QLinearError, match=text):
            Q.paged_attention_shared(**{**args, **kw})


def test_past_32_bits_of_cache(dev):
    """Blocks behind 2^32 bytes: written, copied to the first ones and seen, to the same bits."""
    H, page, D, n = 2, 64, 256, 3
    blocks = (1 << 32) // (H * page * D) + 4
    c = Q.kv_cache_empty(blocks, page, H, D, dev)
    T = n * page
    k, v = (torch.randn((T, H, D), generator=torch.Generator().manual_seed(i)).to(dev, BF16) for i in (1, 2))
    pos, freq = torch.arange(T, device=dev), Q.rotary_frequencies(D, device=dev)
    high = torch.arange(blocks - n, blocks, dtype=torch.int32, device=dev)
    low = torch.arange(n, dtype=torch.int32, device=dev)
    Q.rotary_cache_write(c, None, k, v, pos, freq, (high.long()[:, None] * page + torch.arange(page, device=dev)).flatten())
    Q.kv_cache_copy(c, c, high, low)
    for x in c:
        assert torch.equal(x[low.long()].view(torch.uint8), x[high.long()].view(torch.uint8))
    q = torch.randn((40, 4, D), generator=torch.Generator().manual_seed(3)).to(dev, BF16)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    got = [Q.paged_attention_shared(q, c, t[None, :2], i32(2 * page), i32(0, 2), t[None, 2:].expand(2, -1).contiguous(), i32(0, 20, 40), i32(page, 33),
                                    max_prefix=2 * page, max_q=20, max_kv=page) for t in (low, high)]
    assert same_bits(*got) and bool(got[0].any())
