"""Paged attention on the GPU where batches are split, mixed and replayed: tiles of
many rows, more sequences than a wave has lanes, splits of uneven lengths, windows
over them, and captured graphs of growing sequences.

The oracle is a plain softmax in 64 bits over the cache's values, a sequence and
head at a time; the bounds beside it follow from the stated arithmetic."""
import math

import pytest
import torch

import decoder_ref as R
import phi_qlinear as Q

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
FEW = 128  # rows (new tokens x heads a key/value head) up to which k, v and q are exact integers


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return "cuda"


def oracle(c, *, scale, causal=True, window=0):
    """(out, bound) in 64 bits; NaN for rows of no sequence.

    q k: half a step of q's integers a product, or (many rows) k's rounding to 11
    bits, at least 2^-23 of the largest |k|; five roundings of the logit in 32 bits.
    p v: every weight off by the logits' error, p's 11 (fp32 q: 21) bits; many rows:
    v's scale and v rounded to 11 bits, at least 2^-22 of the largest |v|, and
    weights below 2^-39 of the largest lost.  Then the sums and the output's type."""
    q, k, v, ks, vs, table = (c[x] for x in ("q", "k", "v", "ks", "vs", "table"))
    T, Hq, D = q.shape
    blocks, H, page, _ = k.shape
    G, f32 = Hq // H, q.dtype == F32
    out, bound = (torch.full((T, Hq, D), math.nan, dtype=torch.float64) for _ in range(2))
    for b, kv in enumerate(c["kv_len"]):
        s0, n = c["starts"][b], c["starts"][b + 1] - c["starts"][b]
        t = torch.arange(kv)
        blk = table[b][t // page].long() if kv else t
        pos = kv - n + torch.arange(n)[:, None]
        seen = ((blk >= 0) & (blk < blocks))[None, :].expand(n, -1)
        if causal:
            seen = seen & (t <= pos)
        if window:
            seen = seen & (t > pos - window)
        at, few = (blk.clamp(0, blocks - 1), t % page), f32 or n * G <= FEW
        for h in range(Hq):
            g = h // G
            kd, vd = (torch.where(seen.any(0)[:, None], x[at[0], g, at[1]].double() * s[at[0], g, at[1]].double()[:, None], 0.0)
                      for x, s in ((k, ks), (v, vs)))
            qd = q[s0:s0 + n, h].double()
            if kv == 0:
                out[s0:s0 + n, h], bound[s0:s0 + n, h] = 0.0, 0.0
                continue
            logit = (qd @ kd.T) * scale
            p = torch.where(seen, torch.exp(logit - torch.where(seen, logit, -math.inf).max(1, keepdim=True)[0].clamp(min=-1e300)), 0.0)
            p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
            if few:
                e = 0.5 / (8355711.0 if f32 else 32639.0) * qd.abs().max(1)[0] * kd.abs().sum(1).max()
                bits, least = 2.0 ** (-21 if f32 else -11), 0.0
            else:
                e = 2.0 ** -11 * (qd.abs() @ kd.abs().T).max(1)[0] + 2.0 ** -23 * kd.abs().max() * qd.abs().sum(1)
                bits, least = 2.0 ** -11 + 2.0 ** -10, (2.0 ** -22 + kv * 2.0 ** -39) * float(vd.abs().max())
            e = abs(scale) * e + 5 * 2.0 ** -24 * 1.4427 * torch.where(seen, logit.abs(), 0.0).max(1)[0] + 2.0 ** -22
            o = p @ vd
            out[s0:s0 + n, h] = o
            bound[s0:s0 + n, h] = (torch.expm1(2 * e)[:, None] + bits + 2.0 ** -20) * (p @ vd.abs()) + least + (2.0 ** -23 if f32 else 2.0 ** -8) * o.abs()
    return out, bound


def put(dev, c):
    to = lambda t: torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=dev).copy_(t)  # noqa: E731
    cache = Q.KvCache(*(to(c[x]) for x in ("k", "v", "ks", "vs")))
    starts, lens = (torch.tensor(c[x], dtype=torch.int32, device=dev) for x in ("starts", "kv_len"))
    n = [b - a for a, b in zip(c["starts"], c["starts"][1:])]
    return dict(q=to(c["q"]), cache=cache, table=c["table"].to(dev), starts=starts, lens=lens, max_q=max(n), max_kv=max(c["kv_len"]))


def run(m, **kw):
    return Q.paged_attention(m["q"], m["cache"], m["table"], m["starts"], m["lens"], max_q=m["max_q"], max_kv=m["max_kv"], **kw)


def near(got, want, bound):
    err = (got.cpu().double() - want).abs()
    assert bool((err <= bound).all()), f"{float((err / bound.clamp(min=1e-300)).max()):.3g} times the bound"


def check(dev, c, **kw):
    kw.setdefault("scale", c["q"].shape[2] ** -0.5)
    m = put(dev, c)
    got = run(m, **kw)
    near(got, *oracle(c, **kw))
    again = run(m, **kw)
    assert torch.equal(got.view(torch.uint8), again.view(torch.uint8))


@pytest.mark.parametrize("lens,Hq,H,D,page,window", [
    ([(129, 129)], 1, 1, 64, 16, 0),
    ([(33, 500)], 4, 1, 128, 16, 0),             # 132 rows: a tile, and little of it
    ([(257, 300)], 2, 1, 80, 24, 0),
    ([(256, 1030)], 1, 1, 128, 64, 0),           # just past the length that is never split
    ([(200, 2500)], 4, 2, 128, 32, 0),           # split
    ([(200, 2500), (150, 900), (1, 2400)], 2, 1, 96, 16, 0),
    ([(140, 2049)], 2, 1, 256, 16, 0),
    ([(300, 1400)], 1, 1, 192, 7, 0),
    ([(180, 2300)], 2, 1, 64, 16, 700),          # a window over splits
    ([(300, 2000)], 1, 1, 128, 24, 1),
    ([(140, 50), (200, 100)], 1, 1, 128, 16, 0),  # rows before the first token
    ([(90, 1100), (1, 1100), (2, 7), (1, 0), (30, 600)], 5, 1, 112, 16, 0),
])
def test_many_rows(dev, lens, Hq, H, D, page, window):
    check(dev, R.make_case(lens, Hq=Hq, H=H, D=D, page=page, dtype=BF16, seed=Hq + D, token_major=page % 16 != 0), window=window)


@pytest.mark.parametrize("lens", [[(160, 1500)], [(130, 60), (1, 1300)]])
def test_many_rows_without_the_causal_mask(dev, lens):
    check(dev, R.make_case(lens, Hq=2, H=1, D=64, page=16, dtype=BF16, seed=1), causal=False)


def test_many_rows_holes(dev):
    """Pages without a block in the middle of tiles, and a sequence with none at all."""
    c = R.make_case([(150, 1400), (140, 200)], Hq=1, H=1, D=128, page=16, dtype=BF16, seed=2)
    c["table"][0, 3:9], c["table"][0, 40], c["table"][1, :] = -1, 1 << 20, -7
    check(dev, c)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lens,window", [
    ([(1, 1025)], 0),
    ([(1, 5000), (1, 4999), (1, 1), (1, 130)], 0),
    ([(3, 2200), (7, 1500), (1, 0)], 0),
    ([(20, 1800)], 0),
    ([(1, 7000), (1, 100)], 2500),
    ([(9, 3000), (2, 40)], 1111),
])
def test_few_rows_split(dev, lens, window, dtype):
    check(dev, R.make_case(lens, Hq=4, H=2, D=128, page=16, dtype=dtype, seed=3), window=window)
    check(dev, R.make_case(lens, Hq=3, H=1, D=80, page=24, dtype=dtype, seed=4), window=window)


@pytest.mark.parametrize("batch,longest", [(64, 300), (65, 1300), (131, 1200)])
def test_more_sequences_than_lanes(dev, batch, longest):
    """Lengths all over the range, empty sequences among them, chunks beside single tokens."""
    lens = [(1, 1 + (i * i * 37) % longest) for i in range(batch)]
    lens[batch // 2], lens[-2], lens[-1] = (1, 0), (1, longest), (5, longest - 1)
    check(dev, R.make_case(lens, Hq=2, H=1, D=64, page=16, dtype=BF16, seed=5))
    lens[3], lens[batch - 4] = (140, 400), (70, 150)
    check(dev, R.make_case(lens, Hq=2, H=1, D=64, page=16, dtype=BF16, seed=6))


@pytest.mark.parametrize("lens", [[(1, 2000), (1, 1500), (1, 40)], [(1, 300)], [(140, 1500), (1, 700)]])
def test_captured_graph_of_growing_sequences(dev, lens):
    """One capture serves lengths that change on the device, with other work between replays."""
    c = R.make_case(lens, Hq=2, H=1, D=64, page=16, dtype=BF16, seed=7)
    m, scale = put(dev, c), 0.125
    out = torch.empty_like(m["q"])
    ws = Q.paged_attention_workspace(c["starts"][-1], 2, 1, 64, len(lens), m["max_q"], m["max_kv"], dtype=BF16, device=dev)
    run(m, scale=scale, out=out, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(m, scale=scale, out=out, workspace=ws)
    for cut in (0, 1, 17, 150, 0):
        d = dict(c, kv_len=[max(kv - cut, 0) for kv in c["kv_len"]])
        m["lens"].copy_(torch.tensor(d["kv_len"], dtype=torch.int32))
        if ws is not None:
            ws.fill_(0xff)
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        near(out, *oracle(d, scale=scale))
        eager = run(m, scale=scale)
        assert torch.equal(eager.view(torch.uint8), out.view(torch.uint8))
