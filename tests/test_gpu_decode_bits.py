"""Paged attention of few bf16 rows holds its weights with 16 bits: columns of v whose two
terms all but cancel, so that the output's own rounding hides nothing.

Bound of a value, with w = sum p |v|: p as two bf16, 2^-16 of it; a logit's error e, half
a step of q's 32639 a product, five fp32 roundings and exp2's 2^-22, which moves a
weight and their sum, 2 e w; fp32 sums, 2^-20 w; the output's bf16, 2^-8 of it."""
import pytest
import torch

import phi_qlinear as Q

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,page", [(64, 16), (80, 24), (128, 16), (256, 7)])
@pytest.mark.parametrize("kv", [2, 40, 600, 1300])
@pytest.mark.parametrize("G", [1, 8])
def test_weights_of_sixteen_bits(dev, D, page, kv, G):
    g = torch.Generator().manual_seed(kv + D)
    blocks = -(-kv // page)
    k, v = (torch.zeros((blocks, 1, page, D), dtype=torch.int8) for _ in range(2))
    ks, vs = (torch.full((blocks, 1, page), 0.01) for _ in range(2))
    codes = torch.randint(-90, 91, (kv,), generator=g, dtype=torch.int8)
    q = torch.zeros((1, G, D))
    q[0, :, 0] = 1.0 + torch.rand((G,), generator=g)
    q = q.to(torch.bfloat16)
    flat_k, flat_v = k.view(-1, D), v.view(-1, D)
    flat_k[:kv, 0] = codes
    logit = q[0, :, :1].double() * codes.double() * 0.01  # scale 1
    p = torch.softmax(logit, dim=1)
    for d in range(D):  # two tokens a column, for head d % G: c a + c2 b all but 0
        a, b = (torch.randperm(kv, generator=g)[:2]).tolist()
        a, b = (a, b) if p[d % G, a] <= p[d % G, b] else (b, a)
        c = 127 - d % 60
        flat_v[a, d], flat_v[b, d] = c, -round(float(c * p[d % G, a] / p[d % G, b]))
    got = Q.paged_attention(q.to(dev), Q.KvCache(k.to(dev), v.to(dev), ks.to(dev), vs.to(dev)),
                            torch.arange(blocks, dtype=torch.int32, device=dev)[None], torch.tensor([0, 1], dtype=torch.int32, device=dev),
                            torch.tensor([kv], dtype=torch.int32, device=dev), max_q=1, max_kv=kv, scale=1.0)[0].cpu().double()
    vd = flat_v[:kv].double() * float(vs[0, 0, 0])
    want, weight = p @ vd, p @ vd.abs()
    e = 0.5 / 32639 * q[0].double().abs().max() * 0.9 + 5 * 2.0 ** -24 * 1.4427 * logit.abs().max() + 2.0 ** -22
    bound = (2 * e + 2.0 ** -16 + 2.0 ** -20) * weight + 2.0 ** -8 * want.abs()
    assert bool(((got - want).abs() <= bound).all()), f"{float(((got - want).abs() / bound).max()):.3g} times the bound"
