"""Attention over shared prefixes of at most 128 rows a group holds its weights with 16 bits:
columns of v whose two terms, one in the prefix and one of the own tokens or both in either,
all but cancel, so that the output's own rounding hides nothing.

Bound of a value, with w = sum p |v|: p as two bf16, 2^-16 of it; a logit's error e, half a step
of q's 32639 a product, five fp32 roundings and exp2's 2^-22, which moves a weight and their sum,
2 e w; fp32 sums, 2^-20 w, and the join of the parts, as much; the output's bf16, 2^-8 of it."""
import pytest
import torch

import phi_qlinear as Q

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,page", [(64, 16), (80, 24), (128, 16), (256, 7)])
@pytest.mark.parametrize("prefix,own", [(2, 1), (40, 7), (600, 90), (1300, 1500), (5000, 3)])
@pytest.mark.parametrize("G,rows", [(1, 1), (8, 5), (8, 16), (1, 127)])
def test_weights_of_sixteen_bits(dev, D, page, prefix, own, G, rows):
    g = torch.Generator().manual_seed(prefix + D)
    np, no = -(-prefix // page), -(-own // page)
    kv, blocks = prefix + own, np + no
    where = torch.cat([torch.arange(prefix), np * page + torch.arange(own)])  # a token's place in the cache
    k, v = (torch.zeros((blocks, 1, page, D), dtype=torch.int8) for _ in range(2))
    ks, vs = (torch.full((blocks, 1, page), 0.01) for _ in range(2))
    codes = torch.randint(-90, 91, (kv,), generator=g, dtype=torch.int8)
    q = torch.zeros((rows, G, D))
    q[..., 0] = 1.0 + torch.rand((rows, G), generator=g)
    q = q.to(torch.bfloat16)
    k.view(-1, D)[where, 0] = codes
    logit = q[..., :1].double() * codes.double() * 0.01  # scale 1
    p = torch.softmax(logit, dim=-1)
    vc = torch.zeros((kv, D), dtype=torch.int8)
    for d in range(D):  # two tokens a column, for one row and head: c a + c2 b all but 0
        a, b = (torch.randperm(kv, generator=g)[:2]).tolist()
        at = p[d % rows, d % G]
        a, b = (a, b) if at[a] <= at[b] else (b, a)
        c = 127 - d % 60
        vc[a, d], vc[b, d] = c, -round(float(c * at[a] / at[b]))
    v.view(-1, D)[where] = vc
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    # All rows' own tokens are the same ones; each is the last of them.
    own_table = (np + torch.arange(no, dtype=torch.int32, device=dev)).expand(rows, -1).contiguous()
    got = Q.paged_attention_shared(q.to(dev), Q.KvCache(k.to(dev), v.to(dev), ks.to(dev), vs.to(dev)),
                                   torch.arange(np, dtype=torch.int32, device=dev)[None], i32(prefix), i32(0, rows), own_table,
                                   i32(*range(rows + 1)), i32(*[own] * rows), max_prefix=prefix, max_q=1, max_kv=own, scale=1.0).cpu().double()
    vd = vc.double() * float(vs[0, 0, 0])
    want, weight = p @ vd, p @ vd.abs()
    e = 0.5 / 32639 * q.double().abs().amax() * 0.9 + 5 * 2.0 ** -24 * 1.4427 * logit.abs().max() + 2.0 ** -22
    bound = (2 * e + 2.0 ** -16 + 2 * 2.0 ** -20) * weight + 2.0 ** -8 * want.abs()
    assert bool(((got - want).abs() <= bound).all()), f"{float(((got - want).abs() / bound).max()):.3g} times the bound"
