"""GPU: what the adapters' second product makes of h's bits and of values that are not finite.

A has one element a rank, so that h is x's elements themselves (times 1), exactly; B has few
elements that are not 0, so that the result is known to its last bits."""
import math

import pytest
import torch

import phi_qlinear as Q

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
# rows, K, ranks: few rows and many, ranks within the registers' steps and past them.
SIZES = [(5, 64, 8), (40, 300, 40), (200, 512, 100), (1100, 512, 40), (1030, 520, 72), (1024, 1030, 256)]


def bits(t):
    return t.cpu().contiguous().view({2: torch.int16, 4: torch.int32}[t.element_size()])


def same_bits(a, b):
    return a.dtype == b.dtype and torch.equal(bits(a), bits(b))


def passing(M, K, R, n, dtype):
    """x of zeros and A [n, R, K] of which rank r passes x's element r on."""
    A = torch.zeros((n, R, K), dtype=dtype)
    A[:, torch.arange(R), torch.arange(R)] = 1.0
    return torch.zeros((M, K)), A


@pytest.mark.parametrize("wd,od", [(BF16, BF16), (BF16, F32), (F32, F32), (F32, BF16)])
@pytest.mark.parametrize("M,K,R", SIZES)
def test_infinite_factors(dev, M, K, R, wd, od):
    """h times an infinity is one of h's sign whatever bits h has, NaN where h is 0; the columns
    and adapters beside it keep their bits."""
    n, N = 3, 200
    g = torch.Generator().manual_seed(M)
    x, A = passing(M, K, R, n, wd)
    x[:, :R] = torch.randn((M, R), generator=g)  # of 24 bits, or 8, or none
    x[1::3, :R] = x[1::3, :R].bfloat16().float()
    x[2::7, R - 1] = 0.0
    B = torch.randn((n, N, R), generator=g).to(wd)
    adapter = (torch.arange(M) % (n + 1) - 1).int()
    to = lambda t: t.to(dev)  # noqa: E731
    plain = Q.lora_batched(to(x), to(A), to(B), to(adapter), out_dtype=od).cpu()
    B[1, 7, R - 1], B[1, 70, R - 1], B[1, 130, R // 2], B[1, 199, 0], B[1, 131, R - 1] = math.inf, -math.inf, math.inf, -math.inf, math.nan
    got = Q.lora_batched(to(x), to(A), to(B), to(adapter), out_dtype=od).cpu()
    mine, cols = adapter == 1, [7, 70, 130, 131, 199]
    want = plain.clone()
    for c, r, s in ((7, R - 1, math.inf), (70, R - 1, -math.inf), (130, R // 2, math.inf), (199, 0, -math.inf), (131, R - 1, math.nan)):
        want[mine, c] = (x[mine, r] * s).to(od)
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got[:, cols].nan_to_num(0.0, 9.0, -9.0), want[:, cols].nan_to_num(0.0, 9.0, -9.0))
    rest = torch.ones(N, dtype=torch.bool)
    rest[cols] = False
    assert same_bits(got[:, rest], plain[:, rest]) and same_bits(got[~mine], plain[~mine])


@pytest.mark.parametrize("wd", [BF16, F32])
@pytest.mark.parametrize("M,K,R", SIZES)
def test_h_past_the_largest_bf16(dev, M, K, R, wd):
    """fp32 values that bf16 would round to infinity: one product of 24 by 8 bits, exact before
    the sum of its three parts, each rounded to 24 bits."""
    x, A = passing(M, K, R, 1, wd)
    top = torch.finfo(F32).max
    x[:, 0] = top * (1 - torch.arange(M) * 2.0 ** -24 / M)
    x[1::2, 0] *= -1
    B = torch.zeros((1, 96, R), dtype=wd)
    B[0, :, 0] = torch.arange(1, 97) / 128
    got = Q.lora_batched(x.to(dev), A.to(dev), B.to(dev), torch.zeros(M, dtype=torch.int32, device=dev), out_dtype=F32).cpu().double()
    want = x[:, :1].double() * B[0, :, 0].double()
    assert bool(((got - want).abs() <= 3 * 2.0 ** -23 * want.abs()).all())


@pytest.mark.parametrize("od", [BF16, F32])
@pytest.mark.parametrize("wd", [BF16, F32])
@pytest.mark.parametrize("M,K,R", SIZES)
def test_rows_without_an_adapter_are_copied(dev, M, K, R, wd, od):
    """Zeros of either sign and infinities among them, inside whole columns and at the ragged end,
    into another tensor and in place."""
    n, N = 2, 333
    g = torch.Generator().manual_seed(M)
    x, A = passing(M, K, R, n, wd)
    base = torch.randn((M, N), generator=g).to(od)
    base[:, ::3], base[:, 1::5], base[:, 2::7] = -0.0, 0.0, -math.inf
    adapter = (torch.arange(M) % 4 - 1).int()  # -1 to 2
    none = (adapter < 0) | (adapter >= n)
    B = torch.randn((n, N, R), generator=g).to(wd)
    out = base.to(dev)
    to = [t.to(dev) for t in (x, A, B, adapter)]
    got = Q.lora_batched(*to, base=out)
    assert same_bits(got[none.to(dev)], base[none])
    assert same_bits(Q.lora_batched(*to, base=out, out=out)[none.to(dev)], base[none])
    zero = Q.lora_batched(*to, out_dtype=od)[none.to(dev)]
    assert same_bits(zero, torch.zeros_like(zero))


@pytest.mark.parametrize("wd", [BF16, F32])
@pytest.mark.parametrize("M,K,R", SIZES)
def test_h_has_all_of_its_bits(dev, M, K, R, wd):
    """One rank a column: h of 24 bits times 8, in up to three exact parts whose sum loses at
    most a step, 2^-23, of the largest at each of two additions (two terms instead of three lose
    2^-17, one 2^-9)."""
    n, N = 3, 150
    g = torch.Generator().manual_seed(K)
    x, A = passing(M, K, R, n, wd)
    x[:, :R] = torch.randn((M, R), generator=g)
    rank = torch.randint(0, R, (n, N), generator=g)
    B = torch.zeros((n, N, R), dtype=wd).scatter_(2, rank[..., None], (torch.randint(64, 128, (n, N, 1), generator=g) / 64).to(wd))
    adapter = torch.randint(0, n, (M,), generator=g).int()
    got = Q.lora_batched(*(t.to(dev) for t in (x, A, B, adapter)), out_dtype=F32).cpu().double()
    for a in range(n):
        mine = adapter == a
        want = x[mine].double()[:, rank[a]] * B[a].double().gather(1, rank[a][:, None])[:, 0]
        assert bool(((got[mine] - want).abs() <= 2 * 2.0 ** -23 * want.abs()).all())
