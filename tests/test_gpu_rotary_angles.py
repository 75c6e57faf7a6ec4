"""GPU: the angles of rotary positions, position * freq modulo a turn, against exact rational
arithmetic.

Pairs (1, 0) turn into the cosine and the sine themselves.  The step, freq in turns, is held to
the nearest 2^-64 of a turn, so an angle is within |position| 2 pi 2^-64; beside that the cosine
and the sine are the fp32 nearest to their 64-bit values, half a step, 2^-24 of them, for which
2^-30 more are left to the series and the 64-bit sums."""
import math
from fractions import Fraction

import pytest
import torch

import phi_qlinear as Q

pytestmark = pytest.mark.gpu

BITS = 320


def turns_a_radian():
    """1 / 2 pi as a fraction, by Machin's formula."""
    def arctan_of_inverse(n):
        x = total = (1 << BITS) // n
        k, sign = 3, -1
        while x:
            x //= n * n
            total += sign * (x // k)
            k, sign = k + 2, -sign
        return total
    return Fraction(1 << BITS, 8 * (4 * arctan_of_inverse(5) - arctan_of_inverse(239)))


def exact(positions, freq):
    """cos and sin [positions, freq], fp64."""
    unit = turns_a_radian()
    steps = [Fraction(f) * unit % 1 for f in freq.tolist()]
    angle = [[2 * math.pi * float((p * s + Fraction(1, 2)) % 1 - Fraction(1, 2)) for s in steps] for p in positions.tolist()]
    angle = torch.tensor(angle, dtype=torch.float64)
    return angle.cos(), angle.sin()


def turned(dev, positions, freq, inter=False, scale=1.0):
    n = freq.numel()
    x = torch.zeros((positions.numel(), 1, 2 * n))
    x[..., 0::2] = 1.0
    if not inter:
        x = torch.cat([x[..., 0::2], x[..., 1::2]], dim=-1)
    y = Q.rotary(x.to(dev), positions.to(dev), freq.to(dev), interleaved=inter, scale=scale).cpu().double()[:, 0]
    return (y[:, 0::2], y[:, 1::2]) if inter else (y[:, :n], y[:, n:])


FREQS = [Q.rotary_frequencies(64, 10000.0, device="cpu"), Q.rotary_frequencies(48, 500000.0, scaling="linear", factor=32.0, device="cpu"),
         torch.tensor([100.0, 6.5, 2.0 ** 40 + 0.7, 1e-12, 2.0 ** -60, math.pi, -0.3, 0.0], dtype=torch.float64)]


@pytest.mark.parametrize("freq", FREQS)
@pytest.mark.parametrize("lg", [45, 47, 50])
def test_steps_are_held_to_the_nearest(dev, freq, lg):
    """At positions where a step's last bit is what the result turns on."""
    g = torch.Generator().manual_seed(lg)
    pos = torch.randint(1 << (lg - 1), 1 << lg, (40,), generator=g) * (1 - 2 * (torch.arange(40) % 2))
    away = pos.double().abs()[:, None] * 2 * math.pi * 2.0 ** -64
    for got, want in zip(turned(dev, pos, freq), exact(pos, freq)):
        err = (got - want).abs() - 2.0 ** -22
        assert bool((err <= away).all()), float((err / away).max())


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("freq", FREQS)
@pytest.mark.parametrize("lg,scale", [(4, 1.0), (20, 1.0), (24, 0.75)])
def test_cosines_and_sines_are_the_nearest(dev, freq, lg, scale, inter):
    """Scaled in 64 bits and rounded once."""
    g = torch.Generator().manual_seed(lg)
    pos = torch.randint(-(1 << lg), 1 << lg, (60,), generator=g)
    pos[0] = 0
    away = pos.double().abs()[:, None] * 2 * math.pi * 2.0 ** -64
    for got, want in zip(turned(dev, pos, freq, inter, scale), exact(pos, freq)):
        bound = 2.0 ** -24 * (scale * want).abs() + 2.0 ** -30 * abs(scale) + away
        err = (got - scale * want).abs()
        assert bool((err <= bound).all()), float((err / bound).max())
