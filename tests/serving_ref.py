"""Plain 64-bit forms of the serving operators, on the CPU."""
import torch


def rotated(x, positions, freq, interleaved, scale):
    """x [tokens, heads, dim] turned, in 64 bits, and beside each value the sum of
    its terms' magnitudes (of what was only copied: 0)."""
    half = freq.numel()
    x = x.double()
    angle = positions.double()[:, None] * freq
    cos, sin = torch.cos(angle)[:, None] * scale, torch.sin(angle)[:, None] * scale
    j = torch.arange(half)
    i, k = (2 * j, 2 * j + 1) if interleaved else (j, j + half)
    a, b = x[..., i], x[..., k]
    y, mag = x.clone(), torch.zeros_like(x)
    y[..., i], y[..., k] = a * cos - b * sin, b * cos + a * sin
    mag[..., i] = mag[..., k] = abs(scale) * (a.abs() + b.abs())
    return y, mag


def adapted(x, A, B, adapter, scale, base):
    """base + scale B (A x) of each row's adapter in 64 bits and, beside each value,
    the sum of its terms' magnitudes through both products (0: none)."""
    n, R, K = A.shape
    M, N = x.shape[0], B.shape[1]
    y = torch.zeros((M, N), dtype=torch.float64) if base is None else base.double()
    mag = torch.zeros((M, N), dtype=torch.float64)
    for a in range(n):
        mine = adapter == a
        s = 1.0 if scale is None else scale[a].double()
        xa, Aa, Ba = x[mine].double(), A[a].double(), B[a].double()
        y[mine] += (xa @ Aa.t()) @ Ba.t() * s
        mag[mine] = (xa.abs() @ Aa.abs().t()) @ Ba.abs().t() * abs(s)
    return y, mag
