"""GPU: the adapters' kernels at the sizes of long prompts: several column chunks a block, the last
of them ragged or empty, and so many blocks that they are spread over the chip's parts, a
number that is no whole one of these.  Bounds as in test_gpu_lora_batched.py."""
import pytest
import torch

import phi_qlinear as Q
import serving_ref as R
from test_gpu_lora_batched import inputs, near, same_bits

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32

SIZES = [  # rows, K, N, ranks, adapters, mixed
    (4300, 2100, 4790, 40, 4, False),
    (4300, 512, 5000, 72, 3, True),
    (4225, 2561, 4865, 33, 40, True),
    (16500, 96, 2300, 16, 5, False),
    (16385, 40, 2050, 5, 50, True),
]


@pytest.mark.parametrize("wd,od", [(BF16, BF16), (BF16, F32), (F32, F32), (F32, BF16)])
@pytest.mark.parametrize("M,K,N,rank,n,mixed", SIZES)
def test_long_prompts(dev, M, K, N, rank, n, mixed, wd, od):
    """Out of place, then in place in columns of a wider buffer at an odd element."""
    x, A, B, adapter, scale, base = inputs(M, K, N, rank, n, BF16, wd, od, seed=K, mixed=mixed)
    want, mag = R.adapted(x, A, B, adapter, scale, base)
    x, A, B, adapter, scale = (t.to(dev) for t in (x, A, B, adapter, scale))
    got = Q.lora_batched(x, A, B, adapter, scale=scale, base=base.to(dev))
    fine, by = near(got, want, mag, base, K, rank)
    assert fine, by
    for off in (1, 8):
        wide = torch.full((M, N + off + 7), 9.0, dtype=od, device=dev)
        part = wide[:, off:off + N]
        part.copy_(base)
        assert Q.lora_batched(x, A, B, adapter, scale=scale, base=part, out=part) is part and same_bits(part, got)
        assert bool((wide[:, :off] == 9).all()) and bool((wide[:, off + N:] == 9).all())
