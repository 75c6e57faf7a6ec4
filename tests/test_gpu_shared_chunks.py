"""GPU: chunks of new tokens over long contexts of their own, behind short prefixes or none
(phi_hip_paged_attention_shared): what a prompt in chunks behind cached tokens is.  Against a
plain softmax in 64 bits, with the bounds of serving_ref.shared_attention."""
import pytest
import torch

import phi_qlinear as Q
import serving_ref as R
from test_gpu_shared_prefix import arguments, check, same_bits

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.mark.parametrize("groups,free,Hq,H,D,page", [
    ([(64, [(64, 4096)])], [], 16, 2, 64, 16),
    ([(0, [(300, 2500)])], [], 4, 2, 128, 64),
    ([(33, [(40, 3000), (1, 2000), (70, 700)]), (500, [(150, 1500)])], [(130, 1000), (1, 0)], 8, 2, 80, 16),
    ([(16, [(200, 200)]), (0, [(1, 1)] * 20)], [], 2, 1, 64, 16),
    ([(100, [(20, 2000), (30, 900)])], [], 16, 2, 192, 32),
])
def test_chunks_over_their_own_tokens(dev, groups, free, Hq, H, D, page):
    c = R.shared_case(groups, free, Hq=Hq, H=H, D=D, page=page, dtype=BF16, seed=D)
    got = check(dev, c)
    assert same_bits(got, Q.paged_attention_shared(**arguments(dev, c)))

