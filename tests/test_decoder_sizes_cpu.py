"""Sizes at the ends of the decoder operators' integer ranges, on the CPU: what the C
entries answer before any device work."""
import ctypes

import pytest

import phi_qlinear as Q

A = ctypes.c_void_p(0x100000)  # well-aligned addresses; never dereferenced on these paths
B = ctypes.c_void_p(0x40000000)
C = ctypes.c_void_p(0x80000000)
S = ctypes.c_void_p(0x4000000000)


@pytest.mark.parametrize("kv_heads", [0, -1, 3, 5, 8, 65536, 1 << 31, 1 << 32, (1 << 32) + 2, (1 << 63) - 1])
def test_workspace_of_heads_that_no_call_takes(lib, kv_heads):
    """Key/value heads that do not divide the query heads: nothing to allocate, and no abort."""
    assert lib.phi_hip_paged_attention_workspace_bytes(8, 4, kv_heads, 64, 2, 4, 100000, Q.BF16) == 0


def test_workspace_of_heads_that_divide(lib):
    sizes = [lib.phi_hip_paged_attention_workspace_bytes(8, 4, h, 64, 2, 4, 100000, Q.BF16) for h in (1, 2, 4)]
    assert all(0 < n < 1 << 30 for n in sizes)
