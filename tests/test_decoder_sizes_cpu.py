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


def attend(lib, *, tokens, heads, kv_heads, max_q, qt=0, batch=1):
    cache = Q.KvCacheDesc(k=0x100000, v=0x40000000, k_scale=0x80000000, v_scale=0xC0000000, blocks=10, heads=kv_heads, page=16,
                          dim=16, block_stride=16 * 16 * kv_heads, head_stride=256, token_stride=16, s_block_stride=16 * kv_heads,
                          s_head_stride=16, s_token_stride=1)
    rc = lib.phi_hip_paged_attention(None, A, Q.BF16, qt, 16, tokens, heads, ctypes.byref(cache), B, 4, 4, C, C, batch, max_q, 64,
                                     0.25, 1, 0, S, qt, 16, None, 0)
    return rc, Q.last_error()


@pytest.mark.parametrize("tokens,heads,kv_heads", [((1 << 31) - 1, 2, 1), (1 << 30, 4, 2), ((1 << 24) + 1, 64, 1), (1 << 20, 65535, 1),
                                                   ((1 << 30) + 1, 8, 8)])
def test_rows_past_31_bits_are_refused(lib, tokens, heads, kv_heads):
    """A sequence's rows, new tokens x query heads a key/value head, are counted in 32 bits."""
    rc, text = attend(lib, tokens=tokens, heads=heads, kv_heads=kv_heads, max_q=tokens)
    assert rc == 2 and "out of range" in text
