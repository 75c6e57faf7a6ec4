"""CPU checks of the serving operators at the ends of what they take: records that hold
anything, the largest launches, copies that fail."""
import ctypes
import os
import subprocess

import pytest
import torch

import phi_qlinear as Q

A, B, C, D, E, F, G = (ctypes.c_void_p(x << 40) for x in range(1, 8))  # well aligned and far apart, never dereferenced


def attend(lib, *, tokens=8, heads=4, kv_heads=1, groups=1, batch=1, dim=16, dtype=Q.BF16, max_prefix=64, max_q=1, max_kv=64, ws=1 << 40):
    """paged_attention_shared over a cache and tables that no call reads here."""
    cache = Q.KvCacheDesc(k=8 << 40, v=9 << 40, k_scale=10 << 40, v_scale=11 << 40, blocks=10, heads=kv_heads, page=16, dim=dim,
                          block_stride=16 * dim * kv_heads, head_stride=16 * dim, token_stride=dim, s_block_stride=16 * kv_heads,
                          s_head_stride=16, s_token_stride=1)
    w = 1 << 20
    rc = lib.phi_hip_paged_attention_shared(None, A, dtype, heads * dim, dim, tokens, heads, ctypes.byref(cache), B, w, w, C, C, groups, max_prefix,
                                            B, w, w, D, D, batch, max_q, max_kv, 0.25, E, heads * dim, dim, F, ws)
    return rc, Q.last_error()



def test_records_of_rows_stay_in_their_slots():
    """What attention over shared prefixes reads back of rows that nothing was left for."""
    cdir = os.path.join(os.path.dirname(__file__), "cpp")
    subprocess.run(["make", "-C", cdir, "attn_row"], check=True, capture_output=True)
    out = subprocess.run([os.path.join(cdir, "attn_row")], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0 and "wrong 0" in out.stdout, out.stdout


@pytest.mark.parametrize("tokens,heads", [((1 << 26) - 1, 1), ((1 << 26) - 3, 1), (((1 << 26) - 2) // 2, 2)])
def test_more_rows_than_the_join_has_waves_are_refused(lib, tokens, heads):
    """Four rows a block of 256 threads, and a launch's threads are counted in 32 bits."""
    rc, text = attend(lib, tokens=tokens, heads=heads)
    assert rc == 2 and "out of range" in text
    size = lib.phi_hip_paged_attention_shared_workspace_bytes
    assert size(tokens, heads, 1, 16, 1, 1, 64, 1, 64, Q.BF16) == 0
    assert size((1 << 26) // heads - 4, heads, 1, 16, 1, 1, 64, 1, 64, Q.BF16) > 0


@pytest.mark.parametrize("dtype,dim,kv_heads", [(Q.BF16, 64, 256), (Q.BF16, 256, 512), (Q.F32, 64, 512)])
def test_more_sequences_than_a_launch_has_blocks_for_are_refused(lib, dtype, dim, kv_heads):
    sizes = dict(tokens=65535, heads=kv_heads, kv_heads=kv_heads, groups=65535, batch=65535, dim=dim, dtype=dtype)
    rc, text = attend(lib, **sizes)
    assert rc == 2 and "groups" in text and "too many" in text
    size = lib.phi_hip_paged_attention_shared_workspace_bytes
    assert size(65535, kv_heads, kv_heads, dim, 65535, 65535, 64, 1, 64, dtype) == 0
    assert size(65535, 16, 16, dim, 65535, 65535, 64, 1, 64, dtype) > 0


@pytest.mark.parametrize("a,b", [((1 << 39), 64), (64, (1 << 39)), (1 << 36, 1 << 36)])
def test_factors_that_span_more_than_any_memory_are_refused(lib, a, b):
    """The end of the last adapter's, in bytes, is counted in 63 bits."""
    rc = lib.phi_hip_lora_batched(None, A, Q.BF16, 16, 4, 16, B, a, 16, C, b, 4, Q.BF16, (1 << 31) - 1, 4, 16, D, None, None, 0, E, Q.BF16,
                                  16, F, 1 << 30)
    assert rc == 2 and "adapter stride" in Q.last_error()


def test_copies_that_fail_are_kept(monkeypatch):
    """What a flush could not do is left for the next one, what it did is not."""
    calls, fails = [], [False, True]

    def copy(a, b, frm, to, tokens):
        if fails and fails.pop(0):
            raise ValueError("tensors of another device")
        calls.append(list(zip(frm.tolist(), to.tolist(), tokens.tolist())))

    monkeypatch.setattr(Q.serving, "kv_cache_copy", copy)

    class Host:
        k = torch.zeros(1)

    pages = Q.KvPages(8, 4)
    pages.copies = [(0, 1, 4), (2, 3, 2), (3, 4, 2), (1, 5, 4), (5, 6, 1)]  # in three calls
    with pytest.raises(ValueError):
        pages.flush(Host)
    assert calls == [[(0, 1, 4), (2, 3, 2)]] and pages.copies == [(3, 4, 2), (1, 5, 4), (5, 6, 1)]
    pages.flush(Host)
    assert calls[1:] == [[(3, 4, 2), (1, 5, 4)], [(5, 6, 1)]] and pages.copies == []
    pages.flush(Host)
    assert len(calls) == 3


@pytest.mark.parametrize("tokens,heads,batch,max_prefix", [(64, 64, 1, 64), (64, 64, 1, 0), (1024, 32, 1, 0), (130, 64, 3, 16)])
def test_long_own_contexts_of_chunks_are_split(lib, tokens, heads, batch, max_prefix):
    """Sequences of more than 128 rows, whose own tokens the chunk kernel takes: as much of a
    short prefix' call as of a long one's work is shared out (256 / 8 units a head, a split
    of 3 tiles of 64 tokens or more)."""
    slot = 8 * 256 * (128 + 2) * 4  # of all key/value heads
    size = lambda kv: lib.phi_hip_paged_attention_shared_workspace_bytes(  # noqa: E731
        tokens, heads, 8, 128, 1, batch, max_prefix, 64 if tokens < 1024 else tokens, kv, Q.BF16)
    assert (size(8192) - size(64)) // slot >= 24
