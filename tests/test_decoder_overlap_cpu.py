"""Which tensors' memory the decoder operators' C entries take as shared, on the CPU.
Where nothing is shared a call passes these checks and ends at the launch, for want
of a device."""
import ctypes
import itertools

import pytest
import torch

import phi_qlinear as Q

BASE = 0x7000000000  # of made-up buffers; never dereferenced


def at(byte, buffer=0):
    return ctypes.c_void_p(BASE + (buffer << 32) + byte)


def norm(lib, *, x, ldx, q, ldq, rows=6, K=64, res=None, out=None, ldr=64, y=None, ldy=64, s=at(0, 9)):
    rc = lib.phi_hip_rms_norm_quant(None, x, Q.BF16, ldx, res, out, Q.BF16, ldr, None, None, Q.F32, 1e-6, rows, K, y, Q.BF16, ldy,
                                    q, ldq, s, 127.0, 0, 0)
    return rc, Q.last_error()


def overlaps(rc_text):
    rc, text = rc_text
    assert ("overlap" in text) == (rc == 1), text
    return rc == 1


no_device = pytest.mark.skipif(torch.cuda.is_available(), reason="addresses are made up")


@no_device
@pytest.mark.parametrize("x,res,y,shared", [(0, 64, 128, False), (128, 0, 64, False), (0, 63, 128, True), (0, 64, 127, True),
                                            (0, 128, 64, False), (129, 0, 64, True), (64, 64, 0, False)])
def test_norm_on_columns_of_one_buffer(lib, x, res, y, shared):
    """x, residual (updated in place) and y are 64 columns each of a buffer of 192."""
    r = at(2 * res)
    got = overlaps(norm(lib, x=at(2 * x), ldx=192, res=r, out=None if x == res else r, ldr=192, y=at(2 * y), ldy=192, q=at(0, 1), ldq=64))
    assert got == shared


@no_device
def test_norm_on_columns_of_different_types(lib):
    """Codes in the last 64 bytes of rows whose first 128 are x; a byte earlier they meet."""
    for first, shared in ((128, False), (127, True), (129, True)):
        assert overlaps(norm(lib, x=at(0), ldx=96, q=at(first), ldq=192)) == shared


def brute(a, b):
    """Whether two sets of pieces (start, bytes, n1, s1, n2, s2) share a byte."""
    covered = [{start + i * s1 + j * s2 + k for i in range(n1) for j in range(n2) for k in range(w)} for start, w, n1, s1, n2, s2 in (a, b)]
    return bool(covered[0] & covered[1])


@no_device
def test_attention_beside_its_queries(lib):
    """out and q as parts of one buffer, against the bytes themselves: nothing shared is
    never missed, and the usual layouts that share nothing are taken."""
    T, H, D = 3, 2, 16
    cache = Q.KvCacheDesc(k=0x100000, v=0x200000, k_scale=0x300000, v_scale=0x400000, blocks=10, heads=2, page=16, dim=D, block_stride=512,
                          head_stride=256, token_stride=16, s_block_stride=32, s_head_stride=16, s_token_stride=1)

    def call(q, qt, qh, o, ot, oh):
        rc = lib.phi_hip_paged_attention(None, at(2 * q), Q.BF16, qt, qh, T, H, ctypes.byref(cache), at(0, 1), 4, 4, at(0, 2), at(0, 3), 1, T,
                                         64, 0.25, 1, 0, at(2 * o), ot, oh, None, 0)
        return overlaps((rc, Q.last_error()))

    for q, o, (qt, qh), (ot, oh) in itertools.product((0, 64), range(0, 200, 8), ((32, 16), (64, 16), (64, 32), (16, 48), (96, 32)),
                                                      ((32, 16), (64, 16), (64, 32), (16, 48), (96, 32))):
        shared = brute((q, D, T, qt, H, qh), (o, D, T, ot, H, oh))
        assert call(q, qt, qh, o, ot, oh) or not shared
    assert not call(0, 64, 16, 32, 64, 16)  # [T, q | out, H, D]
    assert not call(0, 64, 32, 16, 64, 32)  # [T, H, q | out, D]
    assert not call(0, 32, 16, 96, 32, 16)  # one after the other
    assert not call(0, 16, 96, 48, 16, 96)  # [H, q | out, T, D]
    assert call(0, 64, 16, 24, 64, 16) and call(0, 64, 32, 0, 64, 32)


def read_into(lib, k, v, kt=32, vt=32, kh=16, vh=16, cache=None):
    """kv_cache_read of 2 heads of 16 into bf16 k and v at these element offsets of a
    buffer; the cache's arrays are 4 MiB apart in another."""
    d = dict(k=BASE + (5 << 32), v=BASE + (5 << 32) + (4 << 20), k_scale=BASE + (5 << 32) + (8 << 20), v_scale=BASE + (5 << 32) + (12 << 20),
             blocks=10, heads=2, page=16, dim=16, block_stride=512, head_stride=256, token_stride=16, s_block_stride=32, s_head_stride=16,
             s_token_stride=1)
    d.update(cache or {})
    to = lambda x: x if isinstance(x, ctypes.c_void_p) else at(2 * x)  # noqa: E731
    rc = lib.phi_hip_kv_cache_read(None, ctypes.byref(Q.KvCacheDesc(**d)), at(0, 1), 3, to(k), kt, kh, to(v), vt, vh, Q.BF16)
    return overlaps((rc, Q.last_error()))


@no_device
def test_read_into_overlapping_outputs(lib):
    for k, v in itertools.product((0, 32), range(0, 200, 8)):
        for (kt, kh), (vt, vh) in itertools.product(((32, 16), (64, 16), (16, 48)), repeat=2):
            shared = brute((k, 16, 3, kt, 2, kh), (v, 16, 3, vt, 2, vh))
            assert read_into(lib, k, v, kt, vt, kh, vh) or not shared
    assert read_into(lib, 0, 0) and read_into(lib, 0, 16)
    assert not read_into(lib, 0, 96)  # one after the other
    assert not read_into(lib, 0, 32, kt=64, vt=64)  # columns of one tensor
    assert not read_into(lib, 0, 16, kt=64, vt=64, kh=32, vh=32)


@no_device
@pytest.mark.parametrize("array,size", [("k", 5120), ("v", 5120), ("k_scale", 1280), ("v_scale", 1280)])
@pytest.mark.parametrize("which", ["k", "v"])
def test_read_into_the_cache(lib, array, size, which):
    """An output that reaches into one of the cache's arrays, at either end of it; 192 bytes."""
    start = 6 << 32
    for byte, shared in ((0, True), (-192, False), (-176, True), (size, False), (size - 16, True)):
        to = {"k": 0, "v": 1024, which: ctypes.c_void_p(BASE + start + byte)}
        assert read_into(lib, to["k"], to["v"], cache={array: BASE + start}) == shared


@no_device
@pytest.mark.parametrize("tokens,ot,oh,refused", [(3, 0, 16, True), (3, 32, 0, True), (3, 8, 48, True), (1, 0, 16, False), (3, 32, 16, False),
                                                  (3, 16, 48, False)])
def test_outputs_whose_vectors_overlap(lib, tokens, ot, oh, refused):
    """Vectors of 16 at smaller strides are written over one another: refused, where there is more than one."""
    def answer(rc):
        assert ("'s vectors overlap" in Q.last_error()) == (rc == 2), Q.last_error()
        return rc == 2

    cache = Q.KvCacheDesc(k=0x100000, v=0x200000, k_scale=0x300000, v_scale=0x400000, blocks=10, heads=2, page=16, dim=16, block_stride=512,
                          head_stride=256, token_stride=16, s_block_stride=32, s_head_stride=16, s_token_stride=1)
    assert answer(lib.phi_hip_paged_attention(None, at(0, 4), Q.BF16, 0, 16, tokens, 2, ctypes.byref(cache), at(0, 1), 4, 4, at(0, 2), at(0, 3), 1,
                                              tokens, 64, 0.25, 1, 0, at(0), ot, oh, None, 0)) == refused
    for k, v in (((ot, oh), (32, 16)), ((32, 16), (ot, oh))):
        assert answer(lib.phi_hip_kv_cache_read(None, ctypes.byref(cache), at(0, 1), tokens, at(0), *k, at(0, 4), *v, Q.BF16)) == refused
    # Inputs may: one vector for all tokens or heads.
    assert not answer(lib.phi_hip_kv_cache_write(None, ctypes.byref(cache), at(0), ot, oh, at(0, 4), ot, oh, Q.BF16, at(0, 1), tokens))


@no_device
@pytest.mark.parametrize("stride,value,refused", [("block_stride", 0, True), ("head_stride", 0, True), ("token_stride", 0, True),
                                                  ("s_block_stride", 0, True), ("s_head_stride", 0, True), ("s_token_stride", 0, True),
                                                  ("token_stride", 16, False)])
def test_writing_to_a_cache_whose_vectors_overlap(lib, stride, value, refused):
    """A cache that holds one vector for several places can be read, not written."""
    d = dict(k=0x100000, v=0x200000, k_scale=0x300000, v_scale=0x400000, blocks=10, heads=2, page=16, dim=16, block_stride=512,
             head_stride=256, token_stride=16, s_block_stride=32, s_head_stride=16, s_token_stride=1)
    one = dict(block_stride="blocks", head_stride="heads", token_stride="page", s_block_stride="blocks", s_head_stride="heads", s_token_stride="page")
    d[stride] = value
    for n, want in ((d[one[stride]], refused), (1, False)):
        cache = Q.KvCacheDesc(**{**d, one[stride]: n})
        rc = lib.phi_hip_kv_cache_write(None, ctypes.byref(cache), at(0), 32, 16, at(0, 4), 32, 16, Q.BF16, at(0, 1), 3)
        assert (rc == 2 and "cache's vectors overlap" in Q.last_error()) == want
        assert lib.phi_hip_kv_cache_read(None, ctypes.byref(cache), at(0, 1), 3, at(0), 32, 16, at(0, 4), 32, 16, Q.BF16) != 2
