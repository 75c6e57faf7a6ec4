"""CPU checks of the decoder layer's operators: what the C entries refuse, before
any device work, and the plain forms that the GPU tests compare with."""
import ctypes
import math

import pytest
import torch

import decoder_ref as R
import phi_qlinear as Q

A = ctypes.c_void_p(0x100000)  # well-aligned addresses; never dereferenced on these paths
B = ctypes.c_void_p(0x40000000)
C = ctypes.c_void_p(0x80000000)
S = ctypes.c_void_p(0xC0000000)
ODD = ctypes.c_void_p(0x100001)


def norm(lib, x=A, xd=Q.F32, ldx=512, res=None, out=None, rd=Q.F32, ldr=512, w=None, sh=None, wd=Q.F32, eps=1e-6,
         rows=4, K=512, y=None, yd=Q.F32, ldy=512, q=B, ldq=512, s=C, qmax=127.0, mode=0, rotate=1):
    rc = lib.phi_hip_rms_norm_quant(None, x, xd, ldx, res, out, rd, ldr, w, sh, wd, eps, rows, K, y, yd, ldy, q, ldq, s,
                                    qmax, mode, rotate)
    return rc, Q.last_error()


@pytest.mark.parametrize("rc,text,kw", [
    (2, "multiple of 256", dict(K=500)),
    (2, "negative", dict(rows=-1)),
    (2, "empty", dict(K=0)),
    (7, "exceeds", dict(K=32769, rotate=0, ldx=40000, ldq=40000)),
    (1, "null", dict(x=None)),
    (1, "null", dict(q=None)),
    (1, "null", dict(s=None)),
    (1, "without residual", dict(out=S)),
    (1, "dtypes", dict(xd=Q.I8)),
    (1, "dtypes", dict(res=S, rd=Q.F16)),
    (1, "dtypes", dict(w=S, wd=Q.I32)),
    (1, "dtypes", dict(y=S, yd=Q.F16)),
    (1, "round", dict(mode=2)),
    (1, "qmax", dict(qmax=128.0)),
    (1, "qmax", dict(qmax=6.5)),
    (1, "qmax", dict(qmax=math.nan)),
    (1, "eps", dict(eps=-1e-6)),
    (1, "eps", dict(eps=math.inf)),
    (2, "leading", dict(ldx=511)),
    (2, "leading", dict(ldq=511)),
    (2, "leading", dict(res=S, ldr=100)),
    (2, "leading", dict(y=S, ldy=511)),
    (2, "too large", dict(ldx=1 << 40)),
    (3, "aligned", dict(x=ODD)),
    (3, "aligned", dict(y=ODD)),
    (1, "output overlaps an input", dict(q=ctypes.c_void_p(0x100000 + 64))),
    (1, "output overlaps an input", dict(res=S, out=ctypes.c_void_p(0xC0000000 + 2048))),
    (1, "two outputs", dict(y=ctypes.c_void_p(0x40000000 + 64))),
])
def test_norm_refuses(lib, rc, text, kw):
    got, msg = norm(lib, **kw)
    assert got == rc and text in msg and "rms_norm_quant" in msg


def test_norm_of_no_rows(lib):
    assert norm(lib, x=None, q=None, s=None, rows=0) == (0, "")


def cache(**kw):
    d = dict(k=0x100000, v=0x40000000, k_scale=0x80000000, v_scale=0xC0000000, blocks=10, heads=2, page=16, dim=64,
             block_stride=2 * 16 * 64, head_stride=16 * 64, token_stride=64, s_block_stride=32, s_head_stride=16,
             s_token_stride=1)
    d.update(kw)
    return Q.KvCacheDesc(**d)


BAD_CACHES = [
    (1, "null cache", dict(k=None)),
    (1, "null cache", dict(v_scale=None)),
    (2, "empty cache", dict(blocks=0)),
    (2, "empty cache", dict(page=-1)),
    (2, "dim=72", dict(dim=72)),
    (2, "dim=272", dict(dim=272)),
    (2, "dim=0", dict(dim=0)),
    (2, "too large", dict(page=(1 << 20) + 1)),
    (2, "too large", dict(heads=70000)),
    (2, "stride", dict(head_stride=-64)),
    (2, "stride", dict(s_token_stride=1 << 50)),
    (3, "16-byte", dict(k=0x100008)),
    (3, "16-byte", dict(token_stride=72)),
    (3, "misaligned", dict(k_scale=0x80000002)),
]


def write(lib, c, k=A, kt=128, kh=64, v=B, vt=128, vh=64, dtype=Q.BF16, slots=C, tokens=3):
    return lib.phi_hip_kv_cache_write(None, ctypes.byref(c) if c else None, k, kt, kh, v, vt, vh, dtype, slots, tokens)


def read(lib, c, k=A, kt=128, kh=64, v=B, vt=128, vh=64, dtype=Q.BF16, slots=C, tokens=3):
    return lib.phi_hip_kv_cache_read(None, ctypes.byref(c) if c else None, slots, tokens, k, kt, kh, v, vt, vh, dtype)


def attend(lib, c, q=A, dtype=Q.BF16, qt=256, qh=64, tokens=8, heads=4, table=B, width=4, stride=4, start=C, lens=C,
           batch=2, max_q=4, max_kv=64, scale=0.1, causal=1, window=0, out=S, ot=256, oh=64, ws=None, wn=0):
    return lib.phi_hip_paged_attention(None, q, dtype, qt, qh, tokens, heads, ctypes.byref(c) if c else None, table, width,
                                       stride, start, lens, batch, max_q, max_kv, scale, causal, window, out, ot, oh, ws, wn)


@pytest.mark.parametrize("rc,text,kw", BAD_CACHES)
def test_bad_caches_are_refused(lib, rc, text, kw):
    for call in (write, read, attend):
        assert call(lib, cache(**kw)) == rc and text in Q.last_error()
    assert write(lib, None) == 1


@pytest.mark.parametrize("rc,text,kw", [
    (2, "negative", dict(tokens=-1)),
    (1, "f32 or bf16", dict(dtype=Q.I8)),
    (1, "null k", dict(k=None)),
    (1, "null v", dict(v=None)),
    (1, "null slots", dict(slots=None)),
    (3, "aligned", dict(k=ctypes.c_void_p(0x100008))),
    (3, "aligned", dict(kt=129)),
    (3, "aligned", dict(vh=66)),
    (3, "slots", dict(slots=ctypes.c_void_p(0x100004))),
    (2, "stride", dict(vt=-128)),
])
def test_write_and_read_refuse(lib, rc, text, kw):
    for call in (write, read):
        assert call(lib, cache(), **kw) == rc and text in Q.last_error()


def test_no_tokens_is_no_work(lib):
    for call in (write, read):
        assert call(lib, cache(), tokens=0, k=None, v=None, slots=None) == 0 and Q.last_error() == ""
    for kw in (dict(tokens=0), dict(batch=0), dict(max_q=0)):
        assert attend(lib, cache(), q=None, out=None, **kw) == 0 and Q.last_error() == ""


@pytest.mark.parametrize("rc,text,kw", [
    (2, "negative", dict(tokens=-1)),
    (2, "negative", dict(max_kv=-1)),
    (1, "f32 or bf16", dict(dtype=Q.F16)),
    (2, "5 query heads for 2", dict(heads=5)),
    (2, "query heads", dict(heads=0)),
    (2, "out of range", dict(max_q=9)),
    (2, "out of range", dict(batch=70000)),
    (2, "block table", dict(max_kv=65)),
    (2, "block table", dict(stride=3)),
    (1, "window", dict(window=-1)),
    (1, "window", dict(window=8, causal=0)),
    (1, "scale", dict(scale=math.inf)),
    (1, "scale", dict(scale=math.nan)),
    (1, "null q", dict(q=None)),
    (1, "null out", dict(out=None)),
    (1, "null pointer", dict(table=None)),
    (1, "null pointer", dict(start=None)),
    (1, "null pointer", dict(lens=None)),
    (3, "aligned", dict(qt=257)),
    (3, "aligned", dict(oh=60)),
    (3, "misaligned", dict(lens=ODD)),
    (1, "overlaps", dict(out=ctypes.c_void_p(0x100000 + 1024))),
])
def test_attention_refuses(lib, rc, text, kw):
    assert attend(lib, cache(), **kw) == rc and text in Q.last_error()


def test_attention_workspace(lib):
    """Where a call needs a workspace, one that is missing, small or misaligned is refused."""
    n = lib.phi_hip_paged_attention_workspace_bytes(1, 4, 2, 64, 1, 1, 100000, Q.BF16)
    kw = dict(tokens=1, batch=1, max_q=1, max_kv=100000, width=6250, stride=6250)
    if n:
        assert attend(lib, cache(), **kw) == 4 and str(n) in Q.last_error()
        assert attend(lib, cache(), ws=ctypes.c_void_p(0x200000000), wn=n - 1, **kw) == 4
        assert attend(lib, cache(), ws=ctypes.c_void_p(0x200000008), wn=n, **kw) == 3
        assert attend(lib, cache(), ws=A, wn=n, **kw) == 1 and "overlaps" in Q.last_error()
    for bad in ((0, 4, 2, 64, 1, 1, 100), (1, 4, 2, 64, 1, 2, 100), (1, 4, 2, 64, 1, 1, 0)):
        assert lib.phi_hip_paged_attention_workspace_bytes(*bad, Q.BF16) == 0


def test_python_refusals():
    t = torch.zeros((2, 256))
    with pytest.raises(ValueError):
        Q.rms_norm_quant(t, None, 1e-6)  # not on the device


def test_the_rotation_is_its_own_inverse():
    h = R.hadamard()
    assert torch.allclose(h @ h, torch.eye(256, dtype=torch.float64), atol=1e-15) and torch.equal(h, h.t())


def test_plain_attention_agrees_with_a_dense_form():
    c = R.make_case([(3, 20), (1, 0), (2, 9)], Hq=4, H=2, D=16, page=8, dtype=torch.float32, seed=1)
    out, bound = R.attention(c["q"], c["k"], c["v"], c["ks"], c["vs"], c["table"], c["starts"], c["kv_len"], scale=0.25)
    ids = c["table"][0, :3].long()
    k = (c["k"][ids].double() * c["ks"][ids].double()[..., None]).permute(1, 0, 2, 3).reshape(2, 24, 16)[:, :20]
    v = (c["v"][ids].double() * c["vs"][ids].double()[..., None]).permute(1, 0, 2, 3).reshape(2, 24, 16)[:, :20]
    for i in range(3):
        n = 18 + i
        for h in range(4):
            p = torch.softmax(k[h // 2, :n] @ c["q"][i, h].double() * 0.25, dim=0)
            assert torch.allclose(out[i, h], p @ v[h // 2, :n], atol=1e-13)
    assert not bool(out[3].any()) and bool((bound[:3] > 0).all())
