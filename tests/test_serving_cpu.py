"""CPU checks of the serving operators: what the C entries refuse, before any
device work, frequencies, and the book-keeping of pages."""
import ctypes
import math
import random

import pytest
import torch

import phi_qlinear as Q
import serving_ref as R
from test_decoder_cpu import BAD_CACHES, cache

A, B, C, D, E, F, G = (ctypes.c_void_p(x << 28) for x in range(1, 8))  # well aligned, never dereferenced
K2, V2, KS2, VS2 = 0x900000000, 0x940000000, 0x980000000, 0x9C0000000
ODD = ctypes.c_void_p((1 << 28) + 1)
OFF8 = ctypes.c_void_p((1 << 28) + 8)
no_device = pytest.mark.skipif(torch.cuda.is_available(), reason="addresses are made up")


def far(**kw):
    """A cache away from the other addresses."""
    return cache(**{**dict(k=K2, v=V2, k_scale=KS2, v_scale=VS2), **kw})


def turn(lib, x=A, dtype=Q.BF16, xt=256, xh=64, tokens=5, heads=4, dim=64, pos=C, freq=D, rot=64, inter=0, scale=1.0,
         out=B, ot=256, oh=64):
    rc = lib.phi_hip_rotary(None, x, dtype, xt, xh, tokens, heads, dim, pos, freq, rot, inter, scale, out, ot, oh)
    return rc, Q.last_error()


@pytest.mark.parametrize("rc,text,kw", [
    (2, "negative", dict(tokens=-1)),
    (2, "negative", dict(heads=-1)),
    (2, "dim=0", dict(dim=0)),
    (2, "dim=1025", dict(dim=1025)),
    (2, "out of range", dict(tokens=1 << 31)),
    (2, "out of range", dict(heads=70000)),
    (1, "f32 or bf16", dict(dtype=Q.F16)),
    (2, "rotated", dict(rot=0)),
    (2, "rotated", dict(rot=7)),
    (2, "rotated", dict(rot=66)),
    (1, "null x", dict(x=None)),
    (1, "null out", dict(out=None)),
    (1, "null pointer", dict(pos=None)),
    (1, "null pointer", dict(freq=None)),
    (1, "scale", dict(scale=math.nan)),
    (1, "scale", dict(scale=math.inf)),
    (2, "stride", dict(xt=-1)),
    (2, "stride", dict(oh=1 << 30)),
    (3, "aligned", dict(x=ODD)),
    (3, "aligned", dict(out=ODD)),
    (3, "misaligned", dict(pos=ctypes.c_void_p((3 << 28) + 4))),
    (3, "misaligned", dict(freq=ctypes.c_void_p((4 << 28) + 4))),
    (2, "vectors overlap", dict(ot=255)),
    (2, "vectors overlap", dict(oh=63)),
    (2, "vectors overlap", dict(ot=64, oh=64)),
    (1, "out overlaps x", dict(out=ctypes.c_void_p((1 << 28) + 128))),
    (1, "out overlaps x", dict(out=A, ot=64, oh=320)),
    (1, "overlaps positions", dict(pos=ctypes.c_void_p((2 << 28) + 64))),
    (1, "overlaps positions", dict(freq=ctypes.c_void_p((2 << 28) + 64))),
])
def test_rotary_refuses(lib, rc, text, kw):
    got, msg = turn(lib, **kw)
    assert got == rc and text in msg and "rotary" in msg


def test_rotary_of_nothing(lib):
    for kw in (dict(tokens=0), dict(heads=0)):
        assert turn(lib, x=None, out=None, pos=None, **kw) == (0, "")


@no_device
def test_rotary_beside_its_input(lib):
    """In place, and where x and out share rows but no element, a call goes on to the launch."""
    for kw in (dict(out=A), dict(xt=512, out=ctypes.c_void_p((1 << 28) + 512), ot=512), dict(tokens=1, out=A, ot=0),
               dict(xt=64, xh=5 * 64, ot=64, oh=5 * 64)):
        rc, text = turn(lib, **kw)
        assert rc not in (1, 2, 3), text


def write(lib, c, q=A, qt=256, qh=64, heads=4, out=B, ot=256, oh=64, k=C, kt=128, kh=64, v=D, vt=128, vh=64, dtype=Q.BF16,
          pos=E, freq=F, rot=64, inter=0, scale=1.0, slots=G, tokens=3):
    return lib.phi_hip_rotary_cache_write(None, ctypes.byref(c) if c else None, q, qt, qh, heads, out, ot, oh, k, kt, kh, v, vt,
                                          vh, dtype, pos, freq, rot, inter, scale, slots, tokens)


@pytest.mark.parametrize("rc,text,kw", BAD_CACHES)
def test_bad_caches_are_refused(lib, rc, text, kw):
    assert write(lib, cache(**kw)) == rc and text in Q.last_error()
    assert copy(lib, cache(**kw), far()) == rc and text in Q.last_error()
    assert copy(lib, far(), cache(**kw)) == rc and text in Q.last_error()
    assert write(lib, None) == copy(lib, None, far()) == copy(lib, far(), None) == 1


@pytest.mark.parametrize("rc,text,kw", [
    (2, "negative", dict(tokens=-1)),
    (2, "negative", dict(heads=-1)),
    (2, "out of range", dict(heads=70000)),
    (1, "f32 or bf16", dict(dtype=Q.I8)),
    (1, "null q", dict(q=None)),
    (1, "null q_out", dict(out=None)),
    (1, "null k", dict(k=None)),
    (1, "null v", dict(v=None)),
    (1, "null slots", dict(slots=None)),
    (1, "null pointer", dict(pos=None)),
    (1, "null pointer", dict(freq=None)),
    (2, "rotated", dict(rot=66)),
    (2, "rotated", dict(rot=1)),
    (1, "scale", dict(scale=math.inf)),
    (3, "aligned", dict(q=OFF8)),
    (3, "aligned", dict(ot=257)),
    (3, "aligned", dict(kt=129)),
    (2, "stride", dict(qt=-256)),
    (2, "vectors overlap", dict(ot=128)),
    (1, "q_out overlaps q", dict(out=ctypes.c_void_p((1 << 28) + 128))),
    (1, "q_out overlaps k", dict(out=ctypes.c_void_p((3 << 28) + 16))),
    (1, "q_out overlaps k", dict(out=D)),
    (1, "q_out overlaps k", dict(out=ctypes.c_void_p(K2 + 512))),
    (1, "q_out overlaps positions", dict(out=E)),
    (1, "q_out overlaps positions", dict(out=G)),
])
def test_rotary_cache_write_refuses(lib, rc, text, kw):
    assert write(lib, far(), **kw) == rc and text in Q.last_error() and "rotary_cache_write" in Q.last_error()


def test_rotary_cache_write_of_a_cache_that_overlaps(lib):
    assert write(lib, far(token_stride=48)) == 2 and "overlap" in Q.last_error()
    assert write(lib, far(s_head_stride=0)) == 2 and "overlap" in Q.last_error()
    assert write(lib, far(), tokens=0, q=None, k=None, v=None, slots=None) == 0 and Q.last_error() == ""


def copy(lib, a, b, frm=A, to=B, tokens=None, n=3):
    return lib.phi_hip_kv_cache_copy(None, ctypes.byref(a) if a else None, ctypes.byref(b) if b else None, frm, to, tokens, n)


@pytest.mark.parametrize("rc,text,a,b,kw", [
    (2, "heads, page, dim", dict(), dict(heads=1), {}),
    (2, "heads, page, dim", dict(page=8), dict(), {}),
    (2, "heads, page, dim", dict(dim=32), dict(), {}),
    (2, "too large", dict(page=1 << 20, heads=65), dict(page=1 << 20, heads=65, token_stride=65 * 64, head_stride=64,
                                                        s_token_stride=65, s_head_stride=1,
                                                        block_stride=1 << 33, s_block_stride=1 << 30), {}),
    (2, "overlap", dict(), dict(block_stride=0), {}),
    (2, "out of range", dict(), dict(), dict(n=-1)),
    (2, "out of range", dict(), dict(), dict(n=1 << 31)),
    (1, "null", dict(), dict(), dict(frm=None)),
    (1, "null", dict(), dict(), dict(to=None)),
    (3, "misaligned", dict(), dict(), dict(to=ODD)),
    (3, "misaligned", dict(), dict(), dict(tokens=ODD)),
])
def test_copy_refuses(lib, rc, text, a, b, kw):
    assert copy(lib, far(**a), far(**b), **kw) == rc and text in Q.last_error()


def test_copy_of_nothing(lib):
    assert copy(lib, far(), far(), frm=None, to=None, n=0) == 0 and Q.last_error() == ""


def adapt(lib, x=A, xd=Q.BF16, ldx=512, rows=4, K=512, a=B, aa=16 * 512, ar=512, b=C, ba=256 * 16, br=16, wd=Q.BF16, n=3, rank=16, N=256,
          adapter=D, scale=E, base=F, ldb=256, out=G, od=Q.BF16, ldo=256, ws=ctypes.c_void_p(8 << 28), wn=1 << 20):
    return lib.phi_hip_lora_batched(None, x, xd, ldx, rows, K, a, aa, ar, b, ba, br, wd, n, rank, N, adapter, scale, base, ldb, out, od,
                                    ldo, ws, wn)


@pytest.mark.parametrize("rc,text,kw", [
    (2, "negative", dict(rows=-1)),
    (2, "negative", dict(rank=-1)),
    (2, "negative", dict(n=-1)),
    (1, "dtypes", dict(xd=Q.F16)),
    (1, "dtypes", dict(wd=Q.I8)),
    (1, "dtypes", dict(od=Q.I32)),
    (2, "empty factors", dict(K=0)),
    (2, "empty factors", dict(rank=0)),
    (2, "empty factors", dict(n=0)),
    (7, "exceeds", dict(rank=257, br=257)),
    (2, "out of range", dict(rows=(1 << 24) + 1)),
    (2, "out of range", dict(N=(1 << 24) + 1, ldo=1 << 25, ldb=1 << 25)),
    (2, "out of range", dict(n=1 << 31)),
    (1, "null", dict(x=None)),
    (1, "null", dict(a=None)),
    (1, "null", dict(b=None)),
    (1, "null", dict(adapter=None)),
    (1, "null", dict(out=None)),
    (2, "leading", dict(ldx=511)),
    (2, "leading", dict(ldo=255)),
    (2, "leading", dict(ldb=255)),
    (2, "leading", dict(ar=511)),
    (2, "leading", dict(br=15)),
    (2, "too large", dict(ldx=1 << 30)),
    (2, "adapter stride", dict(aa=-1)),
    (2, "adapter stride", dict(ba=1 << 41)),
    (3, "aligned", dict(x=ODD)),
    (3, "aligned", dict(out=ODD)),
    (3, "aligned", dict(adapter=ctypes.c_void_p((4 << 28) + 2))),
    (3, "aligned", dict(scale=ctypes.c_void_p((5 << 28) + 2))),
    (4, "workspace", dict(ws=None)),
    (4, "workspace", dict(wn=100)),
    (3, "workspace", dict(ws=ctypes.c_void_p((8 << 28) + 8))),
    (1, "out overlaps an input", dict(out=ctypes.c_void_p((1 << 28) + 64))),
    (1, "out overlaps an input", dict(out=ctypes.c_void_p((2 << 28) + 2 * 16 * 512 * 2 - 64))),
    (1, "out overlaps an input", dict(out=C)),
    (1, "out overlaps an input", dict(adapter=G)),
    (1, "out overlaps base", dict(out=ctypes.c_void_p((6 << 28) + 256))),
    (1, "out overlaps base", dict(out=F, ldo=512)),
    (1, "workspace overlaps", dict(ws=F)),
    (1, "workspace overlaps", dict(ws=G)),
    (1, "workspace overlaps", dict(ws=A)),
])
def test_adapters_refuse(lib, rc, text, kw):
    assert adapt(lib, **kw) == rc and text in Q.last_error() and "lora_batched" in Q.last_error()


def test_adapters_of_nothing(lib):
    for kw in (dict(rows=0), dict(N=0)):
        assert adapt(lib, x=None, out=None, ws=None, **kw) == 0 and Q.last_error() == ""
    size = lib.phi_hip_lora_batched_workspace_bytes
    assert size(0, 5, 5) == size(5, 0, 5) == size(5, 5, 0) == size(5, 5, 257) == size(1 << 25, 5, 5) == 0
    assert size(1, 1, 1) >= 4 and size(1000, 4096, 16) >= 1000 * 16 * 4


H = ctypes.c_void_p(8 << 28)


def shared(lib, c, q=A, dtype=Q.BF16, qt=256, qh=64, tokens=8, heads=4, ptable=B, pwidth=6, pstride=6, plen=C, first=D, groups=2, max_prefix=96,
           table=E, width=4, stride=4, start=F, lens=F, batch=3, max_q=4, max_kv=64, scale=0.1, out=G, ot=256, oh=64, ws=H, wn=1 << 28):
    return lib.phi_hip_paged_attention_shared(None, q, dtype, qt, qh, tokens, heads, ctypes.byref(c) if c else None, ptable, pwidth, pstride, plen,
                                              first, groups, max_prefix, table, width, stride, start, lens, batch, max_q, max_kv, scale, out, ot, oh,
                                              ws, wn)


@pytest.mark.parametrize("rc,text,kw", [
    (2, "negative", dict(tokens=-1)),
    (2, "negative", dict(groups=-1)),
    (2, "negative", dict(max_prefix=-1)),
    (1, "f32 or bf16", dict(dtype=Q.F16)),
    (2, "5 query heads for 2", dict(heads=5)),
    (2, "out of range", dict(max_q=9)),
    (2, "out of range", dict(batch=70000)),
    (2, "out of range", dict(groups=70000)),
    (2, "out of range", dict(max_prefix=(1 << 30) + 1)),
    (2, "out of range", dict(tokens=(1 << 29) + 1)),
    (2, "out of range", dict(tokens=1 << 24)),
    (2, "no groups", dict(groups=0)),
    (2, "block table", dict(max_kv=65)),
    (2, "prefix table", dict(max_prefix=97)),
    (2, "stride", dict(stride=3)),
    (2, "stride", dict(pstride=5)),
    (1, "scale", dict(scale=math.inf)),
    (1, "null q", dict(q=None)),
    (1, "null out", dict(out=None)),
    (1, "null pointer", dict(table=None)),
    (1, "null pointer", dict(ptable=None)),
    (1, "null pointer", dict(plen=None)),
    (1, "null pointer", dict(first=None)),
    (1, "null pointer", dict(start=None)),
    (1, "null pointer", dict(lens=None)),
    (3, "aligned", dict(qt=257)),
    (3, "misaligned", dict(plen=ODD)),
    (3, "misaligned", dict(ptable=ODD)),
    (2, "vectors overlap", dict(ot=128)),
    (1, "out overlaps q", dict(out=ctypes.c_void_p((1 << 28) + 1024))),
    (4, "workspace", dict(ws=None)),
    (4, "workspace", dict(wn=64)),
    (3, "workspace", dict(ws=ctypes.c_void_p((8 << 28) + 8))),
    (1, "workspace overlaps", dict(ws=A)),
    (1, "workspace overlaps", dict(ws=G)),
    (1, "workspace overlaps", dict(ws=ctypes.c_void_p(K2))),
    (1, "out overlaps the cache", dict(out=ctypes.c_void_p(K2))),
])
def test_shared_attention_refuses(lib, rc, text, kw):
    assert shared(lib, far(), **kw) == rc and text in Q.last_error() and "paged_attention_shared" in Q.last_error()


@pytest.mark.parametrize("rc,text,kw", BAD_CACHES)
def test_shared_attention_of_bad_caches(lib, rc, text, kw):
    assert shared(lib, cache(**kw)) == rc and text in Q.last_error()


def test_shared_attention_of_nothing(lib):
    for kw in (dict(tokens=0), dict(batch=0), dict(max_q=0)):
        assert shared(lib, far(), q=None, out=None, ws=None, **kw) == 0 and Q.last_error() == ""
    size = lib.phi_hip_paged_attention_shared_workspace_bytes
    for bad in ((0, 4, 2, 64, 1, 1, 10, 1, 10), (8, 5, 2, 64, 1, 1, 10, 1, 10), (8, 4, 2, 64, 0, 1, 10, 1, 10), (8, 4, 2, 64, 1, 1, 10, 9, 10),
                (8, 4, 2, 64, 1, 70000, 10, 1, 10)):
        assert size(*bad, Q.BF16) == 0
    assert size(8, 4, 2, 64, 1, 8, 10, 1, 0, Q.BF16) > 0


def test_python_refusals():
    t = torch.zeros((2, 3, 64))
    with pytest.raises(ValueError, match="device"):
        Q.rotary(t, torch.zeros(2, dtype=torch.int64), torch.ones(32, dtype=torch.float64))


def test_plain_rotation_is_one():
    x = torch.randn((3, 2, 10), dtype=torch.float64, generator=torch.Generator().manual_seed(1))
    f = torch.tensor([1.0, 0.25, 0.01], dtype=torch.float64)
    p = torch.tensor([0, 5, -3])
    for inter in (False, True):
        y, _ = R.rotated(x, p, f, inter, 1.0)
        assert torch.allclose(y.square().sum(-1), x.square().sum(-1)) and torch.equal(y[0], x[0]) and torch.equal(y[..., 6:], x[..., 6:])
        assert torch.allclose(R.rotated(y, -p, f, inter, 1.0)[0], x, atol=1e-14)


# ------------------------------------------------------------------ frequencies
def test_frequencies():
    f = Q.rotary_frequencies(8, 10000.0, device="cpu")
    assert f.dtype == torch.float64 and torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-15)
    assert torch.allclose(Q.rotary_frequencies(8, scaling="linear", factor=4.0, device="cpu"), f / 4, rtol=1e-15)
    ntk = Q.rotary_frequencies(8, scaling="ntk", factor=4.0, device="cpu")
    assert ntk[0] == 1 and math.isclose(ntk[3], f[3] / 4, rel_tol=1e-14) and bool((ntk[1:] < f[1:]).all())


@pytest.mark.parametrize("rule", ["parts", "ramp"])
def test_frequencies_by_parts(rule):
    """Short waves as they are, long ones stretched, falling between."""
    f = Q.rotary_frequencies(128, 500000.0, device="cpu")
    g = Q.rotary_frequencies(128, 500000.0, scaling=rule, factor=8.0, length=8192, slow=1.0, fast=4.0, device="cpu")
    turns, ratio = 8192 * f / (2 * math.pi), g / f
    few, many = turns < (1.0 if rule == "parts" else 0.7), turns > (4.0 if rule == "parts" else 6.0)
    assert torch.allclose(ratio[few], torch.full_like(ratio[few], 1 / 8), rtol=1e-14) and few.sum() > 5
    assert bool((ratio[many] == 1).all()) and many.sum() > 5
    assert bool((ratio[:-1] >= ratio[1:]).all()) and 1 / 8 < ratio[~few & ~many].median() < 1


@pytest.mark.parametrize("kw", [dict(rot=7), dict(rot=0), dict(rot=8, scaling="other"), dict(rot=2, scaling="ntk")])
def test_frequencies_refuse(kw):
    with pytest.raises(ValueError):
        Q.rotary_frequencies(device="cpu", **kw)


# ------------------------------------------------------------------ pages
class Plain(dict):
    """Sequences' tokens as they should be, and the memory that the pages say."""

    def __init__(self, blocks, page):
        super().__init__()
        self.page, self.memory, self.next = page, [None] * (blocks * page), 0

    def grow(self, pages, seq, n):
        slots = pages.grow(seq, n)
        self.flush(pages)
        for s in slots:
            self.memory[s] = self.next
            self.setdefault(seq, []).append(self.next)
            self.next += 1
        self.setdefault(seq, [])

    def flush(self, pages):
        for a, b, n in pages.copies:
            self.memory[b * self.page:b * self.page + n] = self.memory[a * self.page:a * self.page + n]
        pages.copies = []

    def check(self, pages):
        for seq, want in self.items():
            assert pages.length[seq] == len(want) and len(pages.of[seq]) == -(-len(want) // self.page)
            assert [self.memory[pages.of[seq][t // self.page] * self.page + t % self.page] for t in range(len(want))] == want
        users = [0] * len(pages.users)
        for row in pages.of.values():
            for b in row:
                users[b] += 1
        assert users == pages.users and sorted(pages.free) == [b for b, n in enumerate(users) if not n]


@pytest.mark.parametrize("seed", range(6))
def test_pages_through_a_life(seed):
    """Growth, forks, ends and compaction in any order, copies left for later or not:
    every sequence keeps its tokens."""
    rng = random.Random(seed)
    page, blocks = rng.choice([1, 4, 16]), 60
    pages, plain, names = Q.KvPages(blocks, page), Plain(blocks, page), 0
    for _ in range(300):
        act = rng.choice("gggfec")
        if act == "g":
            seq = rng.choice(list(plain) + [names])
            n = rng.choice([0, 1, 1, 3, page, 2 * page + 1])
            need = -(-(pages.length.get(seq, 0) + n) // page) - len(pages.of.get(seq, []))
            if need > len(pages.free):
                before = (dict(pages.of), dict(pages.length), list(pages.free))
                with pytest.raises(RuntimeError, match="full"):
                    pages.grow(seq, n)
                assert before == (pages.of, pages.length, pages.free)
            else:
                plain.grow(pages, seq, n)
                names += seq == names
        elif act == "f" and plain and pages.free:
            parent = rng.choice(list(plain))
            pages.fork(parent, names)
            plain[names] = list(plain[parent])
            assert pages.shared([parent, names]) == len(plain[parent]) // page
            names += 1
        elif act == "e" and plain:
            seq = rng.choice(list(plain))
            pages.end(seq)
            del plain[seq]
        elif act == "c":
            n = pages.compact()
            assert n == sum(1 for u in pages.users if u) and all(pages.users[:n]) and not any(pages.users[n:])
        if rng.random() < 0.5:
            plain.flush(pages)
            plain.check(pages)
    plain.flush(pages)
    plain.check(pages)


def test_copies_go_in_calls_without_hazards(monkeypatch):
    """What a call writes it neither reads nor writes again, and the order is kept."""
    calls = []
    monkeypatch.setattr(Q.serving, "kv_cache_copy", lambda a, b, frm, to, tokens: calls.append(
        list(zip(frm.tolist(), to.tolist(), tokens.tolist()))))

    class Host:
        k = torch.zeros(1)

    rng = random.Random(3)
    for _ in range(200):
        pages = Q.KvPages(8, 4)
        todo = [(a, b, rng.randint(1, 4)) for a, b in (rng.sample(range(8), 2) for _ in range(rng.randint(1, 8)))]
        pages.copies = list(todo)
        calls.clear()
        pages.flush(Host)
        assert [c for call in calls for c in call] == todo and pages.copies == []
        for call in calls:
            to = [b for _, b, _ in call]
            assert len(set(to)) == len(to) and not set(to) & {a for a, _, _ in call}


def test_pages_refuse():
    pages = Q.KvPages(4, 4)
    pages.grow("a", 5)
    for bad in (lambda: pages.fork("a", "a"), lambda: pages.grow("a", -1)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(KeyError):
        pages.fork("x", "b")
    assert pages.of == {"a": [0, 1]} and pages.copies == []
