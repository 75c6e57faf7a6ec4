"""What a server of many requests runs beside a decoder layer's int8 linears, as
cases that can be timed.

Rotary positions before the paged cache, pages of that cache copied when
sequences fork or are moved together, attention of sequences that share a prefix,
and the low-rank adapters of many requests beside one linear.  Sizes are the
repository's own (4352 and 32760 tokens, hidden 5120, prompts of 77) or generic
ones around them; ``draw`` spreads over the ranges that the listed cases stand
for.

The kinds:

  rotary    vectors of heads rotated by their tokens' positions
  write     the same for a projection's q and k, with k and v quantised into the
            paged cache, and the same slots read back
  copy      pages of the cache copied within it
  shared    a batch's new tokens over their groups' prefixes and their own tokens
  lora      a linear's output plus each row's own adapter

``run`` computes a case with elementary torch operations in 32 bits (angles: 64)
where ``own`` is false, and calls this repository's operators where it is true.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"bf16": 2, "f32": 4}


def _package():
    pkg = os.path.join(os.getcwd(), "phi-agent_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import phi_qlinear

    return phi_qlinear


def listed() -> list[dict]:
    return [
        # Part of a narrow head, neighbouring pairs, activations in 32 bits: a text encoder's prompts.
        dict(name="rotary_part", kind="rotary", T=777, H=20, D=80, rot=64, inter=True, far=4352, stretch=1.0, x="f32"),
        # A long prompt's queries and keys at far positions of a stretched context.
        dict(name="rotary_prompt", kind="rotary", T=32760, H=40, D=128, rot=128, inter=False, far=1 << 20, stretch=8.0,
             x="bf16"),
        # A decode step of 64 sequences (a quarter of the batch's places empty).
        dict(name="write_step", kind="write", T=64, Hq=32, H=8, D=128, rot=128, inter=False, far=131072, stretch=4.0,
             page=16, x="bf16", step=True),
        # A prompt's projection written page by page.
        dict(name="write_prompt", kind="write", T=4352, Hq=40, H=8, D=128, rot=128, inter=False, far=32768, stretch=1.0,
             page=64, x="bf16", step=False),
        # Sixteen sequences fork: the last page of each, in part.
        dict(name="copy_fork", kind="copy", n=16, blocks=1024, H=8, D=128, page=16, part=True),
        # A cache's pages moved together.
        dict(name="copy_compact", kind="copy", n=2048, blocks=4608, H=8, D=128, page=64, part=False),
        # A few answers to one prompt: the smallest attention with a prefix.
        dict(name="shared_few", kind="shared", B=4, groups=1, Hq=32, Hkv=8, D=128, page=16, max_prefix=777, max_q=1,
             max_kv=200, q="bf16"),
        # A full batch behind one long instruction.
        dict(name="shared_batch", kind="shared", B=64, groups=1, Hq=32, Hkv=8, D=128, page=16, max_prefix=8192, max_q=1,
             max_kv=1024, q="bf16"),
        # Several long documents with many questions each, the largest call; a few new tokens each.
        dict(name="shared_documents", kind="shared", B=96, groups=3, Hq=40, Hkv=8, D=128, page=64, max_prefix=32760,
             max_q=4, max_kv=2001, q="bf16"),
        # A decode step in which most rows have an adapter, any of 32.
        dict(name="lora_step", kind="lora", T=64, K=4096, N=6144, R=16, adapters=32, x="bf16", w="bf16", out="bf16",
             runs=False),
        # Prompts of eight requests, an adapter each.
        dict(name="lora_prompts", kind="lora", T=4352, K=5120, N=5120, R=64, adapters=8, x="bf16", w="bf16", out="bf16",
             runs=True),
        # Factors and activations in 32 bits at sizes that are no whole number of anything.
        dict(name="lora_odd", kind="lora", T=77, K=5003, N=1701, R=5, adapters=3, x="f32", w="f32", out="f32", runs=True),
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["rotary", "write", "copy", "shared", "shared", "lora", "lora"])
    x = rng.choice(["bf16", "bf16", "f32"])
    D = rng.choice([64, 80, 96, 128, 128, 192, 256])
    if kind in ("rotary", "write"):
        if kind == "rotary" and rng.random() < 0.3:
            D = rng.randint(9, 160)
        H = _log(rng, 1, 40 if kind == "rotary" else 16)
        rot = rng.choice([D // 2 * 2, D // 2 * 2, D // 4 * 2, 2 * rng.randint(1, D // 2)])
        c = dict(kind=kind, H=H, D=D, rot=rot, inter=rng.random() < 0.4, far=_log(rng, 1 << 10, 1 << 24),
                 stretch=rng.choice([1.0, 1.0, 4.0, 8.0]), x=x)
        if kind == "rotary":
            return dict(c, T=_log(rng, 1, min(32760, 32760 * 40 * 128 // (H * D * BYTES[x] // 2))))
        step = rng.random() < 0.4
        G = rng.choice([1, 2, 4, 5, 8])
        return dict(c, Hq=H * G, page=rng.choice([8, 16, 16, 24, 32, 64, 128]), step=step,
                    T=_log(rng, 1, 256 if step else min(16384, 4352 * 56 * 128 * 4 // (H * (G + 2) * D * BYTES[x]))))
    page = rng.choice([8, 16, 16, 24, 32, 64, 128, 256])
    if kind == "copy":
        H = _log(rng, 1, 16)
        n = _log(rng, 1, max(1, 2048 * 64 * 8 * 128 // (page * H * D)))
        n = min(n, 16384)
        return dict(kind=kind, n=n, blocks=2 * n + rng.randint(1, 99), H=H, D=D, page=page, part=rng.random() < 0.5)
    if kind == "lora":
        K, N, R = _log(rng, 256, 8192), _log(rng, 256, 12288), _log(rng, 1, 128)
        runs = rng.random() < 0.5
        adapters = _log(rng, 1, 64)
        top = 4352 * 10240 // max(K + N, 2 * (K + N) * R * adapters // (8 * 64)) if runs else 256
        return dict(kind=kind, T=_log(rng, 1, min(8192, max(1, top))), K=K, N=N, R=R, adapters=adapters, x=x,
                    w=rng.choice(["bf16", "bf16", "f32"]), out=x, runs=runs)
    H, G = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 4, 4, 5, 7, 8])
    B = _log(rng, 1, 128)
    max_q = 1 if rng.random() < 0.6 else _log(rng, 2, 64)
    groups = min(B, rng.choice([1, 1, 1, 2, 3, 5]))
    max_kv = _log(rng, max(max_q, 8), 4096)
    while B * max_q * H * G * D > 96 * 4 * 40 * 128 or B * H * D * max_kv > 96 * 8 * 128 * 2001:
        B, max_q = max(1, B // 2), max(1, max_q // 2)
        groups, max_kv = min(B, groups), max(max_q, max_kv // 2)
    top = min(65536, 96 * 4 * 40 * 32760 * 128 // (3 * B * max_q * H * G * max(D, 128)))
    return dict(kind="shared", B=B, groups=groups, Hq=H * G, Hkv=H, D=D, page=page, max_prefix=_log(rng, 64, max(64, top)),
                max_q=max_q, max_kv=max_kv, q=x)


def _members(c: dict):
    """Of a shared case: each group's prefix length and its sequences' (new
    tokens, own tokens with them); then those of sequences of no group.  Part of
    the case.  The first of each is the longest; of five sequences or more, the
    last is an empty place of the batch."""
    rng = random.Random(1000003 * c["max_prefix"] + 1009 * c["max_kv"] + 31 * c["B"] + c["max_q"])
    free = 1 if c["B"] >= 5 and c["B"] > c["groups"] else 0
    cuts = sorted(rng.sample(range(1, c["B"] - free), c["groups"] - 1))
    sizes = [b - a for a, b in zip([0] + cuts, cuts + [c["B"] - free])]
    got = []
    for g, n in enumerate(sizes):
        prefix = c["max_prefix"] if g == 0 else rng.randint(c["max_prefix"] // 2, c["max_prefix"])
        seqs = []
        for i in range(n):
            new = c["max_q"] if g == 0 and i == 0 else _log(rng, 1, c["max_q"])
            seqs.append((new, c["max_kv"] if g == 0 and i == 0 else rng.randint(new, c["max_kv"])))
        got.append((prefix, seqs))
    return got, [(1, 0)] * free


# ------------------------------------------------------------------ inputs
def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(shape, seed: int, scale: float = 1.0, dtype=torch.float32) -> torch.Tensor:
    return (torch.randn(shape, generator=_gen(seed), device=DEV) * scale).to(dtype)


def _codes(shape, seed: int) -> torch.Tensor:
    """int8 codes of normally distributed vectors (absmax near 127)."""
    got = torch.empty(shape, dtype=torch.int8, device=DEV)
    flat, g, step = got.view(-1), _gen(seed), 1 << 26
    for i in range(0, flat.numel(), step):
        n = min(step, flat.numel() - i)
        flat[i:i + n] = (torch.randn(n, generator=g, device=DEV) * 42).round_().clamp_(-127, 127).to(torch.int8)
    return got


def _scales(shape, seed: int) -> torch.Tensor:
    return torch.rand(shape, generator=_gen(seed), device=DEV) * 0.02 + 0.01


def _frequencies(rot: int, stretch: float) -> torch.Tensor:
    """Radians a position, 10000^(-2 j / rot); of a context stretched by a factor
    the waves longer than 8192 positions are that much longer, those shorter than
    2048 as they were."""
    f = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if stretch != 1.0:
        wave = 2 * math.pi / f
        keep = ((8192 / wave - 1) / 3).clamp(0, 1)
        f = f * (keep + (1 - keep) / stretch)
    return f.to(DEV)


def prepare(case: dict, seed: int) -> dict:
    s = seed * 16  # a stream of its own for every tensor
    st, c = dict(case=case), case
    if c["kind"] == "lora":
        T, K, N, R, n = c["T"], c["K"], c["N"], c["R"], c["adapters"]
        # The rows of requests: neighbours have one adapter (prompts), or any has any or none (a step).
        if c["runs"]:
            adapter = torch.arange(T, device=DEV) * n // T
        else:
            adapter = torch.randint(-(n // 8), n, (T,), generator=_gen(s), device=DEV).clamp(min=-1)
        w = DTYPES[c["w"]]
        st.update(x=_randn((T, K), s + 1, 1.0, DTYPES[c["x"]]), base=_randn((T, N), s + 2, 1.0, DTYPES[c["out"]]),
                  A=_randn((n, R, K), s + 3, K ** -0.5, w), B=_randn((n, N, R), s + 4, R ** -0.5, w),
                  adapter=adapter.to(torch.int32), scale=torch.rand((n,), generator=_gen(s + 5), device=DEV) + 0.5)
        return st
    H, D = c.get("Hkv", c.get("H")), c["D"]
    if c["kind"] == "rotary":
        T = c["T"]
        start = torch.randint(0, c["far"], (1,), generator=_gen(s), device=DEV)
        st.update(x=_randn((T, H, D), s + 1, 1.0, DTYPES[c["x"]]), pos=start + torch.arange(T, device=DEV),
                  freq=_frequencies(c["rot"], c["stretch"]), factor=0.1 * math.log(c["stretch"]) + 1.0)
        return st
    page = c["page"]
    if c["kind"] == "write":
        T = c["T"]
        # q, k and v are columns of the fused projection's output.
        qkv = _randn((T, c["Hq"] + 2 * H, D), s, 1.0, DTYPES[c["x"]])
        qkv[:, :, ::61] *= 6
        pages = T if c["step"] else -(-T // page)
        blocks = pages + 3
        order = torch.randperm(blocks, generator=_gen(s + 1), device=DEV)[:pages]
        if c["step"]:  # one token a sequence, each on a page of its own; every fourth place is empty
            pos = torch.randint(0, c["far"], (T,), generator=_gen(s + 2), device=DEV)
            slots = order * page + pos % page
            slots[3::4] = -1
        else:
            at = torch.arange(T, device=DEV)
            pos = at + torch.randint(0, c["far"], (1,), generator=_gen(s + 2), device=DEV) // page * page
            slots = order[at // page] * page + at % page
        st.update(q=qkv[:, :c["Hq"]], k=qkv[:, c["Hq"]:c["Hq"] + H], v=qkv[:, c["Hq"] + H:], slots=slots, pos=pos,
                  freq=_frequencies(c["rot"], c["stretch"]), factor=0.1 * math.log(c["stretch"]) + 1.0)
    elif c["kind"] == "copy":
        blocks, n = c["blocks"], c["n"]
        order = torch.randperm(blocks, generator=_gen(s), device=DEV).to(torch.int32)
        st.update(frm=order[:n].contiguous(), to=order[n:2 * n].contiguous(), tokens=None,
                  kc=_codes((blocks, H, page, D), s + 1), vc=_codes((blocks, H, page, D), s + 2),
                  ks=_scales((blocks, H, page), s + 3), vs=_scales((blocks, H, page), s + 4))
        if c["part"]:
            st["tokens"] = torch.randint(1, page + 1, (n,), generator=_gen(s + 5), device=DEV).to(torch.int32)
        return st
    else:
        return _prepare_shared(st, s)
    kc, vc = (torch.zeros((blocks, H, page, D), dtype=torch.int8, device=DEV) for _ in range(2))
    ks, vs = (torch.ones((blocks, H, page), dtype=torch.float32, device=DEV) for _ in range(2))
    st.update(kc=kc, vc=vc, ks=ks, vs=vs)
    return st


def _prepare_shared(st: dict, s: int) -> dict:
    c = st["case"]
    H, D, page = c["Hkv"], c["D"], c["page"]
    groups, free = _members(c)
    seqs = [m for _, members in groups for m in members] + free
    lens = [p for p, _ in groups] + [kv for _, kv in seqs]
    need = [-(-n // page) for n in lens]
    blocks = sum(need) + 1
    order = torch.randperm(blocks, generator=_gen(s), device=DEV).tolist()
    widths = [max(1, -(-c["max_prefix"] // page)), max(1, -(-c["max_kv"] // page))]
    tables = [torch.full((len(groups), widths[0]), -1, dtype=torch.int32),
              torch.full((len(seqs), widths[1]), -1, dtype=torch.int32)]
    kc, vc = _codes((blocks, H, page, D), s + 1), _codes((blocks, H, page, D), s + 2)
    ks, vs = _scales((blocks, H, page), s + 3), _scales((blocks, H, page), s + 4)
    for i, (n, tokens) in enumerate(zip(need, lens)):
        ids = [order.pop() for _ in range(n)]
        table, row = (tables[0], i) if i < len(groups) else (tables[1], i - len(groups))
        table[row, :n] = torch.tensor(ids, dtype=torch.int32)
        if tokens % page:  # what lies past the end in its last page was never written
            ks[ids[-1], :, tokens % page:] = math.nan
            vs[ids[-1], :, tokens % page:] = math.nan
    starts, firsts = [0], [0]
    for new, _ in seqs:
        starts.append(starts[-1] + new)
    for _, members in groups:
        firsts.append(firsts[-1] + len(members))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    # q is columns of the fused projection's output.
    qkv = _randn((starts[-1], c["Hq"] + 2 * H, D), s + 5, 1.5, DTYPES[c["q"]])
    st.update(q=qkv[:, :c["Hq"]], kc=kc, vc=vc, ks=ks, vs=vs, prefix_table=tables[0].to(DEV), table=tables[1].to(DEV),
              prefix_len=i32([p for p, _ in groups]), group_start=i32(firsts), starts=i32(starts),
              kv_len=i32([kv for _, kv in seqs]), scale=D ** -0.5)
    return st


# ------------------------------------------------------------------ one pass
def run(st: dict):
    return (_OWN if own else _PLAIN)[st["case"]["kind"]](st)


def _rotary_own(st: dict):
    return _package().rotary(st["x"], st["pos"], st["freq"], interleaved=st["case"]["inter"], scale=st["factor"])


def _write_own(st: dict):
    Q = _package()
    cache = Q.KvCache(st["kc"], st["vc"], st["ks"], st["vs"])
    q = Q.rotary_cache_write(cache, st["q"], st["k"], st["v"], st["pos"], st["freq"], st["slots"],
                             interleaved=st["case"]["inter"], scale=st["factor"])
    # Codes have 8 bits, so bf16 holds what they stand for.
    return (q, *Q.kv_cache_read(cache, st["slots"], out_dtype=torch.bfloat16))


def _copy_own(st: dict):
    Q = _package()
    cache = Q.KvCache(st["kc"], st["vc"], st["ks"], st["vs"])
    Q.kv_cache_copy(cache, cache, st["frm"], st["to"], tokens=st["tokens"])
    # Codes as they are: a copy rounds nothing, so they are whole numbers that have to be equal.
    return st["kc"], st["vc"], st["ks"], st["vs"]


def _shared_own(st: dict):
    Q, c = _package(), st["case"]
    cache = Q.KvCache(st["kc"], st["vc"], st["ks"], st["vs"])
    return Q.paged_attention_shared(st["q"], cache, st["prefix_table"], st["prefix_len"], st["group_start"], st["table"],
                                    st["starts"], st["kv_len"], max_prefix=c["max_prefix"], max_q=c["max_q"],
                                    max_kv=c["max_kv"], scale=st["scale"])


def _lora_own(st: dict):
    return _package().lora_batched(st["x"], st["A"], st["B"], st["adapter"], scale=st["scale"], base=st["base"])


def _rotated_plain(x: torch.Tensor, st: dict) -> torch.Tensor:
    """x [tokens, heads, dim] rotated, fp32."""
    half = st["case"]["rot"] // 2
    angle = st["pos"].double()[:, None] * st["freq"]
    cos, sin = ((f(angle) * st["factor"]).float()[:, None] for f in (torch.cos, torch.sin))
    x = x.float()
    y = x.clone()
    at = torch.arange(half, device=DEV)
    first, second = (2 * at, 2 * at + 1) if st["case"]["inter"] else (at, at + half)
    a, b = x[..., first], x[..., second]
    y[..., first] = a * cos - b * sin
    y[..., second] = b * cos + a * sin
    return y


def _rotary_plain(st: dict):
    return _rotated_plain(st["x"], st).to(st["x"].dtype)


def _quantise_plain(y: torch.Tensor):
    """Codes (as floats) and scale of the last axis, ties away from zero."""
    amax = y.abs().amax(dim=-1)
    s = torch.where(amax > 1e-30, amax / 127.0, torch.ones_like(amax))
    d = y * (1.0 / s)[..., None]
    return (torch.sign(d) * torch.floor(d.abs() + 0.5)).clamp(-127, 127), s


def _write_plain(st: dict):
    slots, page = st["slots"], st["case"]["page"]
    q = _rotated_plain(st["q"], st).to(st["q"].dtype)
    live = slots >= 0
    # A place without a slot repeats the first that has one.
    at = torch.arange(slots.numel(), device=DEV)
    at = torch.where(live, at, live.to(torch.int32).argmax())
    to = slots[at]
    block, off = to // page, to % page
    got = []
    for x, codes, scales in ((_rotated_plain(st["k"], st), st["kc"], st["ks"]), (st["v"].float(), st["vc"], st["vs"])):
        c, s = _quantise_plain(x)
        codes[block, :, off] = c[at].to(torch.int8)
        scales[block, :, off] = s[at]
        back = codes[block, :, off].float() * scales[block, :, off][..., None]
        got.append(torch.where(live[:, None, None], back, 0.0).bfloat16())
    return (q, *got)


def _copy_plain(st: dict):
    frm, to, page = st["frm"].long(), st["to"].long(), st["case"]["page"]
    for x in (st["kc"], st["vc"], st["ks"], st["vs"]):
        new = x[frm]
        if st["tokens"] is not None:
            taken = (torch.arange(page, device=DEV) < st["tokens"][:, None])[:, None]
            new = torch.where(taken[..., None] if x.dim() == 4 else taken, new, x[to])
        x[to] = new
    return st["kc"], st["vc"], st["ks"], st["vs"]


def _values_plain(st: dict, pages: torch.Tensor, there: torch.Tensor):
    """k and v [.., H, L, D] of the pages [.., width], zeros where a token is not there [.., L]."""
    got = []
    for codes, scales in ((st["kc"], st["ks"]), (st["vc"], st["vs"])):
        x = codes[pages].float() * scales[pages][..., None]  # [.., pages, H, page, D]
        x = x.transpose(-4, -3).flatten(-3, -2)
        got.append(torch.where(there[..., None, :, None], x, 0.0))
    return got


def _shared_plain(st: dict):
    c, q = st["case"], st["q"]
    H, D, n_q, B, page = c["Hkv"], c["D"], c["max_q"], c["B"], c["page"]
    G, T = c["Hq"] // c["Hkv"], q.shape[0]
    starts, kv_len = st["starts"].long(), st["kv_len"].long()
    # Own tokens, as a padded batch.
    pages = st["table"].long().clamp(min=0)
    t = torch.arange(pages.shape[1] * page, device=DEV)
    k, v = _values_plain(st, pages, t < kv_len[:, None])
    i = torch.arange(n_q, device=DEV)
    rows = (starts[:-1, None] + i).clamp(max=T - 1)
    qp = q[rows].float().reshape(B, n_q, H, G, D).permute(0, 2, 3, 1, 4).reshape(B, H, G * n_q, D)
    s = torch.matmul(qp, k.transpose(2, 3).contiguous()) * st["scale"]
    pos = (kv_len - (starts[1:] - starts[:-1]))[:, None] + i  # [B, n_q]
    seen = (t < kv_len[:, None])[:, None, :] & (t <= pos[..., None])
    s = s.reshape(B, H, G, n_q, -1).masked_fill(~seen[:, None, None], -math.inf).flatten(2, 3)
    at = torch.arange(T, device=DEV)
    b = torch.searchsorted(starts, at, right=True) - 1

    def by_rows(x):  # [B, H, G n_q, n] to [H, G, T, n]
        x = x.reshape(B, H, G, n_q, -1)
        return x[b, :, :, at - starts[b]].permute(1, 2, 0, 3)

    m = s.amax(dim=-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    m, l, o = by_rows(m), by_rows(p.sum(dim=-1, keepdim=True)), by_rows(torch.matmul(p, v))
    out = torch.empty((H, G, T, D), device=DEV)
    # Each group's prefix under all its rows, joined with their own part.
    row = 0
    groups, free = _members(c)
    for g, (prefix, members) in enumerate(groups):
        n = sum(new for new, _ in members)
        pages = st["prefix_table"][g].long().clamp(min=0)
        t = torch.arange(pages.shape[0] * page, device=DEV)
        there = t < st["prefix_len"][g]
        k, v = _values_plain(st, pages, there)
        qg = q[row:row + n].float().reshape(n, H, G, D).permute(1, 2, 0, 3).reshape(H, G * n, D)
        s = torch.matmul(qg, k.transpose(1, 2).contiguous()) * st["scale"]
        s = s.masked_fill(~there, -math.inf)
        mine = m[:, :, row:row + n].reshape(H, G * n, 1)
        top = torch.maximum(s.amax(dim=-1, keepdim=True), mine)
        safe = torch.where(top == -math.inf, 0.0, top)
        p, keep = torch.exp(s - safe), torch.exp(mine - safe)
        total = p.sum(dim=-1, keepdim=True) + keep * l[:, :, row:row + n].reshape(H, G * n, 1)
        y = torch.matmul(p, v) + keep * o[:, :, row:row + n].reshape(H, G * n, D)
        out[:, :, row:row + n] = (y / torch.where(total > 0, total, 1.0)).reshape(H, G, n, D)
        row += n
    out[:, :, row:] = o[:, :, row:] / torch.where(l[:, :, row:] > 0, l[:, :, row:], 1.0)
    return out.permute(2, 0, 1, 3).reshape(T, c["Hq"], D).to(q.dtype)


def _lora_plain(st: dict):
    x, adapter = st["x"].float(), st["adapter"]
    y = st["base"].float()
    for a in range(st["case"]["adapters"]):
        h = torch.matmul(x, st["A"][a].float().t())
        h = torch.where((adapter == a)[:, None], h * st["scale"][a], 0.0)
        y = y + torch.matmul(h, st["B"][a].float().t())
    return y.to(st["base"].dtype)


_OWN = dict(rotary=_rotary_own, write=_write_own, copy=_copy_own, shared=_shared_own, lora=_lora_own)
_PLAIN = dict(rotary=_rotary_plain, write=_write_plain, copy=_copy_plain, shared=_shared_plain, lora=_lora_plain)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case: dict) -> dict:
    c = case
    if c["kind"] == "rotary":
        n = c["T"] * c["H"] * c["D"]
        return dict(bytes=2 * n * BYTES[c["x"]] + 8 * c["T"] + 4 * c["rot"], flops=3.0 * c["T"] * c["H"] * c["rot"])
    if c["kind"] == "write":
        e, n = BYTES[c["x"]], c["T"] * c["H"]  # q in and out; k, v in, codes out and in again, values out
        return dict(bytes=2 * c["T"] * c["Hq"] * c["D"] * e + 2 * n * (c["D"] * (e + 4) + 8) + 24 * c["T"],
                    flops=3.0 * c["T"] * (c["Hq"] + c["H"]) * c["rot"] + 12.0 * n * c["D"])
    if c["kind"] == "copy":
        tokens = c["n"] * (c["page"] + 1) / 2 if c["part"] else c["n"] * c["page"]
        return dict(bytes=int(2 * tokens * c["H"] * (2 * c["D"] + 8)) + 8 * c["n"], flops=0.0)
    if c["kind"] == "lora":
        used = min(c["adapters"], c["T"])
        return dict(bytes=c["T"] * (c["K"] * BYTES[c["x"]] + 2 * c["N"] * BYTES[c["out"]])
                    + used * c["R"] * (c["K"] + c["N"]) * BYTES[c["w"]], flops=2.0 * c["T"] * c["R"] * (c["K"] + c["N"]))
    groups, free = _members(c)
    tokens = pairs = rows = 0
    for prefix, members in groups:
        tokens += prefix
        for new, kv in members:
            tokens += kv
            pairs += new * prefix + sum(range(kv - new + 1, kv + 1))
            rows += new
    rows += len(free)
    return dict(bytes=tokens * c["Hkv"] * (2 * c["D"] + 8) + 2 * rows * c["Hq"] * c["D"] * BYTES[c["q"]],
                flops=4.0 * pairs * c["Hq"] * c["D"])


# ------------------------------------------------------------------ the same in 64 bits
def _turned(x: torch.Tensor, st: dict) -> torch.Tensor:
    rot = st["case"]["rot"]
    x = x.double()
    part, rest = x[..., :rot], x[..., rot:]
    if st["case"]["inter"]:
        pairs = part.unflatten(-1, (rot // 2, 2))
    else:
        pairs = part.unflatten(-1, (2, rot // 2)).transpose(-1, -2)
    turn = torch.polar(torch.full_like(st["freq"], st["factor"]).expand(x.shape[0], -1).contiguous(),
                       torch.outer(st["pos"].double(), st["freq"]))
    pairs = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn[:, None])
    part = pairs.flatten(-2) if st["case"]["inter"] else pairs.transpose(-1, -2).flatten(-2)
    return torch.cat([part, rest], dim=-1)


def _quantised_values(y: torch.Tensor):
    top = y.abs().max(dim=-1).values
    s = torch.where(top > 1e-30, top / 127, torch.ones_like(top))
    d = y / s.unsqueeze(-1)
    return torch.copysign(torch.floor(d.abs() + 0.5), d) * s.unsqueeze(-1)


def exact(case: dict, seed: int):
    c, st = case, prepare(case, seed)
    if c["kind"] == "rotary":
        return _turned(st["x"], st)
    if c["kind"] == "write":
        got = [_quantised_values(x) for x in (_turned(st["k"], st), st["v"].double())]
        for x in got:
            x[st["slots"] < 0] = 0
        return (_turned(st["q"], st), *got)
    if c["kind"] == "copy":
        # Token by token: where each comes from.
        at = torch.arange(c["blocks"], device=DEV).repeat_interleave(c["page"]).view(c["blocks"], c["page"])
        frm = at.clone()
        part = st["tokens"] if st["tokens"] is not None else torch.full_like(st["to"], c["page"])
        taken = torch.arange(c["page"], device=DEV) < part.unsqueeze(1)
        frm[st["to"].long()] = torch.where(taken, st["frm"].long().unsqueeze(1), st["to"].long().unsqueeze(1))
        place = torch.arange(c["page"], device=DEV).expand_as(frm)
        return tuple(x.transpose(1, 2)[frm, place].transpose(1, 2) for x in (st["kc"], st["vc"], st["ks"], st["vs"]))
    if c["kind"] == "lora":
        y = st["base"].double()
        for a in range(c["adapters"]):
            mine = torch.nonzero(st["adapter"] == a).flatten()
            if mine.numel():
                low = torch.einsum("tk,rk->tr", st["x"][mine].double(), st["A"][a].double())
                y[mine] += torch.einsum("tr,nr->tn", low, st["B"][a].double()) * st["scale"][a].double()
        return y
    H, G, D, page = c["Hkv"], c["Hq"] // c["Hkv"], c["D"], c["page"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)

    def tokens_of(ids, n, g):
        return [(st[x][ids, g].double() * st[s][ids, g].double().unsqueeze(-1)).reshape(-1, D)[:n]
                for x, s in (("kc", "ks"), ("vc", "vs"))]

    for g in range(H):
        row = seq = 0
        for number, (prefix, members) in enumerate(_members(c)[0]):
            pk, pv = tokens_of(st["prefix_table"][number, :-(-prefix // page)].long(), prefix, g)
            first, parts = row, []
            for new, kv in members:
                k, v = tokens_of(st["table"][seq, :-(-kv // page)].long(), kv, g)
                qs = st["q"][row:row + new, g * G:(g + 1) * G].double()
                logits = (qs.reshape(new * G, D) @ k.t()).view(new, G, kv) * st["scale"]
                later = torch.arange(kv, device=DEV) > torch.arange(kv - new, kv, device=DEV).view(new, 1, 1)
                parts.append((logits.masked_fill(later, -math.inf), v, row, new))
                row, seq = row + new, seq + 1
            for i in range(first, row, 128):
                j = min(row, i + 128)
                qs = st["q"][i:j, g * G:(g + 1) * G].double().reshape(-1, D)
                logits = (qs @ pk.t()) * st["scale"]
                top = logits.max(dim=1, keepdim=True).values
                p = torch.exp(logits - top)
                sums, values = p.sum(dim=1, keepdim=True), p @ pv
                top, sums, values = (x.view(j - i, G, -1) for x in (top, sums, values))
                for own_logits, v, at, new in parts:
                    a, z = max(i, at), min(j, at + new)
                    if a >= z:
                        continue
                    mine = own_logits[a - at:z - at]
                    t0 = top[a - i:z - i]
                    t1 = torch.maximum(t0, mine.max(dim=-1, keepdim=True).values)
                    e, keep = torch.exp(mine - t1), torch.exp(t0 - t1)
                    total = e.sum(dim=-1, keepdim=True) + keep * sums[a - i:z - i]
                    y = torch.matmul(e.reshape(-1, e.shape[-1]), v).view(z - a, G, D) + keep * values[a - i:z - i]
                    out[a:z, g * G:(g + 1) * G] = y / total
    return out
