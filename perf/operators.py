"""The operators between a decoder layer's int8 linears, as cases that can be timed.

A served layer normalises its residual stream into the linear's int8 operand,
writes the new tokens' keys and values into an int8 paged cache, and attends
over that cache; the linears themselves are in ``perf/cases.py``.  Sizes are
the repository's own (4352 and 32760 tokens, hidden 5120, prompts of 77) or
generic ones around them; ``draw`` spreads over the ranges that the listed
cases stand for.

The kinds:

  norm       residual addition, root-mean-square norm, (rotation,) int8 codes
             with one scale a token; the codes come back as the values they
             stand for, in bf16
  cache      new tokens' keys and values quantised into the paged cache, and
             the same slots read back
  attention  a batch of new tokens (one each, or chunks of prompts) over the
             paged int8 cache

``run`` computes a case with elementary torch operations in 32 bits where
``own`` is false, and calls this repository's operators where it is true.
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
EPS = 1e-6


def _package():
    pkg = os.path.join(os.getcwd(), "phi-agent_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import phi_qlinear

    return phi_qlinear


def listed() -> list[dict]:
    return [
        # One sequence's new token before a projection: launches are all there is.
        dict(name="norm_token", kind="norm", rows=1, K=4096, x="bf16", res="bf16", shift=False, rotate=True),
        # An image's or a prompt's tokens, an fp32 residual stream as the transformer keeps it.
        dict(name="norm_prompt", kind="norm", rows=4352, K=5120, x="bf16", res="f32", shift=False, rotate=True),
        # A width that is no whole number of anything, with an adaLN shift: rows that start at odd addresses.
        dict(name="norm_odd", kind="norm", rows=777, K=5003, x="f32", res="f32", shift=True, rotate=False),
        # A decode step of 64 sequences (a quarter of the batch's places empty).
        dict(name="cache_step", kind="cache", T=64, H=8, D=128, page=16, x="bf16", step=True),
        # A long prompt written page by page.
        dict(name="cache_prompt", kind="cache", T=32760, H=8, D=128, page=64, x="bf16", step=False),
        # One sequence's next token: the smallest attention there is.
        dict(name="decode_one", kind="attention", B=1, Hq=32, Hkv=8, D=128, page=16, max_q=1, max_kv=777, q="bf16",
             window=0),
        # A full batch of sequences of very different lengths, one new token each.
        dict(name="decode_batch", kind="attention", B=64, Hq=32, Hkv=8, D=128, page=16, max_q=1, max_kv=8192, q="bf16",
             window=0),
        # Two long contexts: few rows, a long axis.
        dict(name="decode_long", kind="attention", B=2, Hq=32, Hkv=8, D=128, page=64, max_q=1, max_kv=131071, q="bf16",
             window=0),
        # A scheduler's mixed batch: some sequences' prompts in chunks, others' few tokens.
        dict(name="chunks_mixed", kind="attention", B=12, Hq=40, Hkv=8, D=128, page=32, max_q=512, max_kv=4352, q="bf16",
             window=0),
        # A long prompt's next chunk: the largest call.
        dict(name="prefill", kind="attention", B=1, Hq=32, Hkv=8, D=128, page=64, max_q=4096, max_kv=16384, q="bf16",
             window=0),
        # Every head with keys of its own, a narrow head, a sliding window, pages of an odd size, and one
        # sequence without a token in the cache.
        dict(name="window_odd", kind="attention", B=5, Hq=20, Hkv=20, D=80, page=24, max_q=77, max_kv=3001, q="bf16",
             window=1000),
        # Activations in 32 bits, as the reference keeps them: a prompt of the text encoder.
        dict(name="prompt_f32", kind="attention", B=4, Hq=16, Hkv=4, D=128, page=16, max_q=256, max_kv=1111, q="f32",
             window=0),
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["norm", "cache", "attention", "attention", "attention"])
    x = rng.choice(["bf16", "bf16", "f32"])
    if kind == "norm":
        rotate = rng.random() < 0.6
        K = 256 * _log(rng, 2, 32) if rotate else _log(rng, 384, 8192)
        return dict(kind=kind, rows=_log(rng, 1, max(1, 4352 * 5120 // K)), K=K, x=x,
                    res=rng.choice(["none", "bf16", "f32"]), shift=rng.random() < 0.4, rotate=rotate)
    H, D = rng.choice([1, 2, 3, 4, 8, 16]), rng.choice([64, 80, 96, 128, 128, 192, 256])
    page = rng.choice([8, 16, 16, 24, 32, 64, 128, 256])
    if kind == "cache":
        step = rng.random() < 0.4
        top = min(256 if step else 32760, 32760 * 8 * 128 // (H * D))
        return dict(kind=kind, T=_log(rng, 1, top), H=H, D=D, page=page, x=x, step=step)
    G = rng.choice([1, 2, 4, 4, 5, 7, 8, 8, 16])
    B = _log(rng, 1, 64)
    max_q = 1 if rng.random() < 0.45 else _log(rng, 2, 4096)
    kv_cost, qk_cost = 64 * 4096 * 8 * 128, 32 * 4096 * 14000 * 128  # the listed cases' largest
    while True:  # what the padded batch costs, at most: else fewer sequences, then a shorter chunk
        top = min(131071, kv_cost // (B * H * D), qk_cost // (B * H * G * max_q * max(D, 128)))
        if top >= max(max_q, 64) and B * max_q * H * G * D <= 8192 * 32 * 128:
            break
        B, max_q = (B // 2, max_q) if B > 1 else (1, max_q // 2)
    return dict(kind=kind, B=B, Hq=H * G, Hkv=H, D=D, page=page, max_q=max_q, max_kv=_log(rng, max(max_q, 8), top), q=x,
                window=_log(rng, 16, 4096) if rng.random() < 0.2 else 0)


def _lengths(c: dict) -> list[tuple[int, int]]:
    """(new tokens, tokens in the cache with them) of each sequence: part of the
    case.  The first is the longest; of five or more, the last has none in the
    cache (a place of the batch that is empty)."""
    rng = random.Random(1000003 * c["max_kv"] + 1009 * c["max_q"] + c["B"])
    got = [(c["max_q"], c["max_kv"])]
    for _ in range(c["B"] - 1):
        n = _log(rng, 1, c["max_q"])
        got.append((n, rng.randint(n, c["max_kv"])))
    if c["B"] >= 5:
        got[-1] = (1, 0)
    return got


# ------------------------------------------------------------------ inputs
def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(shape, seed: int, scale: float = 1.0, dtype=torch.float32) -> torch.Tensor:
    return (torch.randn(shape, generator=_gen(seed), device=DEV) * scale).to(dtype)


def _hadamard(dtype) -> torch.Tensor:
    """The linear's 256-wide rotation: (J - 2R)^(x4) / 16."""
    j = torch.ones((4, 4), dtype=torch.float64) - 2 * torch.eye(4, dtype=torch.float64).flip(0)
    h = torch.kron(torch.kron(j, j), torch.kron(j, j)) / 16
    return h.to(device=DEV, dtype=dtype)


def _codes(shape, seed: int) -> torch.Tensor:
    """int8 codes of normally distributed vectors (absmax near 127)."""
    got = torch.empty(shape, dtype=torch.int8, device=DEV)
    flat, g, step = got.view(-1), _gen(seed), 1 << 26
    for i in range(0, flat.numel(), step):
        n = min(step, flat.numel() - i)
        flat[i:i + n] = (torch.randn(n, generator=g, device=DEV) * 42).round_().clamp_(-127, 127).to(torch.int8)
    return got


def prepare(case: dict, seed: int) -> dict:
    s = seed * 16  # a stream of its own for every tensor
    st = dict(case=case)
    if case["kind"] == "norm":
        rows, K = case["rows"], case["K"]
        x = _randn((rows, K), s)
        x[:, ::997] *= 20  # a few outlier channels
        st.update(x=x.to(DTYPES[case["x"]]), w=1 + _randn((K,), s + 1, 0.1), h=None, shift=None)
        if case["res"] != "none":
            st["h"] = _randn((rows, K), s + 2, 3.0, DTYPES[case["res"]])
        if case["shift"]:
            st["shift"] = _randn((K,), s + 3, 0.1)
        if case["rotate"]:
            st["had"] = _hadamard(torch.float32)
        return st
    H, D, page = case.get("Hkv", case.get("H")), case["D"], case["page"]
    if case["kind"] == "cache":
        T = case["T"]
        # k and v are columns of the fused projection's output.
        qkv = _randn((T, 4 * H, D), s, 1.0, DTYPES[case["x"]])
        qkv[:, :, ::61] *= 6
        pages = T if case["step"] else -(-T // page)
        blocks = pages + 3
        order = torch.randperm(blocks, generator=_gen(s + 1), device=DEV)[:pages]
        if case["step"]:  # one token a sequence, each on a page of its own; every fourth place is empty
            slots = order * page + torch.randint(0, page, (T,), generator=_gen(s + 2), device=DEV)
            slots[3::4] = -1
        else:
            at = torch.arange(T, device=DEV)
            slots = order[at // page] * page + at % page
        st.update(k=qkv[:, 2 * H:3 * H], v=qkv[:, 3 * H:], slots=slots)
        kc, vc = (torch.zeros((blocks, H, page, D), dtype=torch.int8, device=DEV) for _ in range(2))
        ks, vs = (torch.ones((blocks, H, page), dtype=torch.float32, device=DEV) for _ in range(2))
        st.update(kc=kc, vc=vc, ks=ks, vs=vs)
        return st
    lens = _lengths(case)
    T, B = sum(n for n, _ in lens), case["B"]
    width = -(-case["max_kv"] // page)
    need = [-(-kv // page) for _, kv in lens]
    blocks = sum(need) + 1
    order = torch.randperm(blocks, generator=_gen(s + 1), device=DEV).tolist()
    table = torch.full((B, width), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
    starts = [0]
    for n, _ in lens:
        starts.append(starts[-1] + n)
    kc, vc = _codes((blocks, H, page, D), s + 2), _codes((blocks, H, page, D), s + 3)
    ks, vs = (torch.rand((blocks, H, page), generator=_gen(s + 4 + i), device=DEV) * 0.02 + 0.01 for i in range(2))
    for b, (_, kv) in enumerate(lens):  # what lies past a sequence's end in its last page was never written
        if kv % page:
            last = int(table[b, kv // page])
            ks[last, :, kv % page:] = math.nan
            vs[last, :, kv % page:] = math.nan
    # q is columns of the fused projection's output.
    qkv = _randn((T, case["Hq"] + 2 * H, D), s + 6, 1.5, DTYPES[case["q"]])
    st.update(q=qkv[:, :case["Hq"]], kc=kc, vc=vc, ks=ks, vs=vs, table=table.to(DEV), scale=D ** -0.5,
              starts=torch.tensor(starts, dtype=torch.int32, device=DEV),
              kv_len=torch.tensor([kv for _, kv in lens], dtype=torch.int32, device=DEV))
    return st


# ------------------------------------------------------------------ one pass
def run(st: dict):
    kind = st["case"]["kind"]
    if kind == "norm":
        return _norm_own(st) if own else _norm_plain(st)
    if kind == "cache":
        return _cache_own(st) if own else _cache_plain(st)
    return _attention_own(st) if own else _attention_plain(st)


def _norm_own(st: dict):
    Q, x, h = _package(), st["x"], st["h"]
    new = None if h is None else torch.empty_like(h)
    q, s = Q.rms_norm_quant(x, st["w"], EPS, residual=h, residual_out=new, shift=st["shift"],
                            rotate=st["case"]["rotate"])
    values = torch.empty(x.shape, dtype=torch.bfloat16, device=x.device)
    torch.mul(q, s[:, None], out=values)
    return (values, s) if h is None else (values, s, new)


def _cache_own(st: dict):
    Q = _package()
    cache = Q.KvCache(st["kc"], st["vc"], st["ks"], st["vs"])
    Q.kv_cache_write(cache, st["k"], st["v"], st["slots"])
    return Q.kv_cache_read(cache, st["slots"], out_dtype=st["k"].dtype)


def _attention_own(st: dict):
    Q, c = _package(), st["case"]
    cache = Q.KvCache(st["kc"], st["vc"], st["ks"], st["vs"])
    return Q.paged_attention(st["q"], cache, st["table"], st["starts"], st["kv_len"], max_q=c["max_q"],
                             max_kv=c["max_kv"], scale=st["scale"], window=c["window"])


def _quantise_plain(y: torch.Tensor):
    """Codes (as floats) and scale of the last axis, ties away from zero."""
    amax = y.abs().amax(dim=-1)
    s = torch.where(amax > 1e-30, amax / 127.0, torch.ones_like(amax))
    d = y * (1.0 / s)[..., None]
    return (torch.sign(d) * torch.floor(d.abs() + 0.5)).clamp(-127, 127), s


def _norm_plain(st: dict):
    x, h = st["x"], st["h"]
    r = x.float() if h is None else x.float() + h.float()
    y = r * torch.rsqrt((r * r).mean(dim=1, keepdim=True) + EPS) * st["w"]
    if st["shift"] is not None:
        y = y + st["shift"]
    if st["case"]["rotate"]:
        y = (y.reshape(-1, 256) @ st["had"]).reshape(y.shape)
    codes, s = _quantise_plain(y)
    values = (codes * s[:, None]).bfloat16()
    return (values, s) if h is None else (values, s, r.to(h.dtype))


def _cache_plain(st: dict):
    slots, page = st["slots"], st["case"]["page"]
    live = slots >= 0
    # A place without a slot repeats the first that has one.
    at = torch.arange(slots.numel(), device=DEV)
    at = torch.where(live, at, live.to(torch.int32).argmax())
    to = slots[at]
    block, off = to // page, to % page
    got = []
    for x, codes, scales in ((st["k"], st["kc"], st["ks"]), (st["v"], st["vc"], st["vs"])):
        c, s = _quantise_plain(x.float())
        codes[block, :, off] = c[at].to(torch.int8)
        scales[block, :, off] = s[at]
        back = codes[block, :, off].float() * scales[block, :, off][..., None]
        got.append(torch.where(live[:, None, None], back, 0.0).to(x.dtype))
    return tuple(got)


def _attention_plain(st: dict):
    c, q, starts, kv_len = st["case"], st["q"], st["starts"].long(), st["kv_len"].long()
    B, H, D, n_q = c["B"], c["Hkv"], c["D"], c["max_q"]
    G, T = c["Hq"] // c["Hkv"], q.shape[0]
    pages = st["table"].long().clamp(min=0)
    L = pages.shape[1] * c["page"]
    t = torch.arange(L, device=DEV)
    there = t < kv_len[:, None]  # [B, L]

    def values(codes, scales):
        x = codes[pages].float() * scales[pages][..., None]  # [B, pages, H, page, D]
        x = x.permute(0, 2, 1, 3, 4).reshape(B, H, L, D)
        return torch.where(there[:, None, :, None], x, 0.0)

    new = starts[1:] - starts[:-1]
    i = torch.arange(n_q, device=DEV)
    rows = (starts[:-1, None] + i).clamp(max=T - 1)
    qp = q[rows].float().reshape(B, n_q, H, G, D).permute(0, 2, 3, 1, 4).reshape(B, H, G * n_q, D)
    s = torch.matmul(qp, values(st["kc"], st["ks"]).transpose(2, 3).contiguous()) * st["scale"]
    pos = (kv_len - new)[:, None] + i  # [B, n_q]
    seen = there[:, None, :] & (t <= pos[..., None])
    if c["window"]:
        seen = seen & (t > pos[..., None] - c["window"])
    s = s.reshape(B, H, G, n_q, L).masked_fill(~seen[:, None, None], -math.inf)
    m = s.amax(dim=-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    total = p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p.reshape(B, H, G * n_q, L), values(st["vc"], st["vs"])).reshape(B, H, G, n_q, D)
    o = o / torch.where(total > 0, total, 1.0)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, n_q, c["Hq"], D)
    at = torch.arange(T, device=DEV)
    b = torch.searchsorted(starts, at, right=True) - 1
    return o[b, at - starts[b]].to(q.dtype)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case: dict) -> dict:
    if case["kind"] == "norm":
        n = case["rows"] * case["K"]
        res = 0 if case["res"] == "none" else 2 * BYTES[case["res"]]
        return dict(bytes=n * (BYTES[case["x"]] + res + 1) + 4 * case["rows"] + 4 * case["K"] * (1 + case["shift"]),
                    flops=n * (8.0 + (16.0 if case["rotate"] else 0.0)))
    if case["kind"] == "cache":
        n = 2 * case["T"] * case["H"]  # vectors: in, codes out and in again, values out
        return dict(bytes=n * case["D"] * (2 * BYTES[case["x"]] + 2) + 8 * n + 8 * case["T"], flops=6.0 * n * case["D"])
    H, D, w = case["Hkv"], case["D"], case["window"]
    tokens = pairs = rows = 0
    for n, kv in _lengths(case):
        first = kv - n
        if kv:
            tokens += kv - max(0, first + 1 - w) if w else kv
            pairs += sum(min(p + 1, w) if w else p + 1 for p in range(first, kv))
        rows += n
    return dict(bytes=tokens * H * (2 * D + 8) + 2 * rows * case["Hq"] * D * BYTES[case["q"]],
                flops=4.0 * pairs * case["Hq"] * D)


# ------------------------------------------------------------------ the same in 64 bits
def _quantised_values(y: torch.Tensor):
    top = y.abs().max(dim=-1).values
    s = torch.where(top > 1e-30, top / 127, torch.ones_like(top))
    d = y / s.unsqueeze(-1)
    code = torch.copysign(torch.floor(d.abs() + 0.5), d)
    return code * s.unsqueeze(-1), s


def exact(case: dict, seed: int):
    st = prepare(case, seed)
    if case["kind"] == "norm":
        r = st["x"].double()
        if st["h"] is not None:
            r = r + st["h"].double()
        y = st["w"].double() * r / torch.sqrt(r.pow(2).sum(dim=1, keepdim=True) / case["K"] + EPS)
        if st["shift"] is not None:
            y = y + st["shift"].double()
        if case["rotate"]:
            y = torch.einsum("rgi,ij->rgj", y.view(case["rows"], -1, 256), _hadamard(torch.float64)).reshape(y.shape)
        values, s = _quantised_values(y)
        return (values, s) if st["h"] is None else (values, s, r)
    if case["kind"] == "cache":
        got = [_quantised_values(st[x].double())[0] for x in ("k", "v")]
        for x in got:
            x[st["slots"] < 0] = 0
        return tuple(got)
    H, G, D, page = case["Hkv"], case["Hq"] // case["Hkv"], case["D"], case["page"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    row = 0
    for b, (n, kv) in enumerate(_lengths(case)):
        ids = st["table"][b, :-(-kv // page)].long()
        for g in range(H if kv else 0):
            k, v = ((st[c][ids, g].double() * st[s][ids, g].double().unsqueeze(-1)).reshape(-1, D)[:kv]
                    for c, s in (("kc", "ks"), ("vc", "vs")))
            for i in range(0, n, 512):
                m = min(512, n - i)
                qs = st["q"][row + i:row + i + m, g * G:(g + 1) * G].double()
                pos = torch.arange(kv - n + i, kv - n + i + m, device=DEV).view(m, 1, 1)
                t = torch.arange(kv, device=DEV)
                hide = t > pos
                if case["window"]:
                    hide = hide | (t <= pos - case["window"])
                logits = (qs.reshape(m * G, D) @ k.t()).view(m, G, kv) * st["scale"]
                p = torch.softmax(logits.masked_fill(hide, -math.inf), dim=-1)
                out[row + i:row + i + m, g * G:(g + 1) * G] = (p.view(m * G, kv) @ v).view(m, G, D)
        row += n
    return out
