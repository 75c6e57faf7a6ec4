"""The attention half of a decoder layer for many requests behind shared documents.

    h += W_o attention(rotary(W_qkv norm(h)))     then norm(h) as the next linear's operand

on the int8 linears and the int8 paged cache, as decoder_attention.py, with what a server of
many requests has beside it: positions, each request's own low-rank adapter on both
linears, and requests that begin as forks of a document, whose pages they share and attention
reads for many of them at a time.

    python phi-agent_amd/examples/shared_serving.py [--document 8192] [--requests 64] [--new 64] [--chunk 1024]
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import phi_qlinear as Q  # noqa: E402


class SharedServing:
    """norm -> q, k, v + adapters -> rotary and cache -> attention over prefixes and own
    tokens -> output projection + adapters -> residual and next norm."""

    def __init__(self, width: int, heads: int, kv_heads: int, dim: int, *, blocks: int, page: int, adapters: int, rank: int,
                 rot: int | None = None, device="cuda", eps=1e-6, seed=0):
        g = torch.Generator(device=device).manual_seed(seed)
        rand = lambda *s: torch.randn(s, generator=g, device=device)  # noqa: E731
        self.heads, self.kv_heads, self.dim, self.eps = heads, kv_heads, dim, eps
        self.norm, self.next_norm = 1 + 0.1 * rand(width), 1 + 0.1 * rand(width)
        sizes = ((heads + 2 * kv_heads) * dim, width), (width, heads * dim)
        self.dense = [rand(n, k) * k ** -0.5 for n, k in sizes]
        self.qkv, self.out = (Q.quant_rotate(w) for w in self.dense)  # (codes, a scale a row)
        # Adapter a of a linear: scale[a] B[a] A[a].
        self.factors = [((rand(adapters, rank, k) * k ** -0.5).bfloat16(), rand(adapters, n, rank).bfloat16()) for n, k in sizes]
        self.scale = torch.rand(adapters, generator=g, device=device) * rank ** -0.5
        self.freq = Q.rotary_frequencies(rot or dim, device=device)
        self.cache = Q.kv_cache_empty(blocks, page, kv_heads, dim, device)
        self.pages = Q.KvPages(blocks, page)
        self.adapter, self.document = {}, {}

    def begin(self, seq, adapter: int = -1, document=None) -> None:
        """A sequence with an adapter (-1: none), empty or behind another's tokens, which
        are those of the adapter that made them."""
        if document is not None:
            self.pages.fork(document, seq)
        self.adapter[seq], self.document[seq] = adapter, document

    def end(self, seq) -> None:
        self.pages.end(seq)
        del self.adapter[seq], self.document[seq]

    def groups(self, new: list) -> list:
        """[(first, last + 1, shared pages)] of neighbours in `new` that came from one document."""
        cuts, found = [i for i in range(1, len(new)) if self.document[new[i][0]] is None
                       or self.document[new[i][0]] != self.document[new[i - 1][0]]], []
        for a, b in zip([0] + cuts, cuts + [len(new)]):
            found.append((a, b, self.pages.shared([s for s, _ in new[a:b]]) if b - a > 1 else 0))
        return found

    def step(self, h: torch.Tensor, new: list) -> tuple[torch.Tensor, torch.Tensor]:
        """h [tokens, width] fp32, updated in place: the new tokens of the sequences in
        `new`, [(sequence, tokens)], one after the other.  Returns the next norm's
        (codes, scales)."""
        dev, T, page, pages = h.device, h.shape[0], self.pages.page, self.pages
        slots, starts, positions, adapter = [], [0], [], []
        for seq, n in new:
            at = pages.length.get(seq, 0)
            slots += pages.grow(seq, n)
            positions += range(at, at + n)
            adapter += [self.adapter[seq]] * n
            starts.append(starts[-1] + n)
        assert starts[-1] == T
        groups = self.groups(new)
        prefix = [pages.of[new[a][0]][:m] for a, _, m in groups]
        own = [pages.of[s][m:] for a, b, m in groups for s, _ in new[a:b]]
        lens = [pages.length[s] - m * page for a, b, m in groups for s, _ in new[a:b]]

        def table(rows):
            width = max(map(len, rows + [[0]]))
            return torch.tensor([r + [-1] * (width - len(r)) for r in rows], dtype=torch.int32).to(dev)

        prefix_, own_ = table(prefix), table(own)
        ints = [[len(p) * page for p in prefix], [a for a, _, _ in groups] + [len(new)], starts, lens]
        prefix_len, group_start, starts_, lens_ = (torch.tensor(x, dtype=torch.int32).to(dev) for x in ints)
        slots, positions = (torch.tensor(x, dtype=torch.int64).to(dev) for x in (slots, positions))
        adapter = torch.tensor(adapter, dtype=torch.int32).to(dev)
        pages.flush(self.cache)

        y = torch.empty((T, h.shape[1]), dtype=torch.bfloat16, device=dev)
        a, sa = Q.rms_norm_quant(h, self.norm, self.eps, y=y)
        qkv = Q.i8_gemm(a, self.qkv[0], sa, self.qkv[1])
        Q.lora_batched(y, *self.factors[0], adapter, scale=self.scale, base=qkv, out=qkv)
        q, k, v = qkv.view(T, self.heads + 2 * self.kv_heads, self.dim).split([self.heads, self.kv_heads, self.kv_heads], dim=1)
        Q.rotary_cache_write(self.cache, q, k, v, positions, self.freq, slots, out=q)
        o = Q.paged_attention_shared(q, self.cache, prefix_, prefix_len, group_start, own_, starts_, lens_, max_prefix=max(ints[0]),
                                     max_q=max(n for _, n in new), max_kv=max(lens)).view(T, self.heads * self.dim)
        z = Q.q8_linear(o, *self.out)
        Q.lora_batched(o, *self.factors[1], adapter, scale=self.scale, base=z, out=z)
        return Q.rms_norm_quant(z, self.next_norm, self.eps, residual=h, residual_out=h)


def main():
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, default in (("document", 8192), ("requests", 64), ("new", 64), ("chunk", 1024)):
        p.add_argument("--" + name, type=int, default=default)
    o = p.parse_args()
    page, width, dev = 16, 4096, "cuda"
    layer = SharedServing(width, 32, 8, 128, blocks=-(-o.document // page) + o.requests * (-(-o.new // page) + 2), page=page,
                          adapters=8, rank=16)
    g = torch.Generator(device=dev).manual_seed(1)
    layer.begin("document")
    for at in range(0, o.document, o.chunk):
        n = min(o.chunk, o.document - at)
        layer.step(torch.randn((n, width), generator=g, device=dev), [("document", n)])
    for r in range(o.requests):
        layer.begin(r, r % 9 - 1, "document")
    h = torch.randn((o.requests, width), generator=g, device=dev)
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    for _ in range(o.new):
        layer.step(h.clone(), [(r, 1) for r in range(o.requests)])
    torch.cuda.synchronize()
    t = time.perf_counter() - t0
    print(f"{o.requests} requests behind {o.document} tokens, {o.new} steps: {t / o.new * 1e6:.0f} us a step; "
          f"{len(layer.pages.users) - len(layer.pages.free)} pages in use")


if __name__ == "__main__":
    main()
