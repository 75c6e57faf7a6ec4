"""The attention half of a decoder layer on the int8 linears and the int8 paged cache.

    h += W_o attention(W_qkv norm(h))          then norm(h) as the next linear's operand

for a batch that mixes prompts, taken in chunks, with sequences that add a token a
step.  Pages of the cache are handed out as sequences grow and taken back when they
end.  (The positions' rotation of q and k, which a model has between the projection
and the cache, is left out.)

    python phi-agent_amd/examples/decoder_attention.py [--prompt 2000] [--sequences 16] [--new 64] [--chunk 512]
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import phi_qlinear as Q  # noqa: E402


class Pages:
    """Who has which pages of a cache."""

    def __init__(self, blocks: int, page: int):
        self.page, self.free, self.of, self.length = page, list(range(blocks))[::-1], {}, {}

    def grow(self, seq, tokens: int) -> list[int]:
        """Room for `tokens` more of sequence seq: their slots."""
        at, mine = self.length.get(seq, 0), self.of.setdefault(seq, [])
        while len(mine) * self.page < at + tokens:
            if not self.free:
                raise RuntimeError("the cache is full")
            mine.append(self.free.pop())
        self.length[seq] = at + tokens
        return [mine[t // self.page] * self.page + t % self.page for t in range(at, at + tokens)]

    def end(self, seq) -> None:
        self.free += self.of.pop(seq, [])
        self.length.pop(seq, None)


class DecoderAttention:
    """norm -> q, k, v -> cache -> attention -> output projection -> residual and next norm."""

    def __init__(self, width: int, heads: int, kv_heads: int, dim: int, *, blocks: int, page: int, device="cuda", eps=1e-6, seed=0):
        g = torch.Generator(device=device).manual_seed(seed)
        rand = lambda *s: torch.randn(s, generator=g, device=device)  # noqa: E731
        self.heads, self.kv_heads, self.dim, self.eps = heads, kv_heads, dim, eps
        self.norm, self.next_norm = 1 + 0.1 * rand(width), 1 + 0.1 * rand(width)
        self.dense = rand((heads + 2 * kv_heads) * dim, width) * width ** -0.5, rand(width, heads * dim) * (heads * dim) ** -0.5
        self.qkv, self.out = (Q.quant_rotate(w) for w in self.dense)  # (codes, a scale a row)
        self.cache = Q.kv_cache_empty(blocks, page, kv_heads, dim, device)
        self.pages = Pages(blocks, page)

    def step(self, h: torch.Tensor, new: list) -> tuple[torch.Tensor, torch.Tensor]:
        """h [tokens, width] fp32, updated in place: the new tokens of the sequences in
        `new`, [(sequence, tokens)], one after the other.  Returns the next norm's
        (codes, scales)."""
        dev, T = h.device, h.shape[0]
        slots, starts, lens = [], [0], []
        for seq, n in new:
            slots += self.pages.grow(seq, n)
            starts.append(starts[-1] + n)
            lens.append(self.pages.length[seq])
        assert starts[-1] == T
        width = max(len(self.pages.of[seq]) for seq, _ in new)
        table = torch.tensor([self.pages.of[seq] + [-1] * (width - len(self.pages.of[seq])) for seq, _ in new], dtype=torch.int32)
        table, starts_, lens_ = (torch.as_tensor(x, dtype=torch.int32).to(dev) for x in (table, starts, lens))
        slots = torch.tensor(slots, dtype=torch.int64).to(dev)

        a, sa = Q.rms_norm_quant(h, self.norm, self.eps)
        qkv = Q.i8_gemm(a, self.qkv[0], sa, self.qkv[1]).view(T, self.heads + 2 * self.kv_heads, self.dim)
        q, k, v = qkv.split([self.heads, self.kv_heads, self.kv_heads], dim=1)
        Q.kv_cache_write(self.cache, k, v, slots)
        o = Q.paged_attention(q, self.cache, table, starts_, lens_, max_q=max(n for _, n in new), max_kv=max(lens))
        y = Q.q8_linear(o.view(T, self.heads * self.dim), *self.out)
        return Q.rms_norm_quant(y, self.next_norm, self.eps, residual=h, residual_out=h)


def main():
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, default in (("prompt", 2000), ("sequences", 16), ("new", 64), ("chunk", 512)):
        p.add_argument("--" + name, type=int, default=default)
    o = p.parse_args()
    page, width = 16, 4096
    layer = DecoderAttention(width, 32, 8, 128, blocks=o.sequences * -(-(o.prompt + o.new) // page), page=page)
    g = torch.Generator(device="cuda").manual_seed(1)
    todo = {s: o.prompt for s in range(o.sequences)}  # prompt tokens that are left
    made = dict.fromkeys(todo, 0)
    steps = tokens = 0
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    while made:
        room, new = o.chunk, []
        for s in list(made):  # every running sequence's token, then prompts as far as the chunk goes
            n = min(todo[s], room) if todo[s] else 1
            if n:
                new.append((s, n))
                room -= n if todo[s] else 0
                if todo[s]:
                    todo[s] -= n
                else:
                    made[s] += 1
        layer.step(torch.randn((sum(n for _, n in new), width), generator=g, device="cuda"), new)
        steps, tokens = steps + 1, tokens + sum(n for _, n in new)
        for s in [s for s in made if made[s] == o.new]:
            layer.pages.end(s)
            del made[s]
    torch.cuda.synchronize()
    t = time.perf_counter() - t0
    print(f"{o.sequences} sequences, {o.prompt} + {o.new} tokens: {steps} steps, {tokens} tokens in {t * 1e3:.1f} ms, {t / steps * 1e6:.0f} us a step")


if __name__ == "__main__":
    main()
