"""The attention half of a decoder layer, as the example runs it, against the same
mathematics on the unquantised weights in 64 bits."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

WIDTH, HEADS, KV_HEADS, DIM, PAGE = 512, 8, 2, 64, 16


@pytest.fixture(scope="module")
def example():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    path = os.path.join(os.path.dirname(__file__), "..", "phi-agent_amd", "examples", "decoder_attention.py")
    spec = importlib.util.spec_from_file_location("decoder_attention", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def plain(layer, h):
    """The layer on one whole sequence h [tokens, width], in 64 bits: the new h, its next norm."""
    norm = lambda x, w: x / (x.square().mean(1, keepdim=True) + layer.eps).sqrt() * w.double().cpu()  # noqa: E731
    w_qkv, w_out = (w.double().cpu() for w in layer.dense)
    T = h.shape[0]
    q, k, v = (norm(h, layer.norm) @ w_qkv.T).view(T, HEADS + 2 * KV_HEADS, DIM).split([HEADS, KV_HEADS, KV_HEADS], dim=1)
    o = torch.empty((T, HEADS, DIM), dtype=torch.float64)
    mask = torch.ones((T, T), dtype=torch.bool).triu(1)
    for i in range(HEADS):
        g = i // (HEADS // KV_HEADS)
        o[:, i] = torch.softmax((q[:, i] @ k[:, g].T * DIM ** -0.5).masked_fill(mask, -torch.inf), dim=1) @ v[:, g]
    h = h + o.reshape(T, -1) @ w_out.T
    return h, norm(h, layer.next_norm)


def test_mixed_steps_make_the_layer(example):
    """Two prompts in chunks of different sizes, a third sequence of single tokens, and
    pages used again after a sequence ended.

    An int8 step is amax / 127, its error uniform: 5 / (127 sqrt 12) = 1.1 % of a row
    whose largest element is 5 of its root mean square.  Five quantisers lie on the
    way to the update (both linears' operands and weights, the cache, which softmax
    and values see): 3 % in the root mean square, so 6 % is allowed."""
    layer = example.DecoderAttention(WIDTH, HEADS, KV_HEADS, DIM, blocks=40, page=PAGE, seed=3)
    g = torch.Generator().manual_seed(5)
    length = {"a": 300, "b": 77, "c": 5, "d": 200}
    x = {s: torch.randn((n, WIDTH), generator=g) for s, n in length.items()}
    at, got, nxt = dict.fromkeys(x, 0), {s: [] for s in x}, {s: [] for s in x}

    def step(*new):
        h = torch.cat([x[s][at[s]:at[s] + n] for s, n in new]).cuda()
        codes, scales = layer.step(h, list(new))
        row = 0
        for s, n in new:
            got[s].append(h[row:row + n].cpu()), nxt[s].append((codes[row:row + n].cpu(), scales[row:row + n].cpu()))
            at[s], row = at[s] + n, row + n

    step(("a", 128), ("c", 1))
    step(("c", 1), ("a", 150), ("b", 70))
    for _ in range(3):
        step(("a", 1), ("b", 1), ("c", 1))
    step(("b", 4), ("a", 19))
    layer.pages.end("a")
    step(("d", 200))
    assert len(layer.pages.free) + sum(len(p) for p in layer.pages.of.values()) == 40
    for s in x:
        want, want_norm = plain(layer, x[s].double())
        update, wanted = torch.cat(got[s]).double() - x[s].double(), want - x[s].double()
        assert float((update - wanted).norm() / wanted.norm()) < 0.06, s
        # The next operand: its row norms are those of the norm (the rotation keeps them).
        codes, scales = (torch.cat([p[i] for p in nxt[s]]).double() for i in (0, 1))
        ratio = (codes * scales[:, None]).norm(dim=1) / want_norm.norm(dim=1)
        assert float((ratio - 1).abs().max()) < 0.06, s
