"""The example's decoder layer, prompts and then single tokens, against the
same layer in 64 bits with nothing but the weights quantised; and a captured
step against the eager one.

Bar: E4M3 keeps 4 significant bits (relative step 2^-4 at most, 2.6e-2 rms),
and five roundings to it lie in a row on the way to y - the norm's output, K
and V, attention's output, the norm's output, GELU's - each of which spreads
its rms error over the sums behind it: sqrt(5) 2.6e-2 = 5.8e-2; the bar is
1e-1.  h has three of them behind products of half its size: 5e-2."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
pytestmark = pytest.mark.gpu


def rel(a, b):
    return ((a.double() - b).norm() / b.norm()).item()


@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (4, 4, 80), (2, 1, 128)])
def test_prompts_then_single_tokens(dev, heads, kv_heads, dim):
    from decoder_layer import Cache, DecoderLayer
    hidden, lengths, steps = 512, [37, 1, 90], 4
    layer = DecoderLayer(hidden, heads, kv_heads, dim, 1024, dev, seed=heads)
    cache = Cache(len(lengths), 7, kv_heads, 16, dim, dev)
    g = torch.Generator(device=dev).manual_seed(3)
    history = [None] * len(lengths)
    for step in range(steps):
        n = lengths if step == 0 else [1] * len(lengths)
        x = torch.randn(sum(n), hidden, device=dev, generator=g)
        add = torch.randn(sum(n), hidden, device=dev, generator=g).bfloat16()
        cu = torch.tensor([0] + n, device=dev).cumsum(0).int()
        cache.kv_len.add_(torch.tensor(n, device=dev).int())
        h, y = layer(x, add, cache, cu, max(n))
        hp, yp = layer.plain(x, add, n, history)
        torch.cuda.synchronize()
        assert rel(h, hp) < 5e-2 and rel(y, yp) < 1e-1, (step, rel(h, hp), rel(y, yp))


def test_captured_step_equals_the_eager_one(dev):
    from decoder_layer import Cache, DecoderLayer
    hidden, seqs = 512, 3
    layer = DecoderLayer(hidden, 8, 2, 64, 1024, dev)
    caches = [Cache(seqs, 4, 2, 16, 64, dev) for _ in range(2)]
    one = torch.arange(seqs + 1, dtype=torch.int32, device=dev)
    x, add = torch.zeros(seqs, hidden, device=dev), torch.zeros(seqs, hidden, device=dev, dtype=torch.bfloat16)

    def step(c):
        c.kv_len.add_(1)
        return layer(x, add, c, one, 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for c in caches:
            step(c)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(caches[0])
    g = torch.Generator(device=dev).manual_seed(5)
    for _ in range(20):  # across a page's end
        x.normal_(generator=g)
        add.normal_(generator=g)
        want = step(caches[1])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
