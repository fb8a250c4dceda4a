"""The example's decode loop - plan, norm, rotation, cache write, attention
behind a shared prompt or with sinks - against the same layer in 64 bits with
nothing but the weights quantised, while requests start, grow and end; and a
captured step against the eager one.

Bar: as for the layer without positions (test_gpu_decoder_layer): five roundings
to E4M3 in a row on the way to y, three behind products of half its size on the
way to h; the norms and the rotation of queries and keys round in bf16, 2^-9,
which is nothing beside them."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
pytestmark = pytest.mark.gpu


def rel(a, b):
    return ((a.double() - b).norm() / b.norm()).item()


def setup(dev, prefix, window=0, sinks=0, slots=4, heads=8, kv_heads=2, dim=64, pages=60, rows=200):
    from decode_loop import Requests, RotaryLayer
    layer = RotaryLayer(512, heads, kv_heads, dim, 1024, dev, 400, window, sinks, seed=heads)
    return layer, Requests(slots, prefix, 400, pages, kv_heads, 16, dim, rows, dev)


@pytest.mark.parametrize("prefix,window,sinks", [(96, 0, 0), (0, 0, 0), (0, 30, 3), (16, 0, 0)])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (4, 4, 80), (2, 1, 128)])
def test_requests_come_and_go(dev, prefix, window, sinks, heads, kv_heads, dim):
    layer, batch = setup(dev, prefix, window, sinks, 4, heads, kv_heads, dim)
    pages = len(batch.free_pages)
    g = torch.Generator(device=dev).manual_seed(3)
    none = torch.zeros(0, kv_heads, dim, dtype=torch.float64, device=dev)
    history, length = {b: (none, none) for b in range(5)}, dict.fromkeys(range(5), 0)

    def bring(n, pad=0):
        """{slot: tokens} through both, on a batch padded by `pad` rows."""
        rows = sum(n.values())
        x = torch.randn(rows + pad, 512, device=dev, generator=g)
        add = torch.randn(rows + pad, 512, device=dev, generator=g).bfloat16()
        order = sorted(n)
        batch.brings(n)
        batch.plan(rows + pad)
        h, y = layer(x, add, batch, max(n.values()))
        hp, yp = layer.plain(x, add, order, [(n[b], length[b]) for b in order], history)
        torch.cuda.synchronize()
        for b in order:
            length[b] += n[b]
        assert batch.kv_len.tolist() == [length[b] for b in range(5)]
        assert rel(h[:rows], hp) < 5e-2 and rel(y[:rows], yp) < 1e-1, (rel(h[:rows], hp), rel(y[:rows], yp))

    def start(slots):
        batch.start(slots)
        for b in slots:
            history[b], length[b] = history[4], length[4]
    if prefix:
        bring({4: prefix})
    start([0, 1, 3])
    bring({0: 37, 1: 1, 3: 90})
    for _ in range(3):
        bring({0: 1, 1: 1, 3: 1}, pad=5)
    batch.end([1, 3])
    for b in (1, 3):
        length[b], history[b] = 0, (none, none)
    used = sum(-(-length[b] // 16) for b in (0, 4)) - (prefix // 16 if length[0] else 0)
    assert batch.left.item() == pages - used
    start([2, 3])
    bring({2: 20, 3: 5, 0: 1})  # a chunk beside single tokens
    bring({0: 17, 2: 1, 3: 3}, pad=1)
    owned = [b for b in (0, 2, 3)]
    assert batch.left.item() == pages - prefix // 16 - sum(-(-length[b] // 16) - prefix // 16 for b in owned)
    table = batch.block_table.tolist()
    held = [p for b in owned for p in table[b][prefix // 16:-(-length[b] // 16)]] + table[4][:prefix // 16]
    assert len(set(held)) == len(held) and not set(held) & set(batch.free_pages[:batch.left.item()].tolist())


@pytest.mark.parametrize("prefix,window", [(64, 0), (0, 20)])
def test_captured_step_equals_the_eager_one(dev, prefix, window):
    """Replays, with requests ending and starting eagerly between them."""
    layer, a = setup(dev, prefix, window, 2)
    _, b = setup(dev, prefix, window, 2)
    x, add = torch.zeros(4, 512, device=dev), torch.zeros(4, 512, device=dev, dtype=torch.bfloat16)
    g = torch.Generator(device=dev).manual_seed(5)

    def prompt(lengths):
        rows = sum(lengths.values())
        xs = torch.randn(rows, 512, device=dev, generator=g)
        for r in (a, b):
            r.brings(lengths)
            r.plan(rows)
            layer(xs, torch.zeros(rows, 512, device=dev, dtype=torch.bfloat16), r, max(lengths.values()))

    def step(r):
        r.plan(4)
        return layer(x, add, r, 1)
    if prefix:
        prompt({4: prefix})
    for r in (a, b):
        r.start([0, 1, 2, 3])
    prompt({0: 10, 1: 33, 2: 1, 3: 60})
    for r in (a, b):
        r.brings(dict.fromkeys(range(4), 1))
        step(r)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(a)
    for i in range(25):  # across pages' ends
        if i in (6, 13):
            for r in (a, b):
                r.end([i % 4])
                r.start([i % 4])
            prompt({i % 4: 7})
            for r in (a, b):
                r.brings(dict.fromkeys(range(4), 1))
        if i == 18:  # one slot stands still: the batch has a row to spare
            for r in (a, b):
                r.brings({0: 1, 2: 1, 3: 1})
        x.normal_(generator=g)
        add.normal_(generator=g)
        want = step(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(got, want))
        assert torch.equal(a.kv_len, b.kv_len) and torch.equal(a.block_table, b.block_table) and torch.equal(a.left, b.left)


@pytest.mark.parametrize("argv", [[], ["--window", "100"]])
def test_the_example_runs(dev, monkeypatch, capsys, argv):
    import decode_loop
    monkeypatch.setattr(sys, "argv", ["decode_loop.py", "--steps", "25", "--prefix", "128"] + argv)
    decode_loop.main()
    assert "25 steps of 16 requests" in capsys.readouterr().out
