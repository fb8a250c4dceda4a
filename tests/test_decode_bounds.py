"""The example's decode loop at the lengths that its tables are made for: the
host's count of what each slot holds, and requests that end there."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def requests(**kw):
    from decode_loop import Requests
    a = dict(slots=3, prefix=32, most=100, pages=20, kv_heads=1, page_tokens=16, head_dim=16, rows=8, device="cpu")
    return Requests(**(a | kw))


def test_the_hosts_count():
    r = requests()
    r.start([0, 2])
    r.brings({0: 60, 1: 3, 3: 32})
    r.grow()
    assert r.held == [92, 3, 32, 32]
    r.brings({0: 4, 2: 1})
    for n in range(1, 3):
        r.grow()
        assert r.held == [92 + 4 * n, 3, 32 + n, 32]
    with pytest.raises(ValueError, match="slot 0 holds 100 tokens and brings 4: 100 at most"):
        r.grow()
    assert r.held == [100, 3, 34, 32]  # none of the batch
    r.brings({2: 66, 0: 0})
    r.grow()
    assert r.held[2] == 100


def test_a_step_past_the_tables_is_refused(monkeypatch):
    """Before anything is launched."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    r = requests()
    r.brings({1: 101})
    with pytest.raises(ValueError, match="100 at most"):
        r.plan(101)


@pytest.mark.gpu
@pytest.mark.parametrize("window", [0, 20])
def test_a_request_up_to_its_last_token(dev, window):
    """Single tokens up to the end of the tables, against the layer in 64 bits;
    a request that ends there leaves its pages to the next one."""
    from decode_loop import RotaryLayer
    layer = RotaryLayer(512, 8, 2, 64, 1024, dev, 100, window, 3, seed=1)
    r = requests(prefix=0, kv_heads=2, head_dim=64, pages=9, rows=100, device=dev)
    none = torch.zeros(0, 2, 64, dtype=torch.float64, device=dev)
    g = torch.Generator(device=dev).manual_seed(3)
    for again in range(2):
        r.start([1])
        history = {1: (none, none)}
        for n in (97, 1, 1, 1):
            x, add = torch.randn(n, 512, device=dev, generator=g), torch.randn(n, 512, device=dev, generator=g).bfloat16()
            at = r.held[1]
            r.brings({1: n})
            r.plan(n)
            h, y = layer(x, add, r, n)
            hp, yp = layer.plain(x, add, [1], [(n, at)], history)
            torch.cuda.synchronize()
            assert r.kv_len.tolist() == r.held == [0, at + n, 0, 0]
            rel = [((a.double() - b).norm() / b.norm()).item() for a, b in ((h, hp), (y, yp))]
            assert rel[0] < 5e-2 and rel[1] < 1e-1, rel  # five roundings to E4M3 in a row, three on the way to h
        r.brings({1: 1})
        with pytest.raises(ValueError, match="100 at most"):
            r.plan(1)
        r.end([1])
        assert r.left.item() == 9 and r.held == [0] * 4


@pytest.mark.gpu
@pytest.mark.parametrize("argv", [["--prefix", "128"], ["--window", "100"]])
def test_requests_end_at_the_most_tokens(dev, monkeypatch, capsys, argv):
    """Of 16 slots with 50 + 37 b tokens (behind a prompt 128 more) some get there."""
    import decode_loop
    seen = []
    grow = decode_loop.Requests.grow
    monkeypatch.setattr(decode_loop.Requests, "grow", lambda self: (grow(self), seen.append(list(self.held))))
    most = 620 + (128 if "--prefix" in argv else 0)
    monkeypatch.setattr(sys, "argv", ["decode_loop.py", "--steps", "60", "--most", str(most)] + argv)
    decode_loop.main()
    assert "60 steps of 16 requests" in (out := capsys.readouterr().out)
    held = [s[:16] for s in seen]
    assert max(max(s) for s in held) == most and sum(s.count(most) for s in held) >= 3
    assert f"lengths {held[-1]}," in out
