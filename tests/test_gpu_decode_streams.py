"""The plan, the rotation and attention with sinks or behind shared prefixes on
streams and in graphs: calls given another stream with memory of their own, two
streams at once, two captured graphs that share a workspace."""
import numpy as np
import pytest
import torch

from luisaml_amd import capi, synth
from tests import kv_cases as kc

pytestmark = pytest.mark.gpu
BUSY = 20_000_000  # cycles, about 10 ms: longer than everything the host does meanwhile
NAMES = ["plan", "rope", "sinks", "shared"]


def i32(a, dev):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=dev)


def t(dev, seed, *s):
    return torch.from_numpy(synth.normal(seed, s).astype(np.float32)).to(dev)


def cases(dev, seed=0):
    """name -> (call(**kw) -> tensors, the workspace that it takes, in bytes)"""
    rng = np.random.default_rng(4 + seed)
    seqs, kv = 6, [6000, 2000, 1000, 700, 6000, 300]
    table, pages = kc.tables(kv, 64, rng)
    c = capi.kv_cache(pages, 2, 64, 64, dev)
    tab, lens, cu = i32(table, dev), i32(kv, dev), i32(np.concatenate([[0], np.cumsum(kv)]), dev)
    capi.kv_cache_write(t(dev, 5 + seed, sum(kv), 2, 64), t(dev, 6 + seed, sum(kv), 2, 64), *c, tab, lens, cu, max(kv))
    q, one = t(dev, 7 + seed, seqs, 8, 64), i32(range(seqs + 1), dev)
    tab[1:3, :8] = tab[0, :8]  # sequences 0 to 2 share 512 tokens
    groups = (i32([0, 3], dev), tab[:1, :8], i32([512], dev))
    new, held = i32(rng.integers(0, 2000, seqs), dev), i32([0, 100, 17, 5, 0, 64], dev)
    free, count = torch.arange(900, dtype=torch.int32, device=dev), i32([900], dev)
    rows = int(new.sum().item()) + 10
    x, pos, turns, g = t(dev, 8 + seed, 3000, 10, 64), i32(rng.integers(0, 500, 3000), dev), capi.rope_table(500, 64, device=dev), \
        1 + 0.1 * t(dev, 9, 64)

    def plan(**kw):
        pt = torch.full((seqs, 160), -1, dtype=torch.int32, device=dev)
        torch.cuda.synchronize()
        return (*capi.kv_cache_plan(new, held, pt, free, count, 16, tokens=rows, **kw), pt)  # (kept, as the call may be pending)
    lib = capi.lib()
    return {
        "plan": (plan, lib.lcml_fp8_kv_cache_plan_workspace_bytes(seqs, rows)),
        "rope": (lambda **kw: capi.qk_norm_rope(x[:, :8], x[:, 8:], pos, turns, g, g, **kw), 0),
        "sinks": (lambda **kw: (capi.attention(q, *c, tab, lens, one, 1, 6000, 0.125, window=3000, sinks=4, **kw),),
                  lib.lcml_fp8_attention_workspace_bytes(seqs, seqs, 8, 2, 64, 1, 6000)),
        "shared": (lambda **kw: (capi.attention_shared(q, *c, tab, lens, one, *groups, 1, 5500, 512, 0.125, **kw),),
                   lib.lcml_fp8_attention_shared_workspace_bytes(seqs, seqs, 1, 8, 2, 64, 1, 5500, 512)),
    }


@pytest.mark.parametrize("handle", [False, True])
@pytest.mark.parametrize("name", NAMES)
def test_own_memory_is_its_streams(dev, name, handle):
    """What the current stream allocates and fills while the call waits its turn
    on another one does not reach the call's workspace and results."""
    call = cases(dev)[name][0]
    want = [a.clone() for a in call()]
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    side = torch.cuda.Stream()
    if name != "plan":  # (whose case waits for its own inputs)
        with torch.cuda.stream(side):
            torch.cuda._sleep(BUSY)
    got = call(stream=side.cuda_stream if handle else side)
    junk = [torch.full((n,), 0xFF, dtype=torch.uint8, device=dev) for n in (512, 4096, 1 << 16, 1 << 18, 1 << 20, 3 << 20)
            for _ in range(4)]
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert all(bool((j == 0xFF).all()) for j in junk)


@pytest.mark.parametrize("name", NAMES)
def test_two_streams_at_once(dev, name):
    calls = [cases(dev, seed)[name][0] for seed in (0, 50)]
    want = [[a.clone() for a in call()] for call in calls]
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in calls]
    for _ in range(20):
        got = [call(stream=s) for call, s in zip(calls, sides)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


@pytest.mark.parametrize("name", ["sinks", "shared"])
def test_two_graphs_that_share_a_workspace(dev, name):
    """Replayed one after the other on one stream, with eager work between."""
    both = [cases(dev, seed)[name] for seed in (0, 50)]
    want = [call()[0].clone() for call, _ in both]
    ws = torch.empty(max(16, *(n for _, n in both)), dtype=torch.uint8, device=dev)
    graphs, outs = [], [torch.empty_like(w) for w in want]
    torch.cuda.synchronize()
    for (call, _), out in zip(both, outs):
        call(out=out, workspace=ws)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(out=out, workspace=ws)
        graphs.append(g)
    for step in range(5):
        for out in outs:
            out.fill_(float(step))
        ws.fill_(255)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
