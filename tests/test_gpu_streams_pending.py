"""The plan, the rotation and attention with sinks or behind shared prefixes on
streams that are held back until the host is through: a call that is pending
while the current stream's memory changes hands, and two that start together.
Each test checks that its calls did wait."""
import numpy as np
import pytest
import torch

from luisaml_amd import capi
from tests.test_gpu_decode_streams import NAMES, cases, i32

pytestmark = pytest.mark.gpu
HOLD = 60_000_000  # cycles, about 30 ms
ROUNDS = 4


def calls(dev, seed, name, times):
    """`times` calls(**kw) -> tensors on inputs that are there, each its own
    where it changes them."""
    if name != "plan":
        return [cases(dev, seed)[name][0]] * times
    rng = np.random.default_rng(seed)
    seqs, T = 40, 16
    held, n = rng.integers(0, 900, seqs), rng.integers(0, 2500, seqs)
    ended = (np.arange(seqs) % 5 == 0).astype(np.int32)
    cols, has = 250, -(-held // T)
    table = np.full((seqs, cols), -1, np.int32)
    pages = int(has.sum()) + seqs * cols
    order = rng.permutation(pages)
    for b, k in enumerate(has):
        table[b, :k] = order[has[:b].sum():has[:b].sum() + k]
    stack = np.full(pages, -7, np.int32)
    stack[:pages - has.sum()] = order[has.sum():]
    new, old, gone, count = i32(n, dev), i32(held, dev), i32(ended, dev), i32([pages - has.sum()], dev)
    rows = int(n.sum()) + 10

    def one(pt, free):
        return lambda **kw: (*capi.kv_cache_plan(new, old, pt, free, count, T, tokens=rows, ended=gone, **kw), pt, free)
    made = [one(i32(table, dev), i32(stack, dev)) for _ in range(times)]
    assert capi.lib().lcml_fp8_kv_cache_plan_workspace_bytes(seqs, rows) > 0
    return made


def independent(a, b):
    """Whether b's work runs while a waits: streams can share a hardware queue."""
    with torch.cuda.stream(a):
        torch.cuda._sleep(HOLD // 20)
        over = torch.cuda.Event()
        over.record()
    with torch.cuda.stream(b):
        torch.cuda._sleep(1)
    b.synchronize()
    apart = not over.query()
    torch.cuda.synchronize()
    return apart


def streams(count):
    """Streams none of which holds up another or the current one."""
    found = [torch.cuda.current_stream()]
    for _ in range(32):
        s = torch.cuda.Stream()
        if all(independent(s, t) and independent(t, s) for t in found):
            found.append(s)
        if len(found) > count:
            return found[1:]
    pytest.skip("too few hardware queues")


def hold(sides):
    """Some 30 ms of nothing on each."""
    over = []
    for s in sides:
        with torch.cuda.stream(s):
            torch.cuda._sleep(HOLD)
            over.append(torch.cuda.Event())
            over[-1].record()
    return lambda: not any(e.query() for e in over)


def junk(dev):
    return [torch.full((n,), 0xFF, dtype=torch.uint8, device=dev)
            for n in (512, 4096, 1 << 16, 1 << 18, 1 << 20, 3 << 20) for _ in range(4)]


@pytest.mark.parametrize("handle", [False, True])
@pytest.mark.parametrize("name", NAMES)
def test_own_memory_is_its_streams(dev, name, handle):
    """What the current stream allocates and fills while the call waits does not
    reach the call's workspace and results."""
    made = calls(dev, 0, name, 3)
    want = [a.clone() for a in made[0]()]
    side, = streams(1)
    where = side.cuda_stream if handle else side
    made[1](stream=where)
    del_later = junk(dev)  # so that neither pool has to ask for memory below, which could wait for the call
    torch.cuda.synchronize()
    del del_later
    pending = hold([side])
    got = made[2](stream=where)
    filled = junk(dev)
    torch.cuda.current_stream().synchronize()
    assert pending(), "the call did not wait"
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(bool((j == 0xFF).all()) for j in filled)


@pytest.mark.parametrize("name", NAMES)
def test_two_streams_at_once(dev, name):
    """Both start some ten microseconds apart, each with ROUNDS calls one after the other."""
    made = [calls(dev, seed, name, ROUNDS + 2) for seed in (0, 50)]
    want = [[a.clone() for a in m[0]()] for m in made]
    torch.cuda.synchronize()
    sides = streams(2)
    warm = [[m[1](stream=s) for _ in range(ROUNDS)] for m, s in zip(made, sides)]  # as in the test above: memory for them
    torch.cuda.synchronize()
    del warm
    pending = hold(sides)
    got = [[m[2 + r](stream=s) for r in range(ROUNDS)] for m, s in zip(made, sides)]
    assert pending(), "the calls did not wait"
    torch.cuda.synchronize()
    for rounds, w in zip(got, want):
        assert all(torch.equal(a, b) for g in rounds for a, b in zip(g, w))


@pytest.mark.parametrize("name", ["plan", "rope", "sinks", "shared"])
def test_a_graph_beside_an_eager_call(dev, name):
    """A replay on one stream and an eager call on another, together: neither
    uses the other's workspace."""
    made = [calls(dev, seed, name, 3) for seed in (0, 50)]
    want = [[a.clone() for a in m[0]()] for m in made]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = made[0][1]()
    sides = streams(2)
    made[1][1](stream=sides[1])
    torch.cuda.synchronize()
    pending = hold(sides)
    with torch.cuda.stream(sides[0]):
        graph.replay()
    other = made[1][2](stream=sides[1])
    assert pending(), "the calls did not wait"
    torch.cuda.synchronize()
    for g, w in zip((got, other), want):
        assert all(torch.equal(a, b) for a, b in zip(g, w))
