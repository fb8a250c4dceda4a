"""GPU parity of lcml_fp8_kv_cache_plan with the plain plan, entry by entry."""
import numpy as np
import pytest
import torch

from luisaml_amd import capi
from tests import decode_cases as dc

pytestmark = pytest.mark.gpu


def i32(a, dev):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=dev)


def run(dev, n, held, T=16, cols=None, pages=None, ended=None, own=None, tokens=None, free=None, change=None, seed=0,
        wide=0, rows="both"):
    rng = np.random.default_rng(seed)
    most = max([max(a, 0) + max(b, 0) for a, b in zip(n, held)] + [1])
    cols = -(-most // T) + 1 if cols is None else cols
    need = sum(-(-max(x, 0) // T) for x in held)
    pages = need + sum(-(-max(x, 0) // T) + 1 for x in n) + 3 if pages is None else pages
    table, stack, have = dc.pool(held, T, cols, pages, rng)
    have = have if free is None else free
    if change:
        change(table)
    total = sum(max(x, 0) for x in n)
    tokens = total + 5 if tokens is None else tokens
    want = dc.plan(n, held, table, stack, have, T, ended, own, tokens)
    seqs = len(n)
    big = torch.full((seqs, cols + wide), -3, dtype=torch.int32, device=dev)
    big[:, :cols] = i32(table.reshape(seqs, cols), dev)
    st = i32(stack, dev)
    kw = {}
    if rows in ("both", "positions"):
        kw["positions"] = torch.full((tokens,), 77, dtype=torch.int32, device=dev)
    if rows in ("both", "slots"):
        kw["slots"] = torch.full((tokens,), 77, dtype=torch.int64, device=dev)
    kv, cu, left, pos, slots = capi.kv_cache_plan(
        i32(n, dev), i32(held, dev), big[:, :cols], st, i32([have], dev), T,
        ended=None if ended is None else i32(ended, dev), first_own=None if own is None else i32(own, dev), **kw)
    torch.cuda.synchronize()
    assert kv.tolist() == want[0] and cu.tolist() == want[1] and left.tolist() == [want[2]]
    assert np.array_equal(big[:, :cols].cpu().numpy(), want[5]) and (big[:, cols:] == -3).all()
    assert st.tolist() == list(want[6])
    assert (pos is None) == (rows not in ("both", "positions")) and (slots is None) == (rows not in ("both", "slots"))
    assert pos is None or pos.tolist() == want[3]
    assert slots is None or slots.tolist() == want[4]
    return want


@pytest.mark.parametrize("T", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("rows", ["both", "positions", "slots", "none"])
def test_ragged(dev, T, rows):
    run(dev, [1, 0, 17, 300, 1, 5, 16, 256], [0, 40, 15, 16, 256, 255, 240, 1], T, seed=T, rows=rows, wide=3)


@pytest.mark.parametrize("seqs", [1, 2, 63, 64, 65, 1023, 1024, 1025, 2048, 2049, 5000])
def test_decode_of_many_sequences(dev, seqs):
    rng = np.random.default_rng(seqs)
    held = rng.integers(0, 100, seqs).tolist()
    ended = (rng.random(seqs) < 0.2).astype(int).tolist()
    n = [0 if e and rng.random() < 0.5 else 1 for e in ended]
    run(dev, n, held, 16, ended=ended, own=rng.integers(0, 3, seqs).tolist(), seed=seqs)


@pytest.mark.parametrize("total", [250, 251, 252, 2042, 2043, 2044, 70000])
def test_prompts_around_the_change_of_kernels(dev, total):
    run(dev, [total - total // 3, 0, total // 3], [3, 5, 1000], 16, ended=[0, 1, 0], seed=total)


@pytest.mark.parametrize("free", [-4, 0, 1, 5, 12])
@pytest.mark.parametrize("extra", [0, 4000])
def test_too_few_pages(dev, free, extra):
    """Pages run out inside a sequence: -1 from there on, as many lacking."""
    run(dev, [40, 40 + extra, 1, 100], [5, 0, 16, 33], 16, free=free, seed=free + 9)


def test_tables_that_are_too_narrow(dev):
    want = run(dev, [100, 1, 20], [0, 90, 30], 16, cols=3, seed=1)
    assert -1 in want[4]
    run(dev, [100, 1, 20], [0, 90, 30], 16, cols=0, seed=1, pages=5)
    run(dev, [5000, 1, 20], [0, 90, 30], 16, cols=3, seed=1)


def test_no_sequences_no_pages_no_rows(dev):
    run(dev, [], [], 16, cols=4, pages=3, tokens=7)
    run(dev, [], [], 16, cols=4, pages=3, tokens=0)
    run(dev, [3, 1], [0, 0], 16, pages=0, cols=2)
    run(dev, [0, 0], [0, 17], 16, tokens=0)
    run(dev, [0, 0], [0, 17], 16, tokens=3000)


def test_rows_beyond_the_batch_are_cut(dev):
    run(dev, [10, 20, 30], [1, 2, 3], 16, tokens=25)


def test_negative_counts_and_pages_outside(dev):
    """Negative lengths and tokens count as none; entries that are no pages do
    not come back, and leave no hole in the stack."""
    def change(table):
        table[1, 0], table[1, 2], table[3, 1] = -1, 10 ** 6, -7
    run(dev, [-3, 2, 1, 0], [-5, 60, 20, 40], 16, ended=[0, 1, -2, 5], own=[0, 0, -1, 0], change=change, seed=3)


def test_a_stack_that_is_full(dev):
    """More pages come back than there is room for: the last ones are dropped."""
    run(dev, [1, 0, 0], [0, 100, 100], 16, ended=[0, 1, 1], pages=20, free=15, seed=4)


def test_ended_and_started_again_in_one_step(dev):
    run(dev, [50, 3, 7], [100, 40, 17], 16, ended=[1, 0, 1], seed=5)
    run(dev, [50, 3000, 7], [100, 40, 17], 16, ended=[1, 0, 1], own=[2, 0, 1], seed=5)


@pytest.mark.parametrize("tokens", [12, 2100])
def test_in_place_captured_and_replayed(dev, tokens):
    """Steps in a graph whose lengths and stack run on in place, with eager work
    between the replays; equal to the plain plan after every one."""
    T, seqs = 16, 9
    rng = np.random.default_rng(7)
    held = rng.integers(0, 60, seqs).tolist()
    table, stack, have = dc.pool(held, T, 12, 90, rng)
    kv, tab, st, left = i32(held, dev), i32(table, dev), i32(stack, dev), i32([have], dev)
    n, ended = i32([1] * seqs, dev), i32([0] * seqs, dev)
    cu = i32([0] * (seqs + 1), dev)
    pos, slots = torch.zeros(tokens, dtype=torch.int32, device=dev), torch.zeros(tokens, dtype=torch.int64, device=dev)
    need = capi.lib().lcml_fp8_kv_cache_plan_workspace_bytes(seqs, tokens)
    ws = torch.empty(max(need, 8), dtype=torch.uint8, device=dev)
    args = dict(ended=ended, kv_len_out=kv, cu_q=cu, left=left, positions=pos, slots=slots, workspace=ws)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        capi.kv_cache_plan(n, kv, tab, st, left, T, **args)
    torch.cuda.synchronize()
    now = dict(held=held, table=table, stack=stack.tolist(), free=have)
    for step in range(25):
        e = (rng.random(seqs) < 0.1).astype(int).tolist()
        m = [int(x) for x in rng.integers(0, 3, seqs)]
        n.copy_(i32(m, dev))
        ended.copy_(i32(e, dev))
        g.replay()
        torch.cuda.synchronize()
        want = dc.plan(m, now["held"], now["table"], now["stack"], now["free"], T, e, None, tokens)
        assert kv.tolist() == want[0] and cu.tolist() == want[1] and left.tolist() == [want[2]]
        assert np.array_equal(tab.cpu().numpy(), want[5]) and st.tolist() == want[6]
        assert pos.tolist() == want[3] and slots.tolist() == want[4]
        now = dict(held=want[0], table=want[5], stack=want[6], free=want[2])


def test_slots_past_32_bits(dev):
    """Page numbers times their tokens beyond 2^31."""
    T, seqs = 256, 2
    pages = 1 << 24
    st = torch.arange(pages, dtype=torch.int32, device=dev)
    table = torch.full((seqs, 4), -1, dtype=torch.int32, device=dev)
    kv, cu, left, pos, slots = capi.kv_cache_plan(i32([300, 2], dev), i32([0, 0], dev), table, st, i32([pages], dev), T, tokens=302)
    torch.cuda.synchronize()
    assert slots[:256].tolist() == [(pages - 1) * T + i for i in range(256)]
    assert slots[300:].tolist() == [(pages - 3) * T, (pages - 3) * T + 1] and left.item() == pages - 3


def test_other_stream(dev):
    s = torch.cuda.Stream()
    a = [i32(x, dev) for x in ([3, 1], [0, 20])]
    table, st = torch.full((2, 4), -1, dtype=torch.int32, device=dev), torch.arange(6, dtype=torch.int32, device=dev)
    torch.cuda.synchronize()
    kv, cu, left, pos, slots = capi.kv_cache_plan(*a, table, st, i32([6], dev), 16, tokens=4, stream=s)
    s.synchronize()
    assert kv.tolist() == [3, 21] and cu.tolist() == [0, 3, 4] and pos.tolist() == [0, 1, 2, 20] and left.item() == 5
