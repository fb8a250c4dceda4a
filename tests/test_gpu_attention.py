"""GPU parity of lcml_fp8_attention with the 64-bit definition over the same
codes; tolerances from kv_cases.attention_bound (roundings counted, with the
row's own sums)."""
import numpy as np
import pytest
import torch

from luisaml_amd import capi, synth
from tests import kv_cases as kc

pytestmark = pytest.mark.gpu
DT = {"f": torch.float32, "b": torch.bfloat16}


def i32(a, dev):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=dev)


def filled(kv_len, T, H, D, seed, spread=1.0):
    """A cache with tokens in it, and garbage (NaN codes) everywhere else."""
    rng = np.random.default_rng(seed)
    table, pages = kc.tables(kv_len, T, rng)
    cache = kc.Cache(pages, H, T, D, rng)
    cu = np.concatenate([[0], np.cumsum(kv_len)])
    k = synth.normal(seed + 1, (cu[-1], H, D)) * np.exp(synth.normal(seed + 2, (D,), std=0.4))
    v = synth.normal(seed + 3, (cu[-1], H, D))
    if spread != 1.0:  # pages of very different sizes
        f = np.exp(np.log(spread) * (rng.random((cu[-1] // 16 + 1, H, 1)) - 0.5)).repeat(16, 0)[:cu[-1]]
        v = v * f
    cache.write(k.astype(np.float32), v.astype(np.float32), table, np.array(kv_len), cu)
    return cache, table


def run(dev, kv_len, n, T=16, H=2, G=2, D=64, qt="b", ot="b", causal=True, window=0, seed=0, spread=1.0, q_scale=1.0,
        cache=None, change=None, max_q=None, max_kv=None, check=True):
    kv_len, cu = np.array(kv_len), np.concatenate([[0], np.cumsum(n)])
    cache, table = filled(kv_len, T, H, D, seed, spread) if cache is None else cache
    q = synth.normal(seed + 7, (cu[-1], H * G, D)).astype(np.float32) * np.float32(q_scale)
    q = kc.bf16(q) if qt == "b" else q
    if change:
        table = change(q, cache, table)
    scale = D ** -0.5
    # rows of a wider tensor, off its alignment
    wide = torch.zeros(cu[-1], H * G * D + 3, dtype=DT[qt], device=dev)
    qd = wide[:, 1:1 + H * G * D].view(-1, H * G, D)
    qd.copy_(torch.from_numpy(q))
    out = torch.full((cu[-1], H * G * D + 5), 9.0, dtype=DT[ot], device=dev)
    od = out[:, 3:3 + H * G * D].view(-1, H * G, D)
    c = cache.to(dev)
    idx = (i32(table, dev), i32(kv_len, dev), i32(cu, dev))
    mq = max(list(n) + [1]) if max_q is None else max_q
    mk = int(max(list(kv_len) + [1])) if max_kv is None else max_kv
    capi.attention(qd, *c, *idx, mq, mk, scale, causal=causal, window=window, out=od)
    torch.cuda.synchronize()
    got = od.float().cpu().numpy().astype(np.float64)
    assert (out[:, :3] == 9.0).all() and (out[:, 3 + H * G * D:] == 9.0).all()
    if check:
        o, mass, reach = kc.attention(q, cache, table, kv_len, cu, H, float(np.float32(scale)), causal, window)
        bound = kc.attention_bound(mass, reach, D, max(list(kv_len) + [1]), ot == "b")
        assert np.array_equal(np.isnan(got), np.isnan(o))
        bad = kc.outside(got, o, bound, ot == "b")
        assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], o[bad][:5], bound[bad][:5])
    return got


LENS = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 200]


@pytest.mark.parametrize("T,H,G,D", [(16, 2, 4, 128), (32, 1, 1, 64), (64, 2, 7, 128), (16, 3, 2, 80), (128, 1, 16, 64),
                                     (256, 1, 8, 256), (16, 1, 20, 96), (32, 2, 4, 16), (64, 1, 4, 192)])
@pytest.mark.parametrize("qt,ot", [("b", "b"), ("b", "f"), ("f", "f"), ("f", "b")])
def test_single_tokens(dev, T, H, G, D, qt, ot):
    run(dev, LENS, [1] * len(LENS), T, H, G, D, qt, ot, seed=T + D + G)


@pytest.mark.parametrize("T,H,G,D", [(16, 2, 4, 128), (32, 1, 1, 64), (64, 2, 7, 128), (16, 1, 2, 80), (128, 1, 16, 64),
                                     (256, 1, 8, 256), (16, 1, 4, 192)])
@pytest.mark.parametrize("qt,ot", [("b", "b"), ("f", "f")])
def test_prompts_and_chunks(dev, T, H, G, D, qt, ot):
    run(dev, [1, 17, 64, 70, 130, 150], [1, 17, 64, 35, 130, 7], T, H, G, D, qt, ot, seed=T + D + G)


@pytest.mark.parametrize("n", [2, 3, 4, 5, 8, 9, 16, 17])
def test_a_few_tokens(dev, n):
    run(dev, [n, 30, 100, 257], [n, n, n, n], 16, 2, 4, 64, seed=n)


@pytest.mark.parametrize("window", [1, 5, 16, 40, 1000])
@pytest.mark.parametrize("n", [1, 6, 90])
def test_window(dev, window, n):
    run(dev, [90, 133, 200], [n, n, n], 32, 1, 4, 64, window=window, seed=window + n)


@pytest.mark.parametrize("window", [0, 20])
def test_not_causal(dev, window):
    run(dev, [40, 1, 100, 77], [10, 1, 100, 1], 16, 2, 2, 64, causal=False, window=window, seed=3)


def test_rows_that_see_nothing(dev):
    """No tokens; rows before the first position; missing pages; a table with
    too few columns; no pages at all."""
    def holes(q, cache, table):
        t = table.copy()
        t[4, :], t[5, 1], t[6, 0] = -1, 10 ** 6, -5
        return t[:, :4]
    for n6 in (1, 33):
        got = run(dev, [0, 3, 0, 20, 30, 60, 90], [1, 8, 4, 0, 2, 3, n6], 16, 2, 2, 64, seed=1, change=holes)
        assert (got[:1] == 0).all() and (got[1:6] == 0).all() and not (got[6:9] == 0).any()
    z = capi.kv_cache(0, 2, 16, 64, dev)
    o = capi.attention(torch.ones(2, 4, 64, device=dev), *z, torch.zeros(1, 0, dtype=torch.int32, device=dev), i32([5], dev),
                       i32([0, 2], dev), 2, 5, 0.1)
    assert (o == 0).all()


@pytest.mark.parametrize("n", [1, 50])
@pytest.mark.parametrize("ot", ["b", "f"])
def test_scales_far_apart_and_large_scores(dev, n, ot):
    run(dev, [100, 300], [n, n], 16, 1, 4, 64, "b", ot, seed=9, spread=1e8)
    run(dev, [100, 300], [n, n], 16, 1, 4, 64, "b", ot, seed=9, q_scale=40.0)
    run(dev, [100, 300], [n, n], 16, 1, 4, 64, "b", ot, seed=9, q_scale=1e-6)


@pytest.mark.parametrize("n", [1, 40])
def test_infinite_and_nan_queries_and_codes(dev, n):
    """A query of NaN or with an infinity gives NaN where the formula does; a
    NaN code that is seen reaches its rows, one that is masked does not."""
    def change(q, cache, table):
        q[0, 0, 3] = np.nan
        q[0, 1, :] = 0.0
        cache.codes[1][table[1, 1], :, 2, 5] = kc.NAN_CODE  # position 18 of sequence 1
        return table
    got = run(dev, [60, 60], [n, n], 16, 1, 4, 64, seed=2, change=change, window=0)
    assert np.isnan(got[0, 0]).all() and not np.isnan(got[0, 1]).any()
    assert np.isnan(got[-1, :, 5]).all() and not np.isnan(got[-1, :, 6]).any()
    got = run(dev, [60, 60], [n, n], 16, 1, 4, 64, seed=2, change=change, window=20)
    assert not np.isnan(got[-1]).any()


@pytest.mark.parametrize("n,L", [(1, 5000), (1, 20011), (3, 9000), (40, 6000)])
@pytest.mark.parametrize("ot", ["b", "f"])
def test_long_sequences(dev, n, L, ot):
    """Lengths at which the work of a row is split and joined."""
    run(dev, [L, L // 3, 7], [n, n, min(n, 7)], 64, 1, 4, 64, "b", ot, seed=n)


def test_bounds_of_the_host_hold(dev):
    """max_q and max_kv above the true lengths change nothing but the split;
    the same bits from two calls."""
    a = run(dev, [100, 40], [1, 1], max_q=1, max_kv=100, seed=4, ot="f")
    b = run(dev, [100, 40], [1, 1], max_q=1, max_kv=100, seed=4, ot="f")
    assert np.array_equal(a, b)
    run(dev, [100, 40], [1, 1], max_q=1, max_kv=40000, seed=4, ot="f")
    run(dev, [100, 40], [1, 1], max_q=50, max_kv=100, seed=4, ot="f")


def test_far_larger_max_q(dev):
    """Sequences times max_q beyond the rows that a join could take, where
    nothing is split: workgroups without rows end at once."""
    run(dev, [100, 40], [1, 3], max_q=1 << 22, max_kv=100, seed=4)


@pytest.mark.parametrize("kv,n", [([300, 40], [1, 1]), ([3000, 900], [1, 2]), ([700, 300], [100, 80])])
def test_longer_than_max_kv(dev, kv, n):
    """A graph that outlives its bound: slower, and still the whole sequence."""
    run(dev, kv, n, 16, 1, 2, 64, max_kv=64, seed=9)


def test_other_stream_and_graph(dev):
    """Decode captured in a graph, replayed while lengths grow: equal to the
    eager call each time."""
    kv, B = [30, 64, 200], 3
    cache, table = filled([x + 5 for x in kv], 16, 2, 64, 5)
    c = cache.to(dev)
    q = torch.from_numpy(synth.normal(3, (B, 8, 64))).to(dev).bfloat16()
    idx = (i32(table, dev), i32(kv, dev), i32(range(B + 1), dev))
    need = capi.lib().lcml_fp8_attention_workspace_bytes(B, B, 8, 2, 64, 1, 2048)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)
    out = torch.empty_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        capi.attention(q, *c, *idx, 1, 2048, 0.125, out=out, workspace=ws)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        capi.attention(q, *c, *idx, 1, 2048, 0.125, out=out, workspace=ws)
    for step in range(4):
        idx[1].add_(1)
        q.neg_()
        want = capi.attention(q, *c, *idx, 1, 2048, 0.125)
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_cache_past_32_bit_offsets(dev):
    """Pages past 4 GiB in each cache."""
    H, T, D = 8, 256, 256
    pages = (1 << 32) // (H * T * D) + 2
    c = capi.kv_cache(pages, H, T, D, dev)
    n = 200
    k, v = (torch.from_numpy(synth.normal(s, (n, H, D))).to(dev) for s in (1, 2))
    q = torch.from_numpy(synth.normal(3, (n, H, D))).to(dev).bfloat16()
    outs = []
    for page in (pages - 1, 0):
        idx = (i32([[page]], dev), i32([n], dev), i32([0, n], dev))
        capi.kv_cache_write(k, v, *c, *idx, n)
        outs.append(capi.attention(q, *c, *idx, n, n, D ** -0.5))
        one = (idx[0], idx[1], i32([0, 1], dev))
        outs.append(capi.attention(q[-1:], *c, *one, 1, n, D ** -0.5))
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3]) and outs[0].abs().sum() > 0


# A max_q far above the true one takes the kernel for many rows.
MANY = 1 << 15


def many(dev, *args, **kw):
    capi.kernel_trace()
    got = run(dev, *args, max_q=MANY, **kw)
    assert any("attention_many" in k for k in capi.kernel_trace())
    return got


@pytest.mark.parametrize("T,H,G,D", [(16, 2, 4, 128), (32, 1, 1, 64), (64, 2, 7, 128), (16, 1, 2, 80), (128, 1, 16, 64),
                                     (256, 1, 8, 256), (16, 1, 4, 192), (32, 2, 4, 16)])
@pytest.mark.parametrize("qt,ot", [("b", "b"), ("b", "f"), ("f", "f"), ("f", "b")])
def test_many_rows(dev, T, H, G, D, qt, ot):
    many(dev, [1, 17, 64, 70, 130, 150], [1, 17, 64, 35, 130, 7], T, H, G, D, qt, ot, seed=T + D + G)


@pytest.mark.parametrize("window,causal", [(1, True), (5, True), (40, True), (64, True), (1000, True), (0, False), (20, False)])
def test_many_rows_window_and_not_causal(dev, window, causal):
    many(dev, [90, 133, 200, 1], [90, 6, 101, 1], 32, 1, 4, 64, window=window, causal=causal, seed=window)


def test_many_rows_that_see_nothing(dev):
    def holes(q, cache, table):
        t = table.copy()
        t[4, :], t[5, 1], t[6, 0] = -1, 10 ** 6, -5
        return t[:, :4]
    got = many(dev, [0, 3, 0, 20, 30, 60, 90], [1, 8, 4, 0, 2, 3, 33], 16, 2, 2, 64, seed=1, change=holes)
    assert (got[:1] == 0).all() and (got[1:6] == 0).all() and not (got[6:9] == 0).any()


@pytest.mark.parametrize("ot", ["b", "f"])
def test_many_rows_scales_far_apart_and_large_scores(dev, ot):
    many(dev, [100, 300], [50, 50], 16, 1, 4, 64, "b", ot, seed=9, spread=1e8)
    many(dev, [100, 300], [50, 50], 16, 1, 4, 64, "b", ot, seed=9, q_scale=40.0)
    many(dev, [100, 300], [50, 50], 16, 1, 4, 64, "b", ot, seed=9, q_scale=1e-6)


@pytest.mark.parametrize("D", [64, 80, 256])
def test_many_rows_infinite_and_nan_queries_and_codes(dev, D):
    def change(q, cache, table):
        q[0, 0, 3] = np.nan
        q[0, 1, :] = 0.0
        cache.codes[1][table[1, 1], :, 2, 5] = kc.NAN_CODE  # position 18 of sequence 1
        return table
    got = many(dev, [60, 60], [40, 40], 16, 1, 4, D, seed=2, change=change, window=0)
    assert np.isnan(got[0, 0]).all() and not np.isnan(got[0, 1]).any()
    assert np.isnan(got[-1, :, 5]).all() and not np.isnan(got[-1, :, 6]).any()
    got = many(dev, [60, 60], [40, 40], 16, 1, 4, D, seed=2, change=change, window=20)
    assert not np.isnan(got[-1]).any()


@pytest.mark.parametrize("ot", ["b", "f"])
@pytest.mark.parametrize("n,D,kernel", [(700, 64, "attention_few, attention_join"), (130, 64, "attention_few, attention_join"),
                                        (9, 64, "attention_few, attention_join"), (700, 128, "attention_many, attention_join")])
def test_long_axis_split_and_joined(dev, n, D, kernel, ot):
    """Parts of many rows and of few, joined a workgroup a row and many rows a
    workgroup."""
    capi.kernel_trace()
    run(dev, [3000, 1000], [n, min(n, 100)], 64, 1, 4, D, "b", ot, seed=n)
    assert kernel in ", ".join(capi.kernel_trace())
