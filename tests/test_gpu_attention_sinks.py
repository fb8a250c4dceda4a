"""GPU parity of attention with a window and sinks with the 64-bit definition
over the same codes (decode_cases.check_attention)."""
import numpy as np
import pytest
import torch

from luisaml_amd import capi, synth
from tests import decode_cases as dc
from tests import kv_cases as kc
from tests.test_gpu_attention import DT, MANY, filled, i32

pytestmark = pytest.mark.gpu


def run(dev, kv_len, n, window, sinks, T=16, H=2, G=2, D=64, qt="b", ot="b", causal=True, seed=0, spread=1.0, change=None,
        max_q=None, max_kv=None, kernel=None):
    kv_len, cu = np.array(kv_len), np.concatenate([[0], np.cumsum(n)])
    cache, table = filled(kv_len, T, H, D, seed, spread)
    q = synth.normal(seed + 7, (cu[-1], H * G, D)).astype(np.float32)
    q = kc.bf16(q) if qt == "b" else q
    if change:
        table = change(q, cache, table)
    out = torch.full((cu[-1], H * G * D + 5), 9.0, dtype=DT[ot], device=dev)
    od = out[:, 3:3 + H * G * D].view(-1, H * G, D)
    mq = max(list(n) + [1]) if max_q is None else max_q
    mk = int(max(list(kv_len) + [1])) if max_kv is None else max_kv
    capi.kernel_trace()
    capi.attention(torch.from_numpy(q).to(dev).to(DT[qt]), *cache.to(dev), i32(table, dev), i32(kv_len, dev), i32(cu, dev), mq, mk,
                   D ** -0.5, causal=causal, window=window, sinks=sinks, out=od)
    torch.cuda.synchronize()
    if kernel:
        assert kernel in ", ".join(capi.kernel_trace())
    got = od.float().cpu().numpy().astype(np.float64)
    assert (out[:, :3] == 9.0).all() and (out[:, 3 + H * G * D:] == 9.0).all()
    dc.check_attention(got, q, cache, table, kv_len, cu, H, D ** -0.5, ot == "b", causal=causal, window=window, sinks=sinks)
    return got


LENS = [1, 2, 16, 63, 64, 65, 130, 200, 331]
SHAPES = [(16, 2, 4, 128), (32, 1, 1, 64), (64, 2, 7, 128), (16, 3, 2, 80), (128, 1, 16, 64), (256, 1, 8, 256), (16, 1, 20, 96),
          (32, 2, 4, 16), (64, 1, 4, 192)]


@pytest.mark.parametrize("T,H,G,D", SHAPES)
@pytest.mark.parametrize("qt,ot", [("b", "b"), ("b", "f"), ("f", "f"), ("f", "b")])
def test_single_tokens(dev, T, H, G, D, qt, ot):
    run(dev, LENS, [1] * len(LENS), 40, 5, T, H, G, D, qt, ot, seed=T + D + G)


@pytest.mark.parametrize("T,H,G,D", SHAPES)
@pytest.mark.parametrize("qt,ot", [("b", "b"), ("b", "f"), ("f", "f"), ("f", "b")])
def test_many_rows(dev, T, H, G, D, qt, ot):
    run(dev, [1, 17, 64, 170, 230, 350], [1, 17, 64, 35, 130, 7], 50, 3, T, H, G, D, qt, ot, seed=T + D + G, max_q=MANY,
        kernel="attention_many")


# around the 64 tokens of a step, on both sides of the hole and without one
@pytest.mark.parametrize("sinks", [1, 4, 63, 64, 65, 128, 200, 10 ** 6])
@pytest.mark.parametrize("window", [1, 5, 63, 64, 65, 100, 1000])
@pytest.mark.parametrize("max_q", [None, MANY])
def test_windows_and_sinks(dev, sinks, window, max_q):
    run(dev, [90, 133, 300, 7, 257], [6, 70, 1, 7, 3], window, sinks, 32, 1, 2, 32, seed=window + sinks, max_q=max_q)


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31, 2 ** 40])
@pytest.mark.parametrize("sinks", [2 ** 31 - 1, 2 ** 31, 2 ** 40])
def test_huge_windows_and_sinks(dev, window, sinks):
    run(dev, [90, 7], [6, 7], window, 3)
    run(dev, [90, 7], [6, 7], 5, sinks)
    run(dev, [90, 7], [6, 7], 5, sinks, max_q=MANY)
    run(dev, [90, 7], [6, 7], window, sinks)


@pytest.mark.parametrize("max_q", [None, MANY])
def test_no_window_no_sinks_is_attention(dev, max_q):
    run(dev, [90, 133], [5, 60], 0, 4, max_q=max_q)
    run(dev, [90, 133], [5, 60], 30, 0, max_q=max_q)


@pytest.mark.parametrize("max_q", [None, MANY])
def test_not_causal(dev, max_q):
    run(dev, [40, 1, 200, 77], [10, 1, 100, 1], 20, 6, 16, 2, 2, 64, causal=False, seed=3, max_q=max_q)
    run(dev, [40, 1, 200, 77], [45, 3, 100, 1], 20, 6, 16, 2, 2, 64, causal=False, seed=3, max_q=max_q)  # rows before the first token


@pytest.mark.parametrize("max_q", [None, MANY])
def test_rows_that_see_nothing(dev, max_q):
    """No tokens; rows before the first position; missing pages, the sinks' among
    them; a table with too few columns."""
    def holes(q, cache, table):
        t = table.copy()
        t[4, :], t[5, 1], t[6, 0] = -1, 10 ** 6, -5
        return t[:, :6]
    got = run(dev, [0, 3, 0, 20, 30, 60, 90, 130], [1, 8, 4, 0, 2, 3, 33, 2], 20, 5, 16, 2, 2, 64, seed=1, change=holes, max_q=max_q)
    assert (got[:1] == 0).all() and (got[1:6] == 0).all() and not (got[6:9] == 0).any()


@pytest.mark.parametrize("D", [64, 80, 256])
@pytest.mark.parametrize("max_q", [None, MANY])
@pytest.mark.parametrize("n", [1, 40])
def test_nan_codes_reach_the_rows_that_see_them(dev, D, max_q, n):
    def change(q, cache, table):
        cache.codes[1][table[0, 0], :, 2, 5] = kc.NAN_CODE   # a sink of sequence 0
        cache.codes[1][table[1, 0], :, 9, 6] = kc.NAN_CODE   # past the sinks, hidden from late rows
        cache.codes[1][table[1, 9], :, 2, 7] = kc.NAN_CODE   # in the window of late rows
        return table
    got = run(dev, [160, 160], [n, n], 30, 4, 16, 1, 4, D, seed=2, change=change, max_q=max_q)
    assert np.isnan(got[n - 1, :, 5]).all() and not np.isnan(got[-1, :, 6]).any() and np.isnan(got[-1, :, 7]).all()


@pytest.mark.parametrize("max_q", [None, MANY])
@pytest.mark.parametrize("ot", ["b", "f"])
def test_scales_far_apart(dev, max_q, ot):
    run(dev, [100, 400], [20, 20], 70, 20, 16, 1, 4, 64, "b", ot, seed=9, spread=1e8, max_q=max_q)


@pytest.mark.parametrize("n,L,window,sinks", [(1, 5000, 3000, 4), (1, 20011, 9000, 1000), (3, 9000, 8000, 64), (40, 6000, 2500, 7),
                                              (1, 6000, 40, 5900), (2, 4000, 3990, 4)])
@pytest.mark.parametrize("ot", ["b", "f"])
def test_long_sequences(dev, n, L, window, sinks, ot):
    """Windows at which the work of a row is split and joined, sinks that fill
    whole parts, and holes of a few tokens."""
    run(dev, [L, L // 3, 7], [n, n, min(n, 7)], window, sinks, 64, 1, 4, 64, "b", ot, seed=n,
        kernel="attention_few, attention_join" if n < 40 else None)


@pytest.mark.parametrize("D,kernel", [(64, "attention_few"), (128, "attention_many, attention_join")])
def test_many_queries_over_a_long_window(dev, D, kernel):
    run(dev, [3000, 1000], [700, 100], 1500, 100, 64, 1, 4, D, seed=D, kernel=kernel)


@pytest.mark.parametrize("qt,ot", [("b", "b"), ("b", "f"), ("f", "f"), ("f", "b")])
@pytest.mark.parametrize("D", [32, 64, 80, 128])
def test_eight_wavefronts_and_none_of_their_steps(dev, D, qt, ot):
    """One workgroup a row tile: 9 to 20 steps, of which most wavefronts have two
    or three, some one and in short sequences none."""
    run(dev, [1200, 1, 70, 700, 0, 1130], [1, 1, 1, 1, 1, 1], 900, 130, 16, 2, 4, D, qt, ot, seed=D, max_kv=1200, kernel="attention_few")
    run(dev, [1200, 300], [3, 2], 900, 130, 32, 1, 4, D, qt, ot, seed=D)
    assert "attention_join" not in ", ".join(capi.kernel_trace())


@pytest.mark.parametrize("kv,n", [([300, 40], [1, 1]), ([3000, 900], [1, 2]), ([700, 300], [100, 80])])
def test_longer_than_max_kv(dev, kv, n):
    run(dev, kv, n, 200, 10, 16, 1, 2, 64, max_kv=64, seed=9)


def test_graph_while_sequences_grow(dev):
    kv, B = [30, 64, 200], 3
    cache, table = filled([x + 40 for x in kv], 16, 2, 64, 5)
    c = cache.to(dev)
    q = torch.from_numpy(synth.normal(3, (B, 8, 64))).to(dev).bfloat16()
    idx = (i32(table, dev), i32(kv, dev), i32(range(B + 1), dev))
    need = capi.lib().lcml_fp8_attention_workspace_bytes(B, B, 8, 2, 64, 1, 2048)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)
    out = torch.empty_like(q)
    call = lambda **kw: capi.attention(q, *c, *idx, 1, 2048, 0.125, window=50, sinks=4, **kw)  # noqa: E731
    call(out=out, workspace=ws)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(out=out, workspace=ws)
    for step in range(5):
        idx[1].add_(7)
        q.neg_()
        want = call()
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        kvs = idx[1].cpu().numpy()
        dc.check_attention(out.float().cpu().numpy().astype(np.float64), q.float().cpu().numpy(), cache, table, kvs, range(B + 1), 2,
                           0.125, True, window=50, sinks=4)
