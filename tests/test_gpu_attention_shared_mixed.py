"""attention_shared() where many rows read a prefix and each sequence brings few:
one launch holds the prefix's workgroups of the kernel for many rows and the own
tokens' ones of the kernel for few.  (With a long bound on the prefix a part of
it has 1000 to 2000 tokens: the prefixes here are of one part and a piece of the
next.)"""
import numpy as np
import pytest
import torch

from luisaml_amd import capi, synth
from tests import decode_cases as dc
from tests import kv_cases as kc
from tests.test_gpu_attention import DT, i32
from tests.test_gpu_attention_shared import batch, run

pytestmark = pytest.mark.gpu
MIXED, FEW = "attention_shared_many, attention_join", "attention_shared_few, attention_join"
# every width that the kernels are built for, whole and not
SHAPES = [(16, 2, 8, 64), (32, 2, 5, 48), (16, 1, 7, 80), (64, 2, 4, 96), (16, 2, 4, 128), (128, 1, 6, 112), (32, 1, 8, 256), (16, 1, 5, 192)]
TYPES = [("b", "b"), ("b", "f"), ("f", "f"), ("f", "b")]
OWN = [4, 5, 16, 17, 63, 64, 65, 130]
GROUPS = [(1090, OWN), (2000, OWN[::-1] + [7, 40])]
ROWS = [4, 1, 3, 4, 2, 4, 4, 3, 4, 4, 1, 4, 0, 4, 2, 4, 4, 4]


def mixed(dev, T, H, G, D, qt="b", ot="b", groups=GROUPS, n=ROWS, kernel=MIXED, max_prefix=1 << 16, **kw):
    return run(dev, groups, n, T, H, G, D, qt, ot, kernel=kernel, max_prefix=max_prefix, **kw)


@pytest.mark.parametrize("T,H,G,D", SHAPES)
@pytest.mark.parametrize("qt,ot", TYPES)
def test_all_widths_and_types(dev, T, H, G, D, qt, ot):
    mixed(dev, T, H, G, D, qt, ot, seed=T + D + G)


@pytest.mark.parametrize("qt,ot", TYPES)
def test_single_tokens(dev, qt, ot):
    mixed(dev, 16, 2, 8, 128, qt, ot, groups=[(1090, OWN * 5)], n=1, seed=3)


@pytest.mark.parametrize("prefix", [1, 16, 63, 64, 100, 1023, 1024, 1025, 1664])
def test_prefixes_of_any_length(dev, prefix):
    """Ends inside pages, steps and parts."""
    mixed(dev, 16, 1, 8, 128, groups=[(prefix, OWN), (prefix // 2 + 1, OWN[::-1] + [7, 40])], seed=prefix)


@pytest.mark.parametrize("T,H,G,D", SHAPES[::2])
@pytest.mark.parametrize("qt,ot", [("b", "b"), ("f", "f")])
def test_nan_codes_and_queries(dev, T, H, G, D, qt, ot):
    def change(q, cache, table, kv, first, pt, plen):
        cache.codes[1][pt[0, 1], :, 2, 5] = kc.NAN_CODE       # the first group's prefix
        cache.codes[1][pt[1, 1000 // T], :, 1, 6] = kc.NAN_CODE
        cache.codes[1][table[10, plen[1] // T], :, 0, 7] = kc.NAN_CODE  # one sequence's own tokens (or its copy of a page)
        cache.codes[0][table[3, plen[0] // T + 1], 0, 0, 9] = kc.NAN_CODE
        q[1, 0, 3] = np.nan
        return first, pt, plen
    got = mixed(dev, T, H, G, D, qt, ot, change=change, groups=[(1152, [T + 5] * 8), (2048, [T + 9] * 10)], max_own=140, seed=D)
    a = sum(ROWS[:8])
    assert np.isnan(got[:a, :, 5]).all() and not np.isnan(got[a:, :, 5]).any()
    assert np.isnan(got[a:, :, 6]).all() and np.isnan(got[1, 0]).all()


@pytest.mark.parametrize("T,H,G,D", SHAPES[1::2])
@pytest.mark.parametrize("qt,ot", TYPES)
def test_scales_far_apart(dev, T, H, G, D, qt, ot):
    mixed(dev, T, H, G, D, qt, ot, spread=1e8, seed=9)


@pytest.mark.parametrize("T,H,G,D", SHAPES)
def test_missing_pages(dev, T, H, G, D):
    """Of a prefix, of own tokens; all of a prefix's; a table with too few columns."""
    def change(q, cache, table, kv, first, pt, plen):
        pt[0, 1], pt[0, 3] = -1, 10 ** 6
        table[2, plen[0] // T:], table[9, plen[1] // T] = -1, -1
        return first, pt[:, :1500 // T], plen
    mixed(dev, T, H, G, D, change=change, seed=D)

    def none(q, cache, table, kv, first, pt, plen):
        pt[0, :] = -1
        table[0, :] = -1
        return first, pt, plen
    got = mixed(dev, T, H, G, D, change=none, seed=D)
    assert (got[:ROWS[0]] == 0).all()


def test_groups_and_rows_inside_a_prefix(dev):
    """An empty group, one without a prefix, sequences of none, one that is being
    prefilled, rows before the first token, and without causality."""
    def change(q, cache, table, kv, first, pt, plen):
        return np.array([1, 6, 6, 8, 18]), np.concatenate([pt[:1], pt[:1], pt[:1], pt[1:]]), np.array([plen[0], 50, 0, plen[1]])
    lens = [p + o for p, own in GROUPS for o in own]
    lens[2], lens[4], lens[9], lens[11] = 900, 0, 2003, 2
    for causal in (True, False):
        mixed(dev, 16, 2, 8, 64, change=change, lens=lens, causal=causal)


def test_many_groups(dev):
    """Tiles of rows that end with their group."""
    mixed(dev, 16, 1, 8, 64, groups=[(200 + 16 * (g % 3), [g % 5 + 4, 9]) for g in range(70)], n=[4, 3] * 70, seed=2)


@pytest.mark.parametrize("T,H,G,D", SHAPES)
@pytest.mark.parametrize("qt,ot", [("b", "b"), ("f", "f")])
def test_few_rows_in_both(dev, T, H, G, D, qt, ot):
    mixed(dev, T, H, G, D, qt, ot, groups=[(130, OWN)], n=1, kernel=FEW, max_prefix=130, seed=D)


@pytest.mark.parametrize("qt", ["b", "f"])
def test_graph(dev, qt):
    """Replayed while the sequences grow; the same bits as eager calls, whatever
    the workspace held."""
    cache, table, kv, first, pt, plen = batch([(1090, [120 + b for b in range(20)]), (400, [140] * 20)], 16, 1, 128, 3)
    c = cache.to(dev)
    q = torch.from_numpy(synth.normal(7, (40, 8, 128))).to(dev).to(DT[qt])
    lens, cu = i32(kv - 100, dev), range(41)
    args = (i32(table, dev), lens, i32(cu, dev), i32(first, dev), i32(pt, dev), i32(plen, dev), 1, 200, 1 << 16, 0.1)
    need = capi.lib().lcml_fp8_attention_shared_workspace_bytes(40, 40, 2, 8, 1, 128, 1, 200, 1 << 16)
    ws, out = torch.empty(need, dtype=torch.uint8, device=dev), torch.empty_like(q)
    capi.kernel_trace()
    capi.attention_shared(q, *c, *args, out=out, workspace=ws)
    assert MIXED in ", ".join(capi.kernel_trace())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        capi.attention_shared(q, *c, *args, out=out, workspace=ws)
    for _ in range(4):
        lens.add_(19)
        q.neg_()
        want = capi.attention_shared(q, *c, *args)
        out.zero_()
        ws.fill_(255)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    dc.check_attention(out.double().cpu().numpy(), q.float().cpu().numpy(), cache, table, lens.cpu().numpy(), cu, 1, 0.1, qt == "b",
                       shared=(first, pt, plen))
