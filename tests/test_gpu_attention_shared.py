"""GPU parity of attention behind shared prefixes with the 64-bit definition
over the same codes (decode_cases.check_attention)."""
import numpy as np
import pytest
import torch

from luisaml_amd import capi, synth
from tests import decode_cases as dc
from tests import kv_cases as kc
from tests.test_gpu_attention import DT, i32

pytestmark = pytest.mark.gpu


def batch(groups, T, H, D, seed, spread=1.0):
    """groups: [(prefix, [own tokens of each sequence])].  A cache, block tables
    that begin with the group's pages (a prefix that ends inside a page has a
    copy of that one for each sequence), lengths, and the groups' arrays."""
    rng = np.random.default_rng(seed)
    rows, prefixes, kv, first, order_at = [], [], [], [0], 0
    total = sum(-(-p // T) + sum(-(-(p + o) // T) - p // T for o in own) for p, own in groups) + 2
    order = rng.permutation(total)

    def take(k):
        nonlocal order_at
        order_at += k
        return list(order[order_at - k:order_at])
    for p, own in groups:
        pre = take(-(-p // T))
        prefixes.append(pre)
        for o in own:
            rows.append(pre[:p // T] + take(-(-(p + o) // T) - p // T))
            kv.append(p + o)
        first.append(len(kv))
    cols = max([len(r) for r in rows] + [1])
    table = np.full((len(rows), cols), -1, np.int32)
    for b, r in enumerate(rows):
        table[b, :len(r)] = r
    pt = np.full((len(groups), max([len(p) for p in prefixes] + [1])), -1, np.int32)
    for g, p in enumerate(prefixes):
        pt[g, :len(p)] = p
    cache = kc.Cache(total, H, T, D, rng)

    def fill(tab, start, n, s):
        if n <= start:
            return
        k = synth.normal(s, (n - start, H, D)) * np.exp(synth.normal(s + 1, (D,), std=0.4))
        v = synth.normal(s + 2, (n - start, H, D))
        if spread != 1.0:
            v = v * np.exp(np.log(spread) * (rng.random(((n - start) // 16 + 1, H, 1)) - 0.5)).repeat(16, 0)[:n - start]
        cache.write(k.astype(np.float32), v.astype(np.float32), tab[None], np.array([n]), np.array([0, n - start]))
    for g, (p, own) in enumerate(groups):
        fill(pt[g], 0, p, seed + 10 * g)
        for b in range(first[g], first[g + 1]):
            for w in (0, 1):  # the copies
                if p % T:
                    cache.codes[w][table[b, p // T]] = cache.codes[w][pt[g, p // T]]
                    cache.scale[w][table[b, p // T]] = cache.scale[w][pt[g, p // T]]
            fill(table[b], p, kv[b], seed + 1000 + 10 * b)
    return cache, table, np.array(kv), np.array(first), pt, np.array([p for p, _ in groups])


def run(dev, groups, n, T=16, H=2, G=2, D=64, qt="b", ot="b", causal=True, seed=0, spread=1.0, change=None, max_q=None,
        max_own=None, max_prefix=None, kernel=None, lens=None):
    cache, table, kv, first, pt, plen = batch(groups, T, H, D, seed, spread)
    kv = kv if lens is None else np.array(lens)
    n = [n] * len(kv) if isinstance(n, int) else n
    cu = np.concatenate([[0], np.cumsum(n)])
    q = synth.normal(seed + 7, (cu[-1], H * G, D)).astype(np.float32)
    q = kc.bf16(q) if qt == "b" else q
    if change:
        first, pt, plen = change(q, cache, table, kv, first, pt, plen)
    out = torch.full((cu[-1], H * G * D + 5), 9.0, dtype=DT[ot], device=dev)
    od = out[:, 3:3 + H * G * D].view(-1, H * G, D)
    mq = max(list(n) + [1]) if max_q is None else max_q
    mo = max([o for _, own in groups for o in own] + [1]) if max_own is None else max_own
    mp = max([p for p, _ in groups] + [0]) if max_prefix is None else max_prefix
    capi.kernel_trace()
    capi.attention_shared(torch.from_numpy(q).to(dev).to(DT[qt]), *cache.to(dev), i32(table, dev), i32(kv, dev), i32(cu, dev),
                          i32(first, dev), i32(np.asarray(pt).reshape(len(plen), -1) if len(plen) else np.zeros((0, 1)), dev),
                          i32(plen, dev), mq, mo, mp, D ** -0.5, causal=causal, out=od)
    torch.cuda.synchronize()
    if kernel:
        assert kernel in ", ".join(capi.kernel_trace())
    got = od.float().cpu().numpy().astype(np.float64)
    assert (out[:, :3] == 9.0).all() and (out[:, 3 + H * G * D:] == 9.0).all()
    dc.check_attention(got, q, cache, table, kv, cu, H, D ** -0.5, ot == "b", causal=causal, shared=(first, pt, plen))
    return got


OWN = [1, 2, 16, 17, 63, 64, 65, 130]
SHAPES = [(16, 2, 4, 128), (32, 1, 1, 64), (64, 2, 7, 128), (16, 3, 2, 80), (128, 1, 16, 64), (256, 1, 8, 256), (16, 1, 20, 96),
          (32, 2, 4, 16), (64, 1, 4, 192)]


@pytest.mark.parametrize("T,H,G,D", SHAPES)
@pytest.mark.parametrize("qt,ot", [("b", "b"), ("b", "f"), ("f", "f"), ("f", "b")])
def test_single_tokens(dev, T, H, G, D, qt, ot):
    run(dev, [(2 * T, OWN)], 1, T, H, G, D, qt, ot, seed=T + D + G)


@pytest.mark.parametrize("T,H,G,D", SHAPES)
@pytest.mark.parametrize("qt,ot", [("b", "b"), ("b", "f"), ("f", "f"), ("f", "b")])
def test_many_rows_of_each(dev, T, H, G, D, qt, ot):
    """Rows enough for the kernel for many, in both parts."""
    run(dev, [(2 * T, [130, 70]), (T, [130])], [130, 64, 129], T, H, G, D, qt, ot, seed=T + D + G, max_q=1 << 15, max_prefix=1 << 14,
        kernel="attention_many, attention_join")


@pytest.mark.parametrize("prefix", [1, 15, 16, 17, 31, 63, 64, 65, 100, 128, 200])
@pytest.mark.parametrize("n", [1, 4])
def test_prefixes_of_any_length(dev, prefix, n):
    """Ends inside pages (of which each sequence has a copy) and steps."""
    run(dev, [(prefix, [4, 5, 17, 80])], n, 16, 1, 4, 64, seed=prefix)


def test_groups(dev):
    """Of different sizes and lengths, one sequence alone, one group without a
    prefix, sequences that belong to none, an empty group."""
    def change(q, cache, table, kv, first, pt, plen):
        return np.array([0, 3, 3, 4, 6]), np.concatenate([pt[:1], pt[:1], pt[1:]])[:4], np.array([plen[0], 50, plen[1], 0])
    run(dev, [(64, [3, 20, 40]), (100, [5]), (48, [7, 9]), (32, [11, 1])], 1, 16, 2, 4, 64, change=change)
    run(dev, [(64, [3, 20, 40]), (100, [5]), (48, [7, 9]), (32, [11, 1])], [2, 0, 3, 5, 1, 1, 4, 1], 16, 2, 4, 64, change=change)


@pytest.mark.parametrize("groups", [65, 130])
def test_more_groups_than_lanes(dev, groups):
    run(dev, [(16 * (g % 3 + 1), [g % 5 + 1, 3]) for g in range(groups)], 1, 16, 1, 2, 32, seed=groups)


@pytest.mark.parametrize("n", [1, 40])
def test_sequences_outside_groups_and_rows_out_of_range(dev, n):
    """A first group that does not begin at the first sequence; one that ends past
    the last; a sequence whose rows pass the batch's counts as none, and its
    group's others are as they were."""
    def change(q, cache, table, kv, first, pt, plen):
        return np.array([1, 3, 9]), np.concatenate([pt[:1], pt[:1]]), np.array([64, 64])
    run(dev, [(64, [40, 50, 41, 70, 45])], n, 16, 1, 4, 64, change=change)
    cache, table, kv, first, pt, plen = batch([(64, [40, 50, 41])], 16, 1, 64, 0)
    q = torch.from_numpy(synth.normal(7, (2 * n, 4, 64))).to(dev)
    out = torch.full_like(q, 5.0)
    capi.attention_shared(q, *cache.to(dev), i32(table, dev), i32(kv, dev), i32([0, n, 2 * n, 2 * n + 3], dev), i32(first, dev),
                          i32(pt, dev), i32(plen, dev), n, 50, 64, 0.125, out=out)
    torch.cuda.synchronize()
    dc.check_attention(out.double().cpu().numpy(), q.cpu().numpy(), cache, table[:2], kv[:2], [0, n, 2 * n], 1, 0.125, False,
                       shared=(first, pt, plen))


def test_no_groups(dev):
    def change(q, cache, table, kv, first, pt, plen):
        return np.array([0]), np.zeros((0, 1)), np.array([], dtype=np.int32)
    run(dev, [(64, [3, 20, 40])], 1, change=change)
    run(dev, [(64, [3, 200, 400])], 1, change=change, max_own=500)
    run(dev, [(64, [3, 200, 400])], [3, 100, 130], change=change, max_own=500, max_q=1 << 15, kernel="attention_many, attention_join")


def test_rows_that_do_not_lie_behind_the_prefix(dev):
    """Rows inside it (a sequence just being prefilled), lengths below it, none
    at all, and a prefix of negative length: their own tables throughout."""
    run(dev, [(64, [3, 20, 40, 8])], [3, 21, 70, 8], 16, 1, 4, 64)
    got = run(dev, [(64, [3, 20, 40, 8])], [1, 2, 1, 70], 16, 1, 4, 64, lens=[0, 50, 64, 72])
    assert (got[0] == 0).all()
    run(dev, [(64, [3, 20, 40, 8])], [1, 64, 1, 8], 16, 1, 4, 64, lens=[65, 64, 104, 72])

    def negative(q, cache, table, kv, first, pt, plen):
        return first, pt, -plen
    run(dev, [(64, [3, 20])], 1, change=negative)


@pytest.mark.parametrize("n", [1, 40])
def test_missing_pages(dev, n):
    """Pages that are not there, in the prefix and in the own tokens; all of a
    prefix's; a prefix table with too few columns."""
    def change(q, cache, table, kv, first, pt, plen):
        table[1, 5], pt[0, 1], pt[1, :] = -1, 10 ** 6, -1
        table[4, :] = -1
        return first, pt[:, :3], plen
    got = run(dev, [(64, [60, 70, 50]), (64, [41, 42])], n, 16, 1, 4, 64, change=change)
    assert (got[-1] == 0).all()


def test_not_causal(dev):
    run(dev, [(64, [30, 20, 40])], [30, 1, 4], 16, 2, 2, 64, causal=False)
    run(dev, [(64, [30, 20, 40])], [100, 85, 4], 16, 2, 2, 64, causal=False)  # rows inside the prefix, and before it


@pytest.mark.parametrize("D", [64, 80, 256])
@pytest.mark.parametrize("n", [1, 40])
def test_nan_codes_and_queries(dev, D, n):
    def change(q, cache, table, kv, first, pt, plen):
        cache.codes[1][pt[0, 1], :, 2, 5] = kc.NAN_CODE      # a prefix
        cache.codes[1][table[2, 4], :, 0, 7] = kc.NAN_CODE   # own tokens
        q[0, 0, 3] = np.nan
        return first, pt, plen
    got = run(dev, [(64, [60, 70]), (64, [41, 42])], n, 16, 1, 4, D, change=change)
    assert np.isnan(got[:2 * n, :, 5]).all() and not np.isnan(got[2 * n:, :, 5]).any()
    assert np.isnan(got[3 * n - 1, :, 7]).all() and not np.isnan(got[3 * n:, :, 7]).any()


@pytest.mark.parametrize("ot", ["b", "f"])
@pytest.mark.parametrize("n", [1, 50])
def test_scales_far_apart(dev, ot, n):
    run(dev, [(128, [100, 200])], n, 16, 1, 4, 64, "b", ot, seed=9, spread=1e8)


@pytest.mark.parametrize("n,P,own", [(1, 5000, [10, 3000]), (1, 20000, [5, 1, 40]), (3, 9000, [100, 3]), (40, 4000, [1000, 40])])
@pytest.mark.parametrize("ot", ["b", "f"])
def test_long_ones(dev, n, P, own, ot):
    """Lengths at which a row has many parts of either."""
    run(dev, [(P // 64 * 64, own)], n, 64, 1, 4, 64, "b", ot, seed=n)


@pytest.mark.parametrize("max_own,max_prefix", [(1, 1), (0, 0), (100000, 1), (1, 100000), (100000, 100000)])
def test_bounds_of_the_host_hold(dev, max_own, max_prefix):
    run(dev, [(256, [100, 300]), (128, [7])], 1, max_own=max_own, max_prefix=max_prefix)
    run(dev, [(256, [100, 300]), (128, [37])], 30, max_own=max_own, max_prefix=max_prefix, max_q=200)


def test_rows_past_max_q_are_left_out(dev):
    """As in attention(): the rest as it is without them."""
    cache, table, kv, first, pt, plen = batch([(64, [30, 20])], 16, 1, 64, 0)
    q = torch.from_numpy(synth.normal(7, (20, 4, 64))).to(dev)
    idx = (i32(table, dev), i32(kv, dev), i32([0, 10, 20], dev), i32(first, dev), i32(pt, dev), i32(plen, dev))
    full = capi.attention_shared(q, *cache.to(dev), *idx, 10, 30, 64, 0.125)
    out = torch.full_like(q, 5.0)
    capi.attention_shared(q, *cache.to(dev), *idx, 4, 30, 64, 0.125, out=out)
    torch.cuda.synchronize()
    assert (out[4:10] == 5).all() and (out[14:] == 5).all()
    o, mass, reach = dc.attention(q.cpu().numpy(), cache, table, kv, [0, 10, 20], 1, 0.125, shared=(first, pt, plen))
    bound = kc.attention_bound(mass, reach, 64, int(kv.max()), False)
    for got, rows in ((full, np.r_[0:20]), (out, np.r_[0:4, 10:14])):
        assert not kc.outside(got.double().cpu().numpy(), o, bound, False)[rows].any()


def test_same_bits_twice_graph_and_strided_prefix_table(dev):
    """Groups as rows of the block table itself; a graph replayed while the
    sequences grow; the same bits each time."""
    cache, table, kv, first, pt, plen = batch([(64, [130, 140]), (32, [120, 110])], 16, 2, 64, 3)
    c = cache.to(dev)
    q = torch.from_numpy(synth.normal(7, (4, 8, 64))).to(dev).bfloat16()
    tab, lens, cu = i32(table, dev), i32(kv - 100, dev), i32(range(5), dev)
    args = (tab, lens, cu, i32(first, dev), tab[::2, :4], i32(plen, dev), 1, 1000, 1000, 0.125)
    need = capi.lib().lcml_fp8_attention_shared_workspace_bytes(4, 4, 2, 8, 2, 64, 1, 1000, 1000)
    ws, out = torch.empty(need, dtype=torch.uint8, device=dev), torch.empty_like(q)
    capi.attention_shared(q, *c, *args, out=out, workspace=ws)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        capi.attention_shared(q, *c, *args, out=out, workspace=ws)
    for step in range(5):
        lens.add_(19)
        q.neg_()
        want = capi.attention_shared(q, *c, *args)
        out.zero_()
        ws.fill_(255)  # NaN wherever it is read before it is written
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        dc.check_attention(out.float().cpu().numpy().astype(np.float64), q.float().cpu().numpy(), cache, table, lens.cpu().numpy(),
                           range(5), 2, 0.125, True, shared=(first, table[::2, :4], plen))


def test_equals_attention_over_the_same_cache(dev):
    """A long prefix and many rows: within both results' bounds of each other."""
    cache, table, kv, first, pt, plen = batch([(2048, [40, 300, 1, 77, 64, 500, 10, 20])], 64, 2, 128, 5)
    c = cache.to(dev)
    q = torch.from_numpy(synth.normal(9, (8, 16, 128))).to(dev)
    idx = (i32(table, dev), i32(kv, dev), i32(range(9), dev))
    a = capi.attention(q, *c, *idx, 1, int(kv.max()), 128 ** -0.5)
    b = capi.attention_shared(q, *c, *idx, i32(first, dev), i32(pt, dev), i32(plen, dev), 1, 500, 2048, 128 ** -0.5)
    torch.cuda.synchronize()
    o, mass, reach = kc.attention(q.cpu().numpy(), cache, table, kv, range(9), 2, float(np.float32(128 ** -0.5)))
    bound = kc.attention_bound(mass, reach, 128, int(kv.max()), False)
    for got in (a, b):
        assert not kc.outside(got.double().cpu().numpy(), o, bound, False).any()
