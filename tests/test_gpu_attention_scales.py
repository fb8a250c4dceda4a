"""Attention over V pages whose scales lie far apart, or at the ends of fp32's
range: a row's result is the definition's whatever the scales of pages that it
does not see or hardly weighs.  Tolerance: kv_cases.attention_bound, but with
fp32's own steps below 2^-126 in the place of its absolute term."""
import numpy as np
import pytest
import torch

from luisaml_amd import capi, synth
from tests import kv_cases as kc

pytestmark = pytest.mark.gpu
DT = {"f": torch.float32, "b": torch.bfloat16}
TYPES = [("b", "b"), ("b", "f"), ("f", "f"), ("f", "b")]
MANY = 1 << 15  # a max_q far above the true one takes the kernel for many rows


def run(dev, kv_len, n, size, T=16, H=2, G=2, D=64, qt="b", ot="b", window=0, causal=True, seed=0, lean=None, many=False,
        change=None, q_scale=1.0):
    """size(b, pos): V's size at each position of sequence b; lean(b, pos): what
    is added to the tokens' scores, in units of the scale."""
    rng = np.random.default_rng(seed)
    table, pages = kc.tables(kv_len, T, rng)
    cache = kc.Cache(pages, H, T, D, rng)
    cu = np.concatenate([[0], np.cumsum(kv_len)])
    k, v = synth.normal(seed + 1, (cu[-1], H, D)), synth.normal(seed + 3, (cu[-1], H, D))
    rows = np.concatenate([[0], np.cumsum(n)])
    q = synth.normal(seed + 7, (rows[-1], H * G, D)).astype(np.float32) * np.float32(q_scale)
    scale = float(np.float32(D ** -0.5))
    if lean:  # the first element carries it
        q[:, :, 0] = 1.0
        k[:, :, 0] = np.concatenate([lean(b, np.arange(L)) for b, L in enumerate(kv_len)])[:, None] / scale
    v = v * np.concatenate([size(b, np.arange(L)) for b, L in enumerate(kv_len)])[:, None, None]
    q = kc.bf16(q) if qt == "b" else q
    cache.write(k.astype(np.float32), v.astype(np.float32), table, np.array(kv_len), cu)
    if change:
        change(cache, table)
    c = cache.to(dev)
    idx = tuple(torch.tensor(np.asarray(a), dtype=torch.int32, device=dev) for a in (table, kv_len, rows))
    qd = torch.from_numpy(q).to(dev).to(DT[qt])
    capi.kernel_trace()
    out = capi.attention(qd, *c, *idx, MANY if many else max(n), max(kv_len), scale, causal=causal, window=window, out_dtype=DT[ot])
    torch.cuda.synchronize()
    assert ("attention_many" in ", ".join(capi.kernel_trace())) == many
    got = out.float().cpu().numpy().astype(np.float64)
    o, mass, reach = kc.attention(q, cache, table, kv_len, rows, H, scale, causal, window)
    bound = kc.attention_bound(mass, reach, D, max(kv_len), ot == "b") - 1e-37 + 2.0 ** -147
    assert np.array_equal(np.isnan(got), np.isnan(o))
    bad = kc.outside(got, o, bound, ot == "b")
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], o[bad][:5], bound[bad][:5])
    return got


def steps(*sizes, every=16):
    """A size for each run of `every` tokens, the last one for the rest."""
    s = np.array(sizes)
    return lambda b, pos: s[np.minimum(pos // every, len(s) - 1)]


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("qt,ot", TYPES)
@pytest.mark.parametrize("D", [64, 80, 128, 256])
def test_large_page_before_the_window(dev, D, qt, ot, many):
    """The window hides a page of V near 1; what is seen is near 1e-13."""
    got = run(dev, [64, 100], [1, 5], steps(1.0, 1e-13), D=D, qt=qt, ot=ot, window=16, many=many, seed=D)
    assert 0 < np.abs(got).max() < 1e-11


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("ot", ["b", "f"])
@pytest.mark.parametrize("D", [64, 80, 128, 256])
def test_larger_pages_after_a_row(dev, D, ot, many):
    """A prompt whose later pages are larger, by more and more: early rows see
    none of them."""
    got = run(dev, [96, 200], [96, 200], steps(1e-12, 1e-8, 1.0, 1e3, 1e20, 1e30), D=D, ot=ot, many=many, seed=D)
    assert 0 < np.abs(got[:16]).max() < 1e-10


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("qt,ot", TYPES)
@pytest.mark.parametrize("T", [16, 64, 256])
def test_scales_in_any_order(dev, T, qt, ot, many):
    """Sizes from 1e-35 to 1e30, page by page: rising, falling and at random;
    lengths that end inside a step, a page and a block."""
    r = np.random.default_rng(T)
    for size in (np.geomspace(1e-35, 1e30, 24), np.geomspace(1e30, 1e-35, 24), 10.0 ** r.uniform(-35, 30, 24)):
        run(dev, [900, 333, 1], [40, 7, 1], steps(*size, every=T if T < 64 else 40), T=T, G=4, qt=qt, ot=ot, many=many, seed=T)


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("ot", ["b", "f"])
@pytest.mark.parametrize("spread", [2.0 ** 9, 2.0 ** 11, 2.0 ** 20, 2.0 ** 40, 2.0 ** 80])
def test_weights_that_undo_the_sizes(dev, spread, ot, many):
    """Every other page is larger by `spread` and its scores are lower by
    ln(spread), or all but hidden by it: both kinds count in one, only the small
    one in the other."""
    def size(b, pos):
        return np.where(pos // 16 % 2, spread, 1.0) * 1e-6
    for by in (np.log(spread), 2 * np.log(spread) + 12):
        run(dev, [300, 150], [20, 1], size, lean=lambda b, pos: np.where(pos // 16 % 2, -by, 0.0), qt="f", ot=ot, many=many, G=4)


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("ot", ["b", "f"])
@pytest.mark.parametrize("size", [2e-38, 1e-36, 1e-30, 1e30, 1e36])
def test_ends_of_the_range(dev, size, ot, many):
    """All pages near the smallest scale or near the largest, and long enough to
    be split and joined."""
    got = run(dev, [60, 2500], [6, 2], steps(size), T=32, ot=ot, many=many, seed=5)
    assert np.abs(got).max() > 0.0


@pytest.mark.parametrize("many", [False, True])
def test_large_scale_of_a_page_that_shows_zeros(dev, many):
    """A page's scale comes from a token that is not seen; what is seen of it is
    zeros, and the other pages are small."""
    def size(b, pos):
        return np.where(pos == 0, 1e20, np.where(pos < 16, 0.0, 1e-15))
    got = run(dev, [80], [3], size, window=70, ot="f", many=many)
    assert 0 < np.abs(got).max() < 1e-13


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("window", [0, 40])
def test_nan_codes_among_far_scales(dev, window, many):
    def change(cache, table):
        cache.codes[1][table[0, 1], :, 2, 5] = kc.NAN_CODE  # position 18
    got = run(dev, [130], [40], steps(1.0, 1e-9, 1e9, 1e-20), window=window, many=many, change=change, ot="f")
    assert np.isnan(got[0, :, 5]).all() == (window == 0 or 130 - 40 - window < 18) and not np.isnan(got[:, :, 6]).any()
    if window:
        assert not np.isnan(got[-1]).any()


@pytest.mark.parametrize("many", [False, True])
def test_missing_pages_among_far_scales(dev, many):
    def change(cache, table):
        table[0, 2], table[0, 5] = -1, 10 ** 6
    run(dev, [150, 100], [50, 100], steps(1.0, 1e-9, 1e9, 1e-20, 1.0, 1e15), many=many, change=change, ot="f")


@pytest.mark.parametrize("n,D", [(1, 64), (2, 128), (300, 128)])
@pytest.mark.parametrize("ot", ["b", "f"])
def test_split_over_long_sequences(dev, n, D, ot):
    """Parts whose pages are of one size, and of many, joined."""
    r = np.random.default_rng(n)
    size = 10.0 ** r.uniform(-20, 10, 400)
    run(dev, [5000, 3000], [n, n], steps(*size, every=64), T=64, H=1, G=4, D=D, ot=ot, many=n == 300, seed=n)
    run(dev, [5000, 3000], [n, n], steps(1.0, 1e-10, every=2500), T=64, H=1, G=4, D=D, ot=ot, many=n == 300, seed=n)


@pytest.mark.parametrize("ot", ["b", "f"])
@pytest.mark.parametrize("kv,n,D,many", [([20000], 1, 64, False), ([5000, 3000], 300, 128, True), ([700], 3, 64, False),
                                         ([3000, 2000], 150, 64, False)])
def test_parts_near_the_largest_number_joined(dev, kv, n, D, many, ot):
    """Every value is 448 times 2^119, 7/8 of fp32's range: so is the result,
    however many parts it is joined from."""
    def change(cache, table):
        cache.codes[1][:] = 0x7E
        cache.scale[1][:] = 2.0 ** 119
    got = run(dev, kv, [n] * len(kv), steps(1.0), T=64, H=1, G=4, D=D, ot=ot, many=many, change=change)
    assert (np.abs(got / (448.0 * 2.0 ** 119) - 1.0) < 1e-5).all()
