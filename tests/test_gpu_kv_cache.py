"""GPU parity of lcml_fp8_kv_cache_write / _read: scales and codes bit-exact
with the token-by-token CPU restatement (power-of-two scales leave one
rounding, the encoder's, in the definition; a zero's sign is left open), and
bytes of slots that hold no token of the call unchanged."""
import numpy as np
import pytest
import torch

from luisaml_amd import capi, synth
from tests import kv_cases as kc

pytestmark = pytest.mark.gpu


def i32(a, dev):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=dev)


def values(seed, shape, bf16):
    x = synth.normal(seed, shape) * np.exp(synth.normal(seed + 1, shape[-1:], std=0.5))
    return kc.bf16(x) if bf16 else x.astype(np.float32)


def run(dev, H, T, D, kv_len, n, bf16=True, seed=0, scale=1.0, mutate=None, table=None, max_q=None, strided=True):
    rng = np.random.default_rng(seed)
    kv_len, cu = np.array(kv_len), np.concatenate([[0], np.cumsum(n)])
    made, pages = kc.tables(kv_len, T, rng)
    table = made if table is None else table(made)
    cache = kc.Cache(pages, H, T, D, rng)
    k, v = values(seed + 5, (cu[-1], H, D), bf16) * np.float32(scale), values(seed + 9, (cu[-1], H, D), bf16)
    if mutate:
        mutate(k, v)
    c = cache.to(dev)
    dt = torch.bfloat16 if bf16 else torch.float32
    if strided:  # as the columns of a QKV projection that starts off its alignment
        qkv = torch.zeros(cu[-1], 2 * H * D + H * D + 1, dtype=dt, device=dev)
        kd, vd = (qkv[:, 1 + i * H * D:1 + (i + 1) * H * D].view(-1, H, D) for i in (1, 2))
        kd.copy_(torch.from_numpy(k))
        vd.copy_(torch.from_numpy(v))
    else:
        kd, vd = torch.from_numpy(k).to(dev).to(dt), torch.from_numpy(v).to(dev).to(dt)
    idx = (i32(table, dev), i32(kv_len, dev), i32(cu, dev))
    mq = max(list(n) + [1]) if max_q is None else max_q
    capi.kv_cache_write(kd, vd, *c, *idx, mq)
    cache.write(k, v, table, kv_len, cu)
    torch.cuda.synchronize()
    for w in (0, 1):
        assert np.array_equal(c[2 + w].cpu().numpy(), cache.scale[w]), "scales"
        assert kc.same_codes(c[w].cpu().numpy(), cache.packed(w)), "codes"
    for odt in (torch.float32, torch.bfloat16):
        ko, vo = (torch.full((cu[-1], H, D), 7.0, dtype=odt, device=dev) for _ in range(2))
        capi.kv_cache_read(*c, *idx, mq, ko, vo)
        torch.cuda.synchronize()
        for w, got in ((0, ko), (1, vo)):
            want = np.full((cu[-1], H, D), 7.0)
            for b in range(len(kv_len)):
                nb, L = cu[b + 1] - cu[b], kv_len[b]
                vals, there = cache.values(w, table[b], L)
                for i in range(nb):
                    p = L - nb + i
                    if 0 <= p and there[p]:
                        want[cu[b] + i] = vals[:, p]
            want = want.astype(np.float32)
            assert np.array_equal(got.float().cpu().numpy(), kc.bf16(want) if odt == torch.bfloat16 else want,
                                  equal_nan=True)
    return c, cache, idx


@pytest.mark.parametrize("T", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("D", [16, 48, 64, 80, 128, 256])
@pytest.mark.parametrize("bf16", [True, False])
def test_prompts_chunks_and_single_tokens(dev, T, D, bf16):
    run(dev, 2, T, D, [1, T, T + 1, 3 * T - 1, 300, 40], [1, T, 1, 2 * T, 133, 17], bf16, seed=T + D)


def test_many_heads_and_no_stride(dev):
    run(dev, 40, 16, 64, [5, 17, 33], [5, 2, 33], strided=False)


def test_empty_sequences_missing_tokens_and_pages(dev):
    """No new tokens; no tokens at all; more rows than positions; pages that
    are -1 or out of range; a table with too few columns."""
    def holes(t):
        t = t.copy()
        t[4, 1], t[5, 0] = -1, 10 ** 6
        return t[:, :4]
    run(dev, 3, 16, 64, [0, 20, 3, 0, 40, 20, 90], [0, 0, 5, 2, 40, 20, 60], seed=3, table=holes)


@pytest.mark.parametrize("T,D", [(256, 256), (128, 80), (64, 128)])
@pytest.mark.parametrize("n", [1, 3, 40])
def test_growth_behind_few_new_tokens(dev, T, D, n):
    """Far larger values at the end of pages that are nearly full: more units
    of earlier tokens to encode again than the call has threads."""
    H, L = 2, T - 2
    rng = np.random.default_rng(T + n)
    table, pages = kc.tables([L, L - 5], T, rng)
    cache = kc.Cache(pages, H, T, D, rng)
    c = cache.to(dev)
    for lens, cu, by in (([L - n, L - 5 - n], [0, L - n, 2 * (L - n) - 5], 1.0), ([L, L - 5], [0, n, 2 * n], 900.0)):
        k, v = values(T, (cu[-1], H, D), False) * np.float32(by), values(n, (cu[-1], H, D), False) * np.float32(by)
        capi.kv_cache_write(torch.from_numpy(k).to(dev), torch.from_numpy(v).to(dev), *c, i32(table, dev), i32(lens, dev),
                            i32(cu, dev), max(np.diff(cu)))
        cache.write(k, v, table, np.array(lens), np.array(cu))
        torch.cuda.synchronize()
        for w in (0, 1):
            assert np.array_equal(c[2 + w].cpu().numpy(), cache.scale[w])
            assert kc.same_codes(c[w].cpu().numpy(), cache.packed(w))


def test_tokens_one_by_one_grow_the_scale(dev):
    """A page filled token by token, each larger than the last: the codes that
    stay are encoded again whenever the scale grows."""
    H, T, D = 2, 16, 64
    rng = np.random.default_rng(4)
    table, pages = kc.tables([40], T, rng)
    cache = kc.Cache(pages, H, T, D, rng)
    c = cache.to(dev)
    for p in range(40):
        k = values(100 + p, (1, H, D), True) * np.float32(2.0 ** (p % 7 - 3))
        v = values(200 + p, (1, H, D), True) * np.float32(1.5 ** (p % 11))
        v = kc.bf16(v)
        kd, vd = (torch.from_numpy(x).to(dev).bfloat16() for x in (k, v))
        capi.kv_cache_write(kd, vd, *c, i32(table, dev), i32([p + 1], dev), i32([0, 1], dev), 1)
        cache.write(k, v, table, np.array([p + 1]), np.array([0, 1]))
    torch.cuda.synchronize()
    for w in (0, 1):
        assert np.array_equal(c[2 + w].cpu().numpy(), cache.scale[w])
        assert kc.same_codes(c[w].cpu().numpy(), cache.packed(w))


@pytest.mark.parametrize("scale", [0.0, 1e-44, 1e-38, 448.0 * 2.0 ** -126, 1e-20, 1.0, 1e30])
def test_scales_at_the_ends(dev, scale):
    run(dev, 2, 16, 32, [20, 33], [20, 33], bf16=False, seed=6, scale=scale)


def test_scale_boundary_infinities_and_nan(dev):
    """Maxima of 448 * 2^k exactly (that scale is enough) and one ulp more;
    infinities saturate and do not count; NaN stays NaN; -0 is 0."""
    def put(k, v):
        k[:16, 0], k[16:, 0] = 1.0, 2.0
        k[3, 0, 5] = 448.0 * 4
        k[20, 0, 5] = np.nextafter(np.float32(448.0 * 4), np.float32(1e9))
        v[3, 0, 1], v[4, 0, 2], v[5, 0, 3], v[6, 0, 4] = np.inf, -np.inf, np.nan, -0.0
        v[16:, 1] = np.inf
    _, cache, _ = run(dev, 2, 16, 32, [32], [32], bf16=False, seed=8, mutate=put)
    p = cache.scale[0][:, 0]
    assert 4.0 in p and 8.0 in p


def test_other_stream_and_graph(dev):
    """Single tokens by a captured graph, replayed on new lengths and rows:
    every replay equals the eager call on a copy."""
    H, T, D, B = 2, 16, 64, 3
    rng = np.random.default_rng(5)
    table, pages = kc.tables([60] * B, T, rng)
    cache = kc.Cache(pages, H, T, D, rng)
    c, e = cache.to(dev), cache.to(dev)
    k, v = (torch.zeros(B, H, D, dtype=torch.bfloat16, device=dev) for _ in range(2))
    idx = (i32(table, dev), i32([7, 20, 48], dev), i32(range(B + 1), dev))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        capi.kv_cache_write(k, v, *c, *idx, 1)
        capi.kv_cache_write(k, v, *e, *idx, 1)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        capi.kv_cache_write(k, v, *c, *idx, 1)
    for step in range(4):
        idx[1].add_(1)
        k.copy_(torch.from_numpy(values(step, (B, H, D), True)))
        v.copy_(torch.from_numpy(values(50 + step, (B, H, D), True)))
        g.replay()
        capi.kv_cache_write(k, v, *e, *idx, 1)
        torch.cuda.synchronize()
        for a, b in zip(c, e):
            assert torch.equal(a, b)


def test_cache_past_32_bit_offsets(dev):
    """Pages past 4 GiB in each cache: a page's bytes land in that page."""
    H, T, D = 8, 256, 256
    pages = (1 << 32) // (H * T * D) + 3
    c = capi.kv_cache(pages, H, T, D, dev)
    n = 300
    k, v = values(1, (n, H, D), True), values(2, (n, H, D), True)
    table = np.array([[pages - 1, pages - 2]], np.int32)
    idx = (i32(table, dev), i32([n], dev), i32([0, n], dev))
    kd, vd = (torch.from_numpy(x).to(dev).bfloat16() for x in (k, v))
    capi.kv_cache_write(kd, vd, *c, *idx, n)
    ko, vo = torch.empty_like(kd), torch.empty_like(vd)
    capi.kv_cache_read(*c, *idx, n, ko, vo)
    torch.cuda.synchronize()
    for got, x in ((ko, k), (vo, v)):
        # 4 significant bits, and steps of 2^-9 s below the normal codes
        err, s = np.abs(got.float().cpu().numpy() - x), np.abs(x).max() / 448.0 * 2
        assert (err <= np.maximum(np.abs(x) * 2.0 ** -4, s * 2.0 ** -10)).all()
    assert int(c[0][:pages - 2].count_nonzero()) == 0 and int(c[1][:pages - 2].count_nonzero()) == 0


def test_binding_checks_shapes_and_types(dev):
    """Tensors that do not fit each other: ValueError, nothing launched."""
    c = list(capi.kv_cache(3, 2, 16, 32, dev))
    idx = [i32([[0, 1]], dev), i32([5], dev), i32([0, 5], dev)]
    k = torch.zeros(5, 2, 32, device=dev)
    capi.kernel_trace()

    def bad(what, **kw):
        a = dict(k=k, v=k, kc=c[0], vc=c[1], ks=c[2], vs=c[3], table=idx[0], kv=idx[1], cu=idx[2])
        a.update(kw)
        with pytest.raises(ValueError, match=what):
            capi.kv_cache_write(*a.values(), 5)
    bad("k_cache", kc=c[0].int())
    bad("v_cache", vc=c[1][:2].contiguous())
    bad("k_cache", kc=c[0].transpose(1, 2))
    bad("scale", ks=c[2].double())
    bad("scale", vs=c[3][:, :1].contiguous())
    bad("block_table", table=idx[0].long())
    bad("kv_len", kv=i32([5, 5], dev))
    bad("cu_q", cu=i32([0], dev))
    bad("k:", k=k[:, :1])
    bad("v:", v=k.bfloat16())
    bad("k:", k=k.transpose(1, 2))
    with pytest.raises(capi.LcmlError):
        capi.kv_cache_write(k.half(), k.half(), *c, *idx, 5)
    with pytest.raises(ValueError, match="q:"):
        capi.attention(torch.zeros(5, 4, 16, device=dev), *c, *idx, 5, 5, 0.1)
    with pytest.raises(capi.LcmlError):
        capi.attention(torch.zeros(5, 3, 32, device=dev), *c, *idx, 5, 5, 0.1)
    assert capi.kernel_trace() == []
