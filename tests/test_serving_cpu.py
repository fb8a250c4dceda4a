"""Refusals of the norm, KV cache and attention entry points: the documented
status codes before the device is touched, and the no-op sizes.  And the
plain restatements that the GPU tests compare with, against each other."""
import numpy as np
import pytest

from luisaml_amd import capi
from tests import kv_cases as kc

P = 0x1000
BAD, UNS = capi.ERR_INVALID_ARG, capi.ERR_UNSUPPORTED


def norm(**kw):
    a = dict(M=4, H=64, x=P, xt=16, ldx=64, r=P, ro=P, rt=1, ldr=64, ldro=64, gamma=P, eps=1e-5, y=P, ldy=64, mode=2,
             scale=P, ws=None, wsb=0, stream=None)
    a.update(kw)
    return capi.lib().lcml_fp8_rms_norm(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(M=-1), BAD), (dict(H=0), BAD), (dict(xt=10), UNS), (dict(rt=17), UNS), (dict(mode=3), BAD), (dict(eps=-1.0), BAD),
    (dict(eps=float("nan")), BAD), (dict(ldx=63), BAD), (dict(ldy=60), BAD), (dict(ldr=1), BAD), (dict(ldro=1), BAD),
    (dict(r=None), BAD), (dict(x=None), BAD), (dict(gamma=None), BAD), (dict(y=None), BAD), (dict(scale=None), BAD),
    (dict(x=P + 1), BAD), (dict(r=P + 2), BAD), (dict(gamma=P + 2), BAD), (dict(mode=1), BAD),
    (dict(mode=1, ws=P, wsb=100), BAD), (dict(M=1 << 31), UNS), (dict(H=1 << 31, ldx=1 << 31, ldy=1 << 31, ldr=1 << 31,
                                                                     ldro=1 << 31), UNS)])
def test_norm_refusals(kw, code):
    assert norm(**kw) == code, capi.last_error()
    assert "rms_norm" in capi.last_error()


def test_norm_no_ops_and_workspace():
    assert norm(M=0, x=None, y=None) == capi.OK
    f = capi.lib().lcml_fp8_rms_norm_workspace_bytes
    assert f(8, 64, capi.SCALE_ROW) == 0 and f(1, 64, capi.SCALE_TENSOR) == 0 and f(8, 64, capi.SCALE_TENSOR) > 0


CACHE = dict(kc=P, vc=P, ks=P, vs=P, pages=8, heads=2, dim=64, page=16, table=P, ts=4, tc=4, kv=P, cu=P, seqs=2, mq=4)


def write(**kw):
    a = dict(k=P, v=P, dt=16, tokens=8, kt=128, kh=64, vt=128, vh=64, **CACHE, stream=None)
    a.update(kw)
    return capi.lib().lcml_fp8_kv_cache_write(*a.values())


def read(**kw):
    a = dict(**CACHE, k=P, v=P, dt=16, tokens=8, kt=128, kh=64, vt=128, vh=64, stream=None)
    a.update(kw)
    return capi.lib().lcml_fp8_kv_cache_read(*a.values())


def attend(**kw):
    a = dict(q=P, qd=16, tokens=8, qh=4, qt=256, qs=64, o=P, od=1, ot=256, os=64, **CACHE, mk=64, scale=0.1, causal=1,
             window=0, ws=P, wsb=1 << 40, stream=None)
    a.update(kw)
    return capi.lib().lcml_fp8_attention(*a.values())


SHARED = [(dict(dim=0), UNS), (dict(dim=24), UNS), (dict(dim=272), UNS), (dict(page=8), UNS), (dict(page=48), UNS),
          (dict(page=512), UNS), (dict(heads=0), BAD), (dict(seqs=-1), BAD), (dict(mq=-1), BAD), (dict(pages=-1), BAD),
          (dict(ts=3), BAD), (dict(table=None), BAD), (dict(kv=None), BAD), (dict(cu=None), BAD), (dict(kc=None), BAD),
          (dict(vs=None), BAD), (dict(kc=P + 8), BAD), (dict(vc=P + 8), BAD), (dict(ks=P + 2), BAD), (dict(kv=P + 2), BAD),
          (dict(tokens=-1), BAD), (dict(tokens=1 << 31), UNS), (dict(pages=1 << 31), UNS)]


@pytest.mark.parametrize("kw,code", SHARED)
def test_cache_refusals(kw, code):
    for fn in (write, read, attend):
        assert fn(**kw) == code, (fn.__name__, capi.last_error())
        assert "lcml_fp8_" in capi.last_error()


@pytest.mark.parametrize("kw,code", [(dict(dt=10), UNS), (dict(k=None), BAD), (dict(v=None), BAD), (dict(k=P + 1), BAD),
                                     (dict(seqs=1 << 20, mq=1 << 20), UNS)])
def test_write_and_read_refusals(kw, code):
    for fn in (write, read):
        assert fn(**kw) == code, capi.last_error()


@pytest.mark.parametrize("kw,code", [(dict(qd=10), UNS), (dict(od=17), UNS), (dict(q=None), BAD), (dict(o=None), BAD),
                                     (dict(q=P + 1), BAD), (dict(o=P + 2), BAD), (dict(qh=3), BAD), (dict(qh=0), BAD),
                                     (dict(scale=0.0), BAD), (dict(scale=-1.0), BAD), (dict(scale=float("inf")), BAD),
                                     (dict(scale=float("nan")), BAD), (dict(window=-1), BAD), (dict(mk=-1), BAD),
                                     (dict(mk=1 << 31), UNS)])
def test_attention_refusals(kw, code):
    assert attend(**kw) == code, capi.last_error()


def test_no_ops():
    for fn in (write, read, attend):
        for kw in (dict(tokens=0), dict(seqs=0), dict(mq=0)):
            assert fn(**kw) == capi.OK, capi.last_error()
    assert write(pages=0, kc=None, vc=None, ks=None, vs=None) == capi.OK
    assert capi.lib().lcml_fp8_attention_workspace_bytes(0, 1, 4, 2, 64, 1, 64) == 0


def test_page_scale_is_the_smallest():
    for a in (1.0, 447.9, 448.0, 448.1, 3e38, 1e-30, 2.0 ** -118, 7 * 2.0 ** -3):
        s = kc.page_scale(np.array([a, -a / 2]))
        assert a <= 448.0 * s and (s == 2.0 ** -126 or a > 448.0 * s / 2)
    assert kc.page_scale(np.array([0.0, np.inf, np.nan])) == 2.0 ** -126


def test_plain_cache_holds_what_was_written():
    """Written in two calls or in one, a page that starts with its largest
    token holds the same codes; values come back within half a code step."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((40, 2, 32)).astype(np.float32)
    x[0] *= 4
    x[16] *= 4
    x[32] *= 4
    caches = []
    for cuts in ([0, 40], [0, 5, 20, 40]):
        c = kc.Cache(4, 2, 16, 32, np.random.default_rng(1))
        for a, b in zip(cuts, cuts[1:]):
            c.write(x[a:b], x[a:b], np.array([[2, 0, 3]]), np.array([b]), np.array([0, b - a]))
        caches.append(c)
    got = [c.values(0, np.array([2, 0, 3]), 40)[0] for c in caches]
    assert np.array_equal(got[0], got[1])
    err = np.abs(got[0].transpose(1, 0, 2) - x)
    s = max(float(c) for c in caches[0].scale[0][[2, 0, 3]].reshape(-1))
    assert (err <= np.maximum(np.abs(x) * 2.0 ** -4, s * 2.0 ** -10)).all()


def test_plain_attention_of_one_token_is_its_value():
    c = kc.Cache(2, 1, 16, 16, np.random.default_rng(2))
    x = np.random.default_rng(3).standard_normal((1, 1, 16)).astype(np.float32)
    c.write(x, x, np.array([[1]]), np.array([1]), np.array([0, 1]))
    o, mass, reach = kc.attention(x.repeat(4, 1), c, np.array([[1]]), [1], [0, 1], 1, 0.25)
    v = c.values(1, np.array([1]), 1)[0][0]
    assert np.allclose(o[0], v.repeat(4, 0)) and np.allclose(mass, np.abs(o))


def test_binding_refuses_what_it_cannot_check():
    """Host tensors, wrong types and shapes: ValueError before any call."""
    import torch
    x, g = torch.zeros(2, 8), torch.ones(8)
    out, s = torch.zeros(2, 8, dtype=torch.uint8), torch.ones(2)
    with pytest.raises(ValueError, match="device tensor"):
        capi.rms_norm(x, g, 1e-5, mode=capi.SCALE_ROW, scale=s, out=out, stream=0)
    with pytest.raises(ValueError, match="tensor is expected"):
        capi.rms_norm(None, g, 1e-5, mode=capi.SCALE_ROW, scale=s, out=out, stream=0)
    with pytest.raises(ValueError, match="scale"):
        capi.rms_norm(x, g, 1e-5, mode=capi.SCALE_STATIC, out=out, stream=0)
    with pytest.raises(ValueError, match="number of arguments"):
        capi._binding().attention(x)
    c = [torch.zeros(1)] * 7
    for call in (lambda: capi.kv_cache_write(x, x, *c, 1, stream=0), lambda: capi.kv_cache_read(*c, 1, x, x, stream=0),
                 lambda: capi.attention(torch.zeros(1, 2, 16), *c, 1, 1, 0.1, out=x, workspace=x, stream=0)):
        with pytest.raises(ValueError, match="device tensor"):
            call()
