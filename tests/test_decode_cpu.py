"""Refusals of the plan, rotation, sinks and shared-prefix entry points: the
documented status codes before the device is touched, and the no-op sizes; what
their binding refuses; the plain restatements that the GPU tests compare with."""
import numpy as np
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from luisaml_amd import capi
from tests import decode_cases as dc
from tests import kv_cases as kc

P = 0x1000
BAD, UNS = capi.ERR_INVALID_ARG, capi.ERR_UNSUPPORTED


def plan(**kw):
    a = dict(n=P, held=P, ended=P, own=P, seqs=4, free=P, count=P, pages=8, page=16, table=P, ts=4, tc=4, kv=P, cu=P, left=P,
             pos=P, slots=P, tokens=10 ** 6, ws=None, wsb=0, stream=None)
    a.update(kw)
    return capi.lib().lcml_fp8_kv_cache_plan(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(seqs=-1), BAD), (dict(pages=-1), BAD), (dict(tc=-1), BAD), (dict(tokens=-1), BAD), (dict(page=8), UNS), (dict(page=48), UNS),
    (dict(page=512), UNS), (dict(page=0), UNS), (dict(seqs=2 ** 31 - 1), UNS), (dict(pages=2 ** 31), UNS), (dict(tc=2 ** 31, ts=2 ** 31), UNS),
    (dict(tokens=2 ** 31), UNS), (dict(ts=3), BAD), (dict(n=None), BAD), (dict(held=None), BAD), (dict(kv=None), BAD),
    (dict(table=None), BAD), (dict(free=None), BAD), (dict(count=None), BAD), (dict(cu=None), BAD), (dict(left=None), BAD),
    (dict(n=P + 2), BAD), (dict(ended=P + 1), BAD), (dict(own=P + 1), BAD), (dict(table=P + 2), BAD), (dict(pos=P + 2), BAD),
    (dict(slots=P + 4), BAD), (dict(), BAD), (dict(ws=P, wsb=47), BAD), (dict(ws=P + 4, wsb=1000), BAD)])
def test_plan_refusals(kw, code):
    assert plan(**kw) == code, capi.last_error()
    assert "kv_cache_plan" in capi.last_error()


def test_plan_workspace():
    f = capi.lib().lcml_fp8_kv_cache_plan_workspace_bytes
    assert f(4, 10) == 0 and f(4, 10 ** 6) == 48 and f(5000, 0) == 5002 * 8 and f(-1, 5) == 0


def rope(**kw):
    a = dict(q=P, k=P, dt=16, tokens=4, qh=4, kh=2, dim=64, qt=256, qs=64, kt=128, ks=64, gq=P, gk=P, eps=1e-6, pos=P, table=P,
             rows=10, rot=64, inter=0, qo=P, ko=P, ot=1, qot=256, qos=64, kot=128, kos=64, stream=None)
    a.update(kw)
    return capi.lib().lcml_fp8_qk_norm_rope(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(dt=10), UNS), (dict(ot=17), UNS), (dict(tokens=-1), BAD), (dict(qh=-1), BAD), (dict(kh=-1), BAD), (dict(rows=-1), BAD),
    (dict(dim=8), UNS), (dict(dim=72), UNS), (dict(dim=272), UNS), (dict(rot=-2), BAD), (dict(rot=63), BAD), (dict(rot=66), BAD),
    (dict(eps=-1.0), BAD), (dict(eps=float("nan")), BAD), (dict(qh=65536), UNS), (dict(tokens=2 ** 31), UNS), (dict(rows=2 ** 31), UNS),
    (dict(tokens=2 ** 26), UNS), (dict(q=None), BAD), (dict(k=None), BAD), (dict(qo=None), BAD), (dict(ko=None), BAD),
    (dict(q=P + 1), BAD), (dict(ko=P + 2), BAD), (dict(pos=None), BAD), (dict(table=None), BAD), (dict(gq=P + 2), BAD),
    (dict(gk=P + 2), BAD), (dict(pos=P + 2), BAD), (dict(table=P + 2), BAD)])
def test_rope_refusals(kw, code):
    assert rope(**kw) == code, capi.last_error()
    assert "qk_norm_rope" in capi.last_error()


def test_rope_no_ops():
    assert rope(tokens=0, q=None) == capi.OK and rope(qh=0, kh=0, q=None, k=None) == capi.OK


CACHE = dict(kc=P, vc=P, ks=P, vs=P, pages=8, heads=2, dim=64, page=16, table=P, ts=4, tc=4, kv=P, cu=P, seqs=2)


def sinks(**kw):
    a = dict(q=P, qd=16, tokens=8, qh=4, qt=256, qs=64, o=P, od=1, ot=256, os=64, **CACHE, mq=4, mk=64, scale=0.1, causal=1, window=8,
             sinks=4, ws=P, wsb=1 << 40, stream=None)
    a.update(kw)
    return capi.lib().lcml_fp8_attention_sinks(*a.values())


def shared(**kw):
    a = dict(q=P, qd=16, tokens=8, qh=4, qt=256, qs=64, o=P, od=1, ot=256, os=64, **CACHE, gs=P, pt=P, ps=4, pc=4, pl=P, groups=1, mq=4,
             mk=64, mp=64, scale=0.1, causal=1, ws=P, wsb=1 << 40, stream=None)
    a.update(kw)
    return capi.lib().lcml_fp8_attention_shared(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(dim=0), UNS), (dict(dim=24), UNS), (dict(dim=272), UNS), (dict(page=8), UNS), (dict(heads=0), BAD), (dict(seqs=-1), BAD),
    (dict(mq=-1), BAD), (dict(pages=-1), BAD), (dict(ts=3), BAD), (dict(table=None), BAD), (dict(kv=None), BAD), (dict(cu=None), BAD),
    (dict(kc=None), BAD), (dict(vs=None), BAD), (dict(kc=P + 8), BAD), (dict(ks=P + 2), BAD), (dict(tokens=-1), BAD),
    (dict(tokens=1 << 31), UNS), (dict(qd=10), UNS), (dict(od=17), UNS), (dict(q=None), BAD), (dict(o=None), BAD), (dict(q=P + 1), BAD),
    (dict(o=P + 2), BAD), (dict(qh=3), BAD), (dict(qh=0), BAD), (dict(scale=0.0), BAD), (dict(scale=float("nan")), BAD),
    (dict(mk=-1), BAD), (dict(mk=1 << 31), UNS), (dict(seqs=1 << 20, mq=1 << 20), UNS)])
def test_attention_refusals(kw, code):
    for fn in (sinks, shared):
        assert fn(**kw) == code, (fn.__name__, capi.last_error())
        assert "lcml_fp8_attention_" in capi.last_error()


@pytest.mark.parametrize("kw,code", [
    (dict(gs=None), BAD), (dict(pl=None), BAD), (dict(pt=None), BAD), (dict(gs=P + 2), BAD), (dict(pl=P + 1), BAD), (dict(pt=P + 2), BAD),
    (dict(groups=-1), BAD), (dict(pc=-1), BAD), (dict(mp=-1), BAD), (dict(ps=3), BAD), (dict(mp=1 << 31), UNS), (dict(groups=1 << 25), UNS),
    (dict(pc=1 << 31, ps=1 << 31), UNS), (dict(ws=None), BAD), (dict(wsb=100), BAD), (dict(ws=P + 8), BAD), (dict(tokens=1 << 29), UNS)])
def test_shared_refusals(kw, code):
    assert shared(**kw) == code, capi.last_error()


def test_sinks_refusals():
    assert sinks(sinks=-1) == BAD and "sinks" in capi.last_error()
    assert sinks(window=-1) == BAD
    assert sinks(mk=1 << 20, ws=None) == BAD and "workspace" in capi.last_error()


def test_no_ops():
    for fn in (sinks, shared):
        for kw in (dict(tokens=0), dict(seqs=0), dict(mq=0)):
            assert fn(**kw) == capi.OK, capi.last_error()
    assert capi.lib().lcml_fp8_attention_shared_workspace_bytes(0, 1, 1, 4, 2, 64, 1, 64, 64) == 0


def test_binding_refuses_what_it_cannot_check():
    with FakeTensorMode():
        new = lambda *s, dt=torch.int32: torch.empty(*s, dtype=dt, device="cuda:0")  # noqa: E731
        f32 = torch.float32
        ok = dict(new_tokens=new(2), kv_len=new(2), block_table=new(2, 4), free_pages=new(8), free_count=new(1), page_tokens=16,
                  kv_len_out=new(2), cu_q=new(3), left=new(1), workspace=new(8), stream=0)

        def refused(match, **kw):
            with pytest.raises(ValueError, match=match):
                capi.kv_cache_plan(**(ok | kw))
        refused("new_tokens", new_tokens=new(3))
        refused("kv_len_out", kv_len_out=new(2, dt=torch.int64))
        refused("block_table", block_table=new(1, 4).expand(2, 4))
        refused("cu_q", cu_q=new(2))
        refused("ended", ended=new(2, dt=torch.bool))
        refused("first_own", first_own=new(4)[::2])
        refused("positions", positions=new(8)[::2])
        refused("slots", slots=new(8))
        refused("slots", positions=new(8), slots=new(9, dt=torch.int64))
        refused("free_count", free_count=new(2))
        refused("workspace", workspace=new(8, 2)[:, :1])
        q, k, table = new(3, 4, 64, dt=f32), new(3, 2, 64, dt=f32), new(9, 64, dt=f32)

        def turned(match, q=q, k=k, positions=new(3), table=table, **kw):
            with pytest.raises(ValueError, match=match):
                capi.qk_norm_rope(q, k, positions, table, stream=0, **({"q_out": q, "k_out": k} | kw))
        turned("positions", positions=new(4))
        turned("table", table=new(9, 128, dt=f32)[:, ::2])
        turned("q_gamma", q_gamma=new(32, dt=f32))
        turned("k_gamma", k_gamma=new(64))
        turned("k_out", k_out=new(3, 2, 64, dt=torch.bfloat16))
        turned("k:", k=new(3, 2, 64, dt=torch.bfloat16))
        turned("k:", k=new(2, 2, 64, dt=f32))
        turned("q:", q=new(3, 4, 128, dt=f32)[..., ::2])
        turned("without k", k=None, k_out=k)
        cache = (new(8, 2, 16, 64, dt=torch.uint8), new(8, 2, 16, 64, dt=torch.uint8), new(8, 2, dt=f32), new(8, 2, dt=f32), new(2, 4),
                 new(2), new(3))

        def share(match, gs=new(2), pt=new(1, 4), pl=new(1), o=q, **kw):
            with pytest.raises(ValueError, match=match):
                capi.attention_shared(q, *cache, gs, pt, pl, 1, 9, 9, 0.1, out=o, workspace=q, stream=0, **kw)
        share("group_seq", gs=new(3))
        share("prefix_len", pl=new(1, dt=torch.int64))
        share("prefix_table", pt=new(2, 4))
        share("prefix_table", pt=new(1, 8)[:, ::2])
        share("out", o=new(3, 4, 32, dt=f32))
        with pytest.raises(ValueError, match="sinks"):
            capi.attention(q, *cache, 1, 9, 0.1, out=q, workspace=q, stream=0, sinks=1.5)


def test_plain_plan_by_hand():
    table, stack = np.array([[4, -1, -1], [2, 3, -1]], np.int32), [0, 1, 5, -9, -9, -9]
    kv, cu, left, pos, slots, table, stack = dc.plan([17, 0], [16, 20], table, stack, 3, 16, ended=[0, 1], own=[0, 1], tokens=18)
    assert (kv, cu, left) == ([33, 0], [0, 17, 17], 2) and stack == [0, 1, 5, 3, -9, -9]
    assert table.tolist() == [[4, 3, 5], [2, 3, -1]]
    assert pos == list(range(16, 33)) + [-1] and slots == [3 * 16 + i for i in range(16)] + [5 * 16, -1]


def test_plain_rotation_keeps_lengths_and_angles():
    x = np.random.default_rng(0).standard_normal((4, 2, 32))
    t = dc.turns(50, 32)
    for inter in (False, True):
        a = dc.norm_rope(x, None, 0, t, np.array([0, 5, 20, 49]), 32, inter)[0]
        b = dc.norm_rope(x, None, 0, t, np.array([0, 5, 20, 49]) - np.array([0, 5, 20, 0]), 32, inter)[0]
        assert np.allclose((a ** 2).sum(2), (x ** 2).sum(2), rtol=1e-6) and np.array_equal(a[0], x[0]) and np.allclose(a[3], b[3])
    # a product of two rotated heads depends on the distance of their positions alone
    y = dc.norm_rope(np.repeat(x[:1], 4, 0), None, 0, t, np.array([3, 10, 20, 27]), 32, True)[0][:, 0]
    assert np.isclose(y[0] @ y[1], y[2] @ y[3], rtol=1e-5)


def test_rope_table_is_the_rounded_definition():
    assert np.abs(capi.rope_table(300, 48, base=500.0).double().numpy() - dc.turns(300, 48, 500.0)).max() <= dc.TURNS_APART
    assert capi.rope_table(5, 0).shape == (5, 0)


def test_plain_attention_with_sinks_and_prefix():
    """Sinks that cover all that the window hides give plain attention; a prefix
    read through another row is the same tokens."""
    rng = np.random.default_rng(1)
    c = kc.Cache(6, 1, 16, 16, rng)
    x = rng.standard_normal((50, 1, 16)).astype(np.float32)
    table = np.array([[4, 0, 2, 5]])
    c.write(x, x, table, np.array([50]), np.array([0, 50]))
    q = rng.standard_normal((3, 2, 16)).astype(np.float32)
    a = kc.attention(q, c, table, [50], [0, 3], 1, 0.25)
    b = dc.attention(q, c, table, [50], [0, 3], 1, 0.25, window=5, sinks=45)
    d = dc.attention(q, c, np.array([[1, 1, 2, 5]]), [50], [0, 3], 1, 0.25, shared=([0, 1], np.array([[4, 0]]), [32]))
    for u, v, w in zip(a, b, d):
        assert np.allclose(u, v) and np.allclose(u, w)
    e = dc.attention(q, c, table, [50], [0, 3], 1, 0.25, window=5, sinks=2)[0]
    f = kc.attention(q, c, table, [50], [0, 3], 1, 0.25, window=5)[0]
    assert not np.allclose(e, f) and not np.allclose(e, a[0])
