"""Queries with infinite elements, of both types and in both kernels, against
the definition in 64 bits: scores of -inf weigh nothing (a row of nothing else
is 0), one of +inf or of 0 times an infinity makes the row NaN."""
import numpy as np
import pytest
import torch

from luisaml_amd import capi, synth
from tests import kv_cases as kc

pytestmark = pytest.mark.gpu
DT = {"f": torch.float32, "b": torch.bfloat16}
MANY = 1 << 15  # a max_q far above the true one takes the kernel for many rows


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("qt,ot", [("b", "b"), ("b", "f"), ("f", "f"), ("f", "b")])
@pytest.mark.parametrize("D", [64, 80, 128, 256])
@pytest.mark.parametrize("window", [0, 20])
def test_infinite_elements(dev, D, qt, ot, many, window):
    H, G, T, kv_len, n = 1, 8, 16, [90], 12
    rng = np.random.default_rng(D)
    table, pages = kc.tables(kv_len, T, rng)
    cache = kc.Cache(pages, H, T, D, rng)
    k, v = (synth.normal(s, (90, H, D)).astype(np.float32) for s in (1, 2))
    k[:, :, 3] = np.abs(k[:, :, 3]) + 0.5  # of one sign in every token
    k[:, :, 9] = -np.abs(k[:, :, 9]) - 0.5
    k[:, :, 11] = np.where(np.arange(90) % 2, 1.0, -1.0)[:, None]  # of either
    k[:, :, 13] = np.where(np.arange(90) == 85, 0.0, 1.0)[:, None]  # 0 in one
    cache.write(k, v, table, np.array(kv_len), [0, 90])
    q = synth.normal(3, (n, G, D)).astype(np.float32)
    inf = np.inf
    q[:, 0, 3] = -inf  # all scores -inf: 0
    q[:, 1, 9] = inf  # likewise
    q[:, 2, 3] = inf  # all +inf: NaN
    q[:, 3, 11] = inf  # both: NaN
    q[:, 4, 13] = -inf  # NaN once position 85 is seen, 0 before
    q[:, 5, 3], q[:, 5, 9] = -inf, inf  # -inf twice: 0
    q[:, 6, 3], q[:, 6, 9] = inf, inf  # inf - inf: NaN
    q = kc.bf16(q) if qt == "b" else q
    idx = tuple(torch.tensor(np.asarray(a), dtype=torch.int32, device=dev) for a in (table, kv_len, [0, n]))
    scale = float(np.float32(D ** -0.5))
    capi.kernel_trace()
    out = capi.attention(torch.from_numpy(q).to(dev).to(DT[qt]), *cache.to(dev), *idx, MANY if many else n, 90, scale,
                         window=window, out_dtype=DT[ot])
    torch.cuda.synchronize()
    assert ("attention_many" in ", ".join(capi.kernel_trace())) == many
    got = out.float().cpu().numpy().astype(np.float64)
    o, mass, reach = kc.attention(q, cache, table, kv_len, [0, n], H, scale, True, window)
    for h in (0, 1, 5):
        assert (got[:, h] == 0).all(), h
    for h in (2, 3, 6):
        assert np.isnan(got[:, h]).all(), h
    assert (got[:7, 4] == 0).all() and np.isnan(got[7:, 4]).all()  # row 7 is position 85
    assert np.array_equal(np.isnan(got), np.isnan(o))
    bound = kc.attention_bound(mass, np.where(np.isfinite(reach), reach, 0.0), D, 90, ot == "b")
    assert not kc.outside(got[:, 7], o[:, 7], bound[:, 7], ot == "b").any()
