"""attention_shared() over batches whose sequences bring very different numbers
of rows: the join goes through the batch's rows and finds each one's sequence."""
import numpy as np
import pytest
import torch

from luisaml_amd import capi, synth
from tests import decode_cases as dc
from tests import kv_cases as kc
from tests.test_gpu_attention import DT, i32
from tests.test_gpu_attention_shared import batch

pytestmark = pytest.mark.gpu


def run(dev, groups, n, H, G, D, before=0, behind=0, max_q=None, max_prefix=None, ot="f", seed=0):
    """n: rows of each sequence, after `before` rows of no sequence and before
    `behind` ones, which stay as they are; those past max_q too."""
    cache, table, kv, first, pt, plen = batch(groups, 16, H, D, seed)
    cu = before + np.concatenate([[0], np.cumsum(n)])
    rows, mq = cu[-1] + behind, max(n) if max_q is None else max_q
    q = synth.normal(seed + 7, (rows, H * G, D)).astype(np.float32)
    out = torch.full((rows, H * G, D), 9.0, dtype=DT[ot], device=dev)
    capi.attention_shared(torch.from_numpy(q).to(dev), *cache.to(dev), i32(table, dev), i32(kv, dev), i32(cu, dev), i32(first, dev),
                          i32(pt, dev), i32(plen, dev), mq, max(max(o) for _, o in groups),
                          max(plen) if max_prefix is None else max_prefix, 0.2, out=out)
    torch.cuda.synchronize()
    got = out.double().cpu().numpy()
    row = np.concatenate([np.arange(c, c + min(k, mq)) for c, k in zip(cu, n)])
    assert (np.delete(got, row, 0) == 9.0).all()
    o, mass, reach = dc.attention(q, cache, table, kv, cu, H, float(np.float32(0.2)), shared=(first, pt, plen))
    bound = kc.attention_bound(mass, reach, D, int(kv.max()), ot == "b")
    bad = kc.outside(got, o, bound, ot == "b")[row]
    assert not bad.any(), np.argwhere(bad)[:5]


@pytest.mark.parametrize("most", [None, 300])
def test_single_tokens_beside_a_chunk(dev, most):
    """More rows than a launch has workgroups, if every sequence had as many as
    the longest one."""
    n = np.ones(2100, dtype=int)
    n[1234] = 500
    assert len(n) * 300 * 32 > 1 << 24
    own = [510 if k > 1 else 1 + b % 3 for b, k in enumerate(n)]
    run(dev, [(64, own[:1000]), (32, own[1000:1500]), (0, own[1500:])], n, 1, 32, 16, behind=3, max_q=most)


@pytest.mark.parametrize("rows", [0.9, 0.3, 0.02])
@pytest.mark.parametrize("seqs", [1, 2, 63, 64, 65, 127, 128, 129, 500, 4095, 4096, 4097])
def test_sequence_of_a_row(dev, seqs, rows):
    """Sequences with none, one or a few rows, some of them first and last; joins
    of many rows a workgroup, and (few rows) of one."""
    rng = np.random.default_rng(seqs)
    n = np.where(rng.random(seqs) < rows, rng.integers(1, 4, seqs), 0)
    n[seqs // 2] = 3
    own = [int(k) + int(x) for k, x in zip(n, rng.integers(1, 3, seqs))]
    half = seqs // 2
    run(dev, [(32, own[:half]), (48, own[half:])] if half else [(32, own)], n, 1, 2, 16, before=2, behind=5, seed=seqs)


@pytest.mark.parametrize("D", [16, 64, 80, 256])
@pytest.mark.parametrize("ot", ["b", "f"])
def test_many_parts(dev, D, ot):
    """More parts than the join of many rows takes, with more rows than it begins at."""
    n = [1, 0, 40, 1, 2, 0, 1, 25]
    run(dev, [(64, [4, 2, 70, 3]), (48, [5, 1, 2, 33])], n, 1, 8, D, before=1, behind=2, max_prefix=1 << 20, ot=ot, seed=D)
