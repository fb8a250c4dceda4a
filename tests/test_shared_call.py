"""attention_shared() with and without a bound on a group's rows: the same call
of the entry point."""
import numpy as np
import pytest
import torch

from luisaml_amd import capi
from tests.test_gpu_attention import i32
from tests.test_gpu_attention_shared import batch

SHORT, LONG = (7, 90, 640, 0.25), (7, 90, 33, 640, 0.25)


@pytest.fixture
def passed(monkeypatch):
    """calls(*numbers, **kw): what the binding is given for them."""
    class Binding:
        def attention_shared(self, *args):
            self.args = args
            return capi.OK
    binding = Binding()
    monkeypatch.setattr(capi, "_binding", lambda: binding)
    monkeypatch.setattr(capi, "_where", lambda stream: (stream, -1))
    tensors = [torch.zeros(3, 4, 64)] + [torch.zeros(1) for _ in range(10)]

    def calls(*numbers, **kw):
        out, workspace = tensors[0], tensors[1]
        assert capi.attention_shared(*tensors, *numbers, **({"out": out, "workspace": workspace} | kw)) is out
        at = [i for i, a in enumerate(binding.args) if a is workspace][-1]
        return binding.args[at - 5:at]  # max_q, max_own, max_prefix, scale, causal
    return calls


@pytest.mark.parametrize("number", [float, np.float64, np.float32])
def test_bound_on_a_groups_rows_by_place(passed, number):
    *bounds, scale = LONG
    assert passed(*bounds, number(scale)) == (7, 90, 640, 0.25, True)
    assert passed(*bounds, number(scale), False) == (7, 90, 640, 0.25, False)
    assert passed(*bounds, number(scale), causal=False) == (7, 90, 640, 0.25, False)
    assert passed(*bounds, scale=number(scale)) == (7, 90, 640, 0.25, True)


def test_without_it_and_by_name(passed):
    for kw in ({}, {"max_group_q": 33}, {"max_group_q": None}):
        assert passed(*SHORT, **kw) == (7, 90, 640, 0.25, True)
        assert passed(*SHORT, False, **kw) == (7, 90, 640, 0.25, False)
        assert passed(*SHORT, 0, **kw) == (7, 90, 640, 0.25, 0)
        assert passed(7, 90, max_prefix=640, scale=0.25, causal=False, **kw) == (7, 90, 640, 0.25, False)
        assert passed(7, 90, 640, scale=1, **kw) == (7, 90, 640, 1, True)


def test_refused(passed):
    for call in (lambda: passed(7, 90, -1, 640, 0.25), lambda: passed(*SHORT, max_group_q=-1)):
        with pytest.raises(ValueError, match="max_group_q"):
            call()
    for call in (lambda: passed(7, 90, 1.5, 640, 0.25), lambda: passed(*LONG, max_group_q=33), lambda: passed(7, 90, 640)):
        with pytest.raises(TypeError):
            call()


P = 0x1000


def entry(tokens, seqs, max_q, workspace=None, heads=32):
    return capi.lib().lcml_fp8_attention_shared(
        P, 16, tokens, heads, heads * 128, 128, P, 16, heads * 128, 128, P, P, P, P, 8, 8, 128, 16, P, 4, 4, P, P, seqs, P, P, 4, 4, P,
        1, max_q, 800, 4096, 0.1, 1, workspace, 0, None)


@pytest.mark.parametrize("tokens,seqs,max_q", [(8255, 64, 8192), (2303, 256, 2048), (100000, 64, 65536), (1000000, 4, 250000)])
def test_single_tokens_beside_a_chunk_are_accepted(tokens, seqs, max_q):
    """Up to the check of the workspace, which comes last."""
    assert entry(tokens, seqs, max_q) == capi.ERR_INVALID_ARG and "workspace" in capi.last_error()


@pytest.mark.parametrize("tokens,seqs,max_q", [(1 << 27, 1, 1 << 27), (1 << 20, 1 << 20, 1 << 20)])
def test_sizes_past_a_launch(tokens, seqs, max_q):
    assert entry(tokens, seqs, max_q) == capi.ERR_UNSUPPORTED and "exceeds one launch" in capi.last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 40])
def test_same_bits(dev, n):
    cache, table, kv, first, pt, plen = batch([(64, [60, 70, 50]), (32, [41, 42])], 16, 2, 64, 1)
    q = torch.randn(5 * n, 8, 64, device=dev, generator=torch.Generator(device=dev).manual_seed(n))
    args = (q, *cache.to(dev), i32(table, dev), i32(kv, dev), i32(range(0, 5 * n + 1, n), dev), i32(first, dev), i32(pt, dev),
            i32(plen, dev))
    want = capi.attention_shared(*args, n, 70, 64, 0.125)
    for got in (capi.attention_shared(*args, n, 70, 3 * n, 64, 0.125), capi.attention_shared(*args, n, 70, 64, 0.125, max_group_q=3 * n)):
        torch.cuda.synchronize()
        assert torch.equal(got, want)
