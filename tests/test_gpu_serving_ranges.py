"""Ranges of the norm and of attention between those of their own files: rows
past the registers with one scale for the tensor and in place, rows that all
but fill three groups of 256 threads, and windows over rows that are split."""
import numpy as np
import pytest
import torch

from luisaml_amd import capi, synth
from tests import kv_cases as kc
from tests.test_gpu_attention import MANY, run
from tests.test_gpu_rms_norm import MODES, T, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H", [16383, 16384, 16385, 16390, 20000, 40003])
@pytest.mark.parametrize("M", [2, 37])
@pytest.mark.parametrize("mode", ["static", "tensor", "row"])
@pytest.mark.parametrize("xt,rt,place", [("f", None, "none"), ("b", "b", "own"), ("b", "f", "residual"), ("f", "b", "residual")])
def test_norm_of_rows_past_the_registers(dev, H, M, mode, xt, rt, place):
    x = synth.normal(M + H, (M, H), std=2.0)
    x = kc.bf16(x) if xt == "b" else x
    gamma = 1.0 + synth.normal(H, (H,), std=0.2)
    res = synth.normal(M + 2 * H, (M, H), std=3.0) if rt else None
    res = kc.bf16(res) if rt == "b" else res
    xd, rd = torch.from_numpy(x).to(dev).to(T[xt]), None if res is None else torch.from_numpy(res).to(dev).to(T[rt])
    s = torch.full((1,), 0.01, device=dev) if mode == "static" else None
    y, s, h = capi.rms_norm(xd, torch.from_numpy(gamma).to(dev), 1e-5, residual=rd, mode=MODES[mode], scale=s,
                            residual_out=rd if place == "residual" else None)
    torch.cuda.synchronize()
    hn = None
    if res is not None:
        assert (h is rd) == (place == "residual")
        hn = x + res
        hn = kc.bf16(hn) if rt == "b" else hn
        assert np.array_equal(h.float().cpu().numpy(), hn)
    check(x, res, gamma, 1e-5, mode, y.cpu().numpy(), s.cpu().numpy(), hn)


@pytest.mark.parametrize("H", [3068, 3071, 6140])
@pytest.mark.parametrize("M,mode", [(2, "row"), (257, "tensor"), (300, "row")])
def test_norm_of_rows_that_all_but_fill_three_groups(dev, H, M, mode):
    x, res = kc.bf16(synth.normal(M + H, (M, H), std=2.0)), synth.normal(M + 2 * H, (M, H), std=3.0)
    gamma = 1.0 + synth.normal(H, (H,), std=0.2)
    y, s, h = capi.rms_norm(torch.from_numpy(x).to(dev).bfloat16(), torch.from_numpy(gamma).to(dev), 1e-5,
                            residual=torch.from_numpy(res).to(dev), mode=MODES[mode])
    torch.cuda.synchronize()
    hn = x + res
    assert np.array_equal(h.cpu().numpy(), hn)
    check(x, res, gamma, 1e-5, mode, y.cpu().numpy(), s.cpu().numpy(), hn)


@pytest.mark.parametrize("ot", ["b", "f"])
@pytest.mark.parametrize("kv,n,window,D,T,kernel", [
    ([20000, 3000], 1, 4000, 64, 64, "attention_few"), ([20000], 1, 12345, 128, 16, "attention_few"),
    ([9000, 5000], 5, 4097, 64, 32, "attention_few"), ([6000], 100, 2500, 64, 64, "attention_few"),
    ([6000, 4000], 200, 2049, 128, 64, "attention_many"), ([5000], 130, 3333, 256, 128, "attention_few")])
def test_windows_over_parts(dev, kv, n, window, D, T, kernel, ot):
    """A window over rows whose tokens are divided: parts start at the window,
    and the workspace, sized without one, holds them."""
    capi.kernel_trace()
    run(dev, kv, [n] * len(kv), T=T, H=1, G=8 if n >= 130 else 4, D=D, ot=ot, window=window, seed=n + D)
    assert capi.kernel_trace()[-2:] == [kernel, "attention_join"]


@pytest.mark.parametrize("window,causal", [(2000, True), (777, False), (5000, True)])
def test_windows_in_the_kernel_for_many_rows(dev, window, causal):
    """Long windows by a max_q above the true one, where nothing is split."""
    capi.kernel_trace()
    run(dev, [4100, 1500], [20, 150], T=64, H=1, G=4, D=64, window=window, causal=causal, max_q=MANY, seed=window)
    assert "attention_many" in ", ".join(capi.kernel_trace())
