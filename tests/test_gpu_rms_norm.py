"""GPU parity of lcml_fp8_rms_norm: residual addition, RMS norm and E4M3 codes.

Bars: the stored h is bit-exact (one fp32 addition, rounded once); the scale
is within EPS of max|v|/448 in 64 bits, and every code lies between the codes
of q (1 - EPS) and q (1 + EPS), q the 64-bit quotient by the scale returned.
EPS: the sum of squares of H terms in H/256 + 16 steps at most (all terms
positive), half of it after the square root, and eight more roundings."""
import numpy as np
import pytest
import torch

from luisaml_amd import capi, synth
from tests import kv_cases as kc

pytestmark = pytest.mark.gpu
T = {"f": torch.float32, "b": torch.bfloat16}
MODES = {"static": capi.SCALE_STATIC, "tensor": capi.SCALE_TENSOR, "row": capi.SCALE_ROW}


def eps_of(H):
    return ((H / 256 + 16) / 2 + 8) * 2.0 ** -24


def padded(a, dt, dev, pad):
    """a as the columns of a wider tensor, starting off its alignment."""
    t = torch.zeros(a.shape[0], a.shape[1] + pad, dtype=dt, device=dev)
    v = t[:, pad // 2:pad // 2 + a.shape[1]]
    v.copy_(torch.from_numpy(a))
    return v


def check(x, res, gamma, eps, mode, y, s, h):
    """x, res fp32 arrays of values of their types; results as numpy."""
    M, H = x.shape
    e = eps_of(H)
    hv = x if res is None else h.astype(np.float64)
    hv = hv.astype(np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        v = hv / np.sqrt((hv ** 2).mean(axis=1, keepdims=True) + eps) * gamma.astype(np.float64)
    a = np.where(np.isnan(v), 0.0, np.abs(v))
    if mode != "static":
        want = (a.max(axis=1) if mode == "row" else a.max(keepdims=True).reshape(1)) / 448.0
        want = np.where((want > 0) & np.isfinite(want), want, 1.0)
        assert np.all(np.abs(s - want) <= e * want), np.abs(s / want - 1).max()
    sv = s.astype(np.float64)
    sv = sv[:, None] if mode == "row" else sv
    with np.errstate(invalid="ignore", over="ignore"):
        q = v / sv
        lo, hi = (kc.encode(np.clip(q * (1 + t), -3e38, 3e38)) for t in (-e, e))
    got, a, b = kc.decode(y), kc.decode(lo), kc.decode(hi)
    ok = ((got >= np.minimum(a, b)) & (got <= np.maximum(a, b))) | (np.isnan(got) & np.isnan(a))
    assert ok.all(), (np.argwhere(~ok)[:4], got[~ok][:4], q[~ok][:4])


@pytest.mark.parametrize("M,H", [(1, 1), (1, 16), (3, 63), (2, 64), (5, 1000), (2, 1024), (7, 1025), (1, 4096),
                                 (33, 4096), (1030, 272), (2, 4097), (2, 5003), (3, 11008), (1, 40000)])
@pytest.mark.parametrize("mode", ["static", "tensor", "row"])
@pytest.mark.parametrize("xt,rt", [("f", None), ("b", "b"), ("b", "f"), ("f", "b")])
def test_matches_64_bit(dev, M, H, mode, xt, rt):
    x = synth.normal(M + H, (M, H), std=2.0)
    x = kc.bf16(x) if xt == "b" else x
    gamma = 1.0 + synth.normal(H, (H,), std=0.2)
    res = synth.normal(M + 2 * H, (M, H), std=3.0) if rt else None
    res = kc.bf16(res) if rt == "b" else res
    xd, rd = torch.from_numpy(x).to(dev).to(T[xt]), None if res is None else torch.from_numpy(res).to(dev).to(T[rt])
    s = torch.full((1,), 0.01, device=dev) if mode == "static" else None
    y, s, h = capi.rms_norm(xd, torch.from_numpy(gamma).to(dev), 1e-5, residual=rd, mode=MODES[mode], scale=s)
    torch.cuda.synchronize()
    hn = None
    if res is not None:
        hn = x + res
        hn = kc.bf16(hn) if rt == "b" else hn
        assert np.array_equal(h.float().cpu().numpy(), hn)
    else:
        assert h is None
    check(x, res, gamma, 1e-5, mode, y.cpu().numpy(), s.cpu().numpy(), hn)


@pytest.mark.parametrize("H", [256, 257, 511, 514, 768, 771, 1026, 2048, 2049, 2560, 3074, 4095, 4100, 6144, 6146, 8191,
                               8196])
@pytest.mark.parametrize("M,mode", [(2, "row"), (257, "tensor"), (300, "row")])
def test_either_side_of_each_width(dev, H, M, mode):
    """Rows that just fill the registers of a number of threads, and that just
    do not, of few rows and of many."""
    x, res = kc.bf16(synth.normal(M + H, (M, H), std=2.0)), synth.normal(M + 2 * H, (M, H), std=3.0)
    gamma = 1.0 + synth.normal(H, (H,), std=0.2)
    y, s, h = capi.rms_norm(torch.from_numpy(x).to(dev).bfloat16(), torch.from_numpy(gamma).to(dev), 1e-5,
                            residual=torch.from_numpy(res).to(dev), mode=MODES[mode])
    torch.cuda.synchronize()
    hn = x + res
    assert np.array_equal(h.cpu().numpy(), hn)
    check(x, res, gamma, 1e-5, mode, y.cpu().numpy(), s.cpu().numpy(), hn)


@pytest.mark.parametrize("mode", ["static", "tensor", "row"])
@pytest.mark.parametrize("H", [100, 4200])
def test_pitches_alignment_in_place_and_other_stream(dev, mode, H):
    """Columns of wider tensors that start off their alignment, the residual
    updated in place, pitched codes, a stream of its own; the same bytes as
    the dense call."""
    M = 9
    x, res = kc.bf16(synth.normal(1, (M, H))), kc.bf16(synth.normal(2, (M, H)))
    gamma = torch.from_numpy(1.0 + synth.normal(3, (H,), std=0.2)).to(dev)
    s0 = torch.full((1,), 0.02, device=dev) if mode == "static" else None
    want = capi.rms_norm(torch.from_numpy(x).to(dev).bfloat16(), gamma, 1e-6,
                         residual=torch.from_numpy(res).to(dev).bfloat16(), mode=MODES[mode], scale=s0)
    xd, rd = padded(x, torch.bfloat16, dev, 5), padded(res, torch.bfloat16, dev, 7)
    y = torch.full((M, H + 3), 0xAA, dtype=torch.uint8, device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = capi.rms_norm(xd, gamma, 1e-6, residual=rd, residual_out=rd, mode=MODES[mode], scale=s0, out=y[:, 1:H + 1])
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(rd, want[2])
    assert (y[:, 0] == 0xAA).all() and (y[:, H + 1:] == 0xAA).all()


@pytest.mark.parametrize("mode", ["static", "tensor", "row"])
def test_zero_infinite_and_nan_rows(dev, mode):
    M, H = 6, 300
    x = synth.normal(5, (M, H))
    x[1] = 0.0
    x[2, 7] = np.inf
    x[3, 9] = np.nan
    x[4] *= 1e-30
    x[5] *= 1e25  # the sum of squares overflows: zeros
    gamma = 1.0 + synth.normal(6, (H,), std=0.1)
    s = torch.full((1,), 0.01, device=dev) if mode == "static" else None
    y, s, _ = capi.rms_norm(torch.from_numpy(x).to(dev), torch.from_numpy(gamma).to(dev), 1e-5, mode=MODES[mode], scale=s)
    y, s = y.cpu().numpy(), s.cpu().numpy()
    assert (y[1] == 0).all() and (kc.decode(y[5]) == 0).all()
    assert (y[3] == 0x7F).all()
    assert (y[2] == 0x7F).sum() == 1 and y[2, 7] == 0x7F and (kc.decode(np.delete(y[2], 7)) == 0).all()
    if mode == "row":
        assert s[1] == 1.0 and s[2] == 1.0 and s[3] == 1.0 and s[5] == 1.0
    keep = [0, 1, 4]
    if mode != "tensor":
        check(x[keep], None, gamma, 1e-5, mode, y[keep], s[keep] if mode == "row" else s, None)


def test_tensor_scale_feeds_the_gemm(dev):
    """The codes and the scale as lcml_fp8_gemm's operands, graph-captured:
    the same bits on every replay."""
    M, H, N = 40, 512, 192
    x = torch.from_numpy(synth.normal(1, (M, H))).to(dev).bfloat16()
    gamma = torch.ones(H, device=dev)
    w = torch.from_numpy(synth.normal(2, (H, N), std=0.05)).to(dev)
    sw = w.abs().amax(dim=0) / 448.0
    wp = capi.pack_weight(capi.quantize(w, sw, axis=1), w_is_nk=False)
    y, s, _ = capi.rms_norm(x, gamma, 1e-5)
    want = capi.gemm(y, s, wp, sw, N, H)
    ref = (x.double() / (x.double().square().mean(dim=1, keepdim=True) + 1e-5).sqrt()) @ w.double()
    torch.cuda.synchronize()
    assert ((want - ref).norm() / ref.norm()).item() < 0.06  # two operands of 4 significant bits
    out, so, ws = torch.empty_like(y), torch.empty_like(s), torch.empty(1 << 16, dtype=torch.uint8, device=dev)
    g = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        capi.rms_norm(x, gamma, 1e-5, out=out, scale=so, workspace=ws)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        capi.rms_norm(x, gamma, 1e-5, out=out, scale=so, workspace=ws)
        got = capi.gemm(out, so, wp, sw, N, H)
    for k in range(3):
        x.mul_(1.0)
        got.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(out, y)


def test_kernel_trace_and_empty(dev):
    capi.kernel_trace()
    x = torch.zeros(0, 64, device=dev)
    y, s, _ = capi.rms_norm(x, torch.ones(64, device=dev), 1e-5, mode=capi.SCALE_ROW)
    assert y.shape == (0, 64) and capi.kernel_trace() == []
    capi.rms_norm(torch.ones(2, 64, device=dev), torch.ones(64, device=dev), 1e-5)
    assert capi.kernel_trace() == ["lcml_fp8_rms_norm"]
