"""GPU parity of lcml_fp8_qk_norm_rope with the 64-bit definition; tolerances
from decode_cases.norm_rope (fp32 roundings counted, then the result's own)."""
import numpy as np
import pytest
import torch

from luisaml_amd import capi, synth
from tests import decode_cases as dc
from tests import kv_cases as kc

pytestmark = pytest.mark.gpu
DT = {"f": torch.float32, "b": torch.bfloat16}


def close(got, x, gamma, eps, turn, pos, rot, inter, bf16):
    want, bound = dc.norm_rope(x, gamma, eps, turn, pos, rot, inter)
    bad = kc.outside(got, want, bound, bf16)
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5], bound[bad][:5])


def run(dev, tokens=7, H=4, K=2, D=128, rot=None, inter=False, norm=True, it="b", ot="b", rows=50, seed=0, positions=None,
        eps=1e-6, in_place=False, std=1.0):
    rot = D if rot is None else rot
    rng = np.random.default_rng(seed)
    x = synth.normal(seed + 1, (tokens, H + K, D)).astype(np.float32) * np.float32(std) if H + K else np.zeros((tokens, 0, D), np.float32)
    x = kc.bf16(x) if it == "b" else x
    gq, gk = (1 + 0.2 * synth.normal(seed + 2, (2, D))).astype(np.float32) if norm else (None, None)
    turn = dc.turns(rows, rot)
    pos = rng.integers(0, rows, tokens) if positions is None else np.array(positions)
    # columns of a wider projection, off its alignment
    wide = torch.zeros(tokens, (H + K) * D + 3, dtype=DT[it], device=dev)
    xd = wide[:, 1:1 + (H + K) * D].view(tokens, H + K, D)
    xd.copy_(torch.from_numpy(x))
    if in_place:
        out, od = wide, xd
    else:
        out = torch.full((tokens, (H + K) * D + 5), 9.0, dtype=DT[ot], device=dev)
        od = out[:, 3:3 + (H + K) * D].view(tokens, H + K, D)
    up = lambda a: None if a is None else torch.from_numpy(a).to(dev)  # noqa: E731
    q, k = capi.qk_norm_rope(xd[:, :H], xd[:, H:] if K else None, torch.tensor(pos, dtype=torch.int32, device=dev),
                             up(turn), q_gamma=up(gq), k_gamma=up(gk), eps=eps, interleaved=inter, q_out=od[:, :H],
                             k_out=od[:, H:] if K else None)
    torch.cuda.synchronize()
    got = od.float().cpu().numpy().astype(np.float64)
    if in_place:
        assert (out[:, :1] == 0).all() and (out[:, 1 + (H + K) * D:] == 0).all()
    else:
        assert (out[:, :3] == 9.0).all() and (out[:, 3 + (H + K) * D:] == 9.0).all()
    there = (pos >= 0) & ((pos < rows) | (rot == 0))
    before = x.astype(np.float64) if in_place else np.full_like(got, 9.0)
    assert np.array_equal(got[~there], before[~there])
    close(got[there][:, :H], x[there][:, :H], gq, eps, turn, pos[there], rot, inter, ot == "b")
    close(got[there][:, H:], x[there][:, H:], gk, eps, turn, pos[there], rot, inter, ot == "b")
    return got


@pytest.mark.parametrize("D", [16, 32, 48, 64, 80, 96, 112, 128, 192, 240, 256])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_head_sizes(dev, D, inter, norm):
    run(dev, 5, 5, 3, D, inter=inter, norm=norm, seed=D)


@pytest.mark.parametrize("it,ot", [("b", "b"), ("b", "f"), ("f", "f"), ("f", "b")])
@pytest.mark.parametrize("rot", [0, 2, 14, 16, 30, 32, 62, 64, 96])
@pytest.mark.parametrize("inter", [False, True])
def test_partial_rotation_and_types(dev, it, ot, rot, inter):
    run(dev, 6, 7, 2, 96, rot=rot, inter=inter, it=it, ot=ot, seed=rot)


@pytest.mark.parametrize("D,rot", [(16, 6), (64, 40), (128, 100), (256, 10), (256, 254)])
def test_odd_rotations(dev, D, rot):
    run(dev, 3, 9, 1, D, rot=rot, seed=rot)
    run(dev, 3, 9, 1, D, rot=rot, inter=True, it="f", ot="f", seed=rot)


@pytest.mark.parametrize("H,K", [(1, 1), (32, 8), (28, 4), (7, 7), (64, 1), (3, 0), (8, 8), (9, 17)])
@pytest.mark.parametrize("tokens", [1, 2, 65])
def test_heads_and_tokens(dev, H, K, tokens):
    run(dev, tokens, H, K, 128, seed=H + K)


def test_many_tokens(dev):
    """As many as take one wavefront, or fewer than all, for a token."""
    for tokens in (2049, 4099, 9001):
        run(dev, tokens, 12, 4, 64, rows=9001, seed=tokens)


def test_positions_without_a_row(dev):
    pos = [0, -1, 49, 50, 10 ** 6, -2 ** 31, 7]
    run(dev, positions=pos)
    run(dev, positions=pos, rot=0)
    run(dev, positions=pos, inter=True, in_place=True)
    run(dev, positions=[-1] * 7, in_place=True)


@pytest.mark.parametrize("D,rot,inter", [(128, 128, False), (96, 62, False), (80, 32, True), (256, 256, False)])
@pytest.mark.parametrize("t", ["b", "f"])
def test_in_place(dev, D, rot, inter, t):
    run(dev, 70, 9, 3, D, rot=rot, inter=inter, it=t, ot=t, in_place=True)


def test_no_positions_no_tokens_no_keys(dev):
    x = torch.randn(4, 3, 64, device=dev)
    g = torch.ones(64, device=dev)
    q, k = capi.qk_norm_rope(x, None, None, None, q_gamma=g)
    assert k is None
    close(q.double().cpu().numpy(), x.cpu().numpy(), g.cpu().numpy(), 1e-6, None, None, 0, False, False)
    q, k = capi.qk_norm_rope(x[:0], x[:0], torch.zeros(0, dtype=torch.int32, device=dev), capi.rope_table(5, 64, device=dev))
    assert q.shape == (0, 3, 64) and k.shape == (0, 3, 64)


def test_small_and_large_elements(dev):
    run(dev, std=1e-8, it="f", ot="f")
    run(dev, std=1e-3, eps=0.0, it="f", ot="f")
    run(dev, std=1e15, it="f", ot="f")
    got = capi.qk_norm_rope(torch.full((1, 1, 64), 1e30, device=dev), None, None, None, q_gamma=torch.ones(64, device=dev))[0]
    assert (got == 0).all()  # the squares' sum is infinite
    got = capi.qk_norm_rope(torch.zeros(1, 1, 64, device=dev), None, None, None, q_gamma=torch.ones(64, device=dev))[0]
    assert (got == 0).all()


def test_nan_and_infinity_stay_in_their_head(dev):
    x = torch.randn(3, 4, 128, device=dev)
    x[1, 2, 5], x[2, 0, 7] = float("nan"), float("inf")
    pos = torch.arange(3, dtype=torch.int32, device=dev)
    q, _ = capi.qk_norm_rope(x, None, pos, capi.rope_table(3, 128, device=dev), q_gamma=torch.ones(128, device=dev))
    bad = torch.isnan(q).any(dim=2)
    assert bad.tolist() == [[False] * 4, [False, False, True, False], [True, False, False, False]]
    assert torch.isnan(q[1, 2]).all() and (q[2, 0] != 0).sum() == torch.isnan(q[2, 0]).sum()


def test_far_positions_and_the_table(dev):
    """rope_table's rows are the roundings of the 64-bit cosines and sines."""
    t = capi.rope_table(200001, 64, device=dev)
    assert np.abs(t.double().cpu().numpy() - dc.turns(200001, 64)).max() <= dc.TURNS_APART
    run(dev, 4, 2, 1, 64, rows=200001, positions=[0, 1, 131072, 200000])


def test_rows_past_32_bit_offsets(dev):
    """Rows whose distance passes 2^31 elements and 4 GiB."""
    pitch = 600_000_000
    big = torch.zeros(5 * pitch, dtype=torch.bfloat16, device=dev)
    x = big.as_strided((5, 2, 64), (pitch, 64, 1))
    x.copy_(torch.from_numpy(synth.normal(3, (5, 2, 64))))
    pos = torch.arange(5, dtype=torch.int32, device=dev)
    g = torch.ones(64, device=dev)
    want = capi.qk_norm_rope(x.contiguous(), None, pos, capi.rope_table(5, 64, device=dev), q_gamma=g)[0]
    capi.qk_norm_rope(x, None, pos, capi.rope_table(5, 64, device=dev), q_gamma=g, q_out=x)
    torch.cuda.synchronize()
    assert torch.equal(x, want)


def test_graph_and_other_stream(dev):
    x = torch.randn(6, 5, 128, device=dev).bfloat16()
    pos, t, g = torch.arange(6, dtype=torch.int32, device=dev), capi.rope_table(40, 128, device=dev), torch.ones(128, device=dev)
    q, k = torch.empty(6, 4, 128, device=dev), torch.empty(6, 1, 128, device=dev)
    call = lambda **kw: capi.qk_norm_rope(x[:, :4], x[:, 4:], pos, t, q_gamma=g, k_gamma=g, **kw)  # noqa: E731
    call(q_out=q, k_out=k)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(q_out=q, k_out=k)
    side = torch.cuda.Stream()
    for step in range(4):
        pos.add_(3)
        x.neg_()
        want = call(out_dtype=torch.float32)
        q.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(q, want[0]) and torch.equal(k, want[1])
        other = call(out_dtype=torch.float32, stream=side)
        side.synchronize()
        assert torch.equal(q, other[0]) and torch.equal(k, other[1])
