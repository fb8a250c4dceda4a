"""Tensor arguments that the compiled binding refuses, on fake device tensors
(no storage, any device): whatever passes the binding meets the C ABI's NULL
checks, and nothing is launched."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from luisaml_amd import capi

U8, I32 = torch.uint8, torch.int32


@pytest.fixture
def fake():
    with FakeTensorMode():
        yield lambda *s, dt=torch.float32, dev="cuda:0": torch.empty(*s, dtype=dt, device=dev)


def cache(fake, seqs=2, cols=4, pages=8, heads=2, T=16, D=64):
    return dict(kc=fake(pages, heads, T, D, dt=U8), vc=fake(pages, heads, T, D, dt=U8), ks=fake(pages, heads),
                vs=fake(pages, heads), table=fake(seqs, cols, dt=I32), kv=fake(seqs, dt=I32), cu=fake(seqs + 1, dt=I32))


def calls(fake, c, tokens=2, heads=2, D=64):
    k = fake(tokens, heads, D)
    return (lambda: capi.kv_cache_write(k, k, *c.values(), 1, stream=0),
            lambda: capi.kv_cache_read(*c.values(), 1, k, k, stream=0),
            lambda: capi.attention(k, *c.values(), 1, 64, 0.1, out=k, workspace=k, stream=0))


def reaches_the_library(call):
    with pytest.raises(capi.LcmlError, match="NULL"):
        call()


def test_block_tables_whose_rows_overlap(fake):
    """An expanded row has a row stride of 0: taken for a pitch of its columns,
    rows past the first would be read past the table's end."""
    for table in (fake(1, 4, dt=I32).expand(2, 4), fake(8, dt=I32).as_strided((2, 4), (3, 1))):
        for call in calls(fake, cache(fake) | dict(table=table)):
            with pytest.raises(ValueError, match="block_table"):
                call()
    # a wider pitch, and one row whatever its stride
    for c in (cache(fake) | dict(table=fake(2, 9, dt=I32)[:, 2:6]),
              cache(fake, seqs=1) | dict(table=fake(4, dt=I32).as_strided((1, 4), (1, 1)))):
        for call in calls(fake, c):
            reaches_the_library(call)


@pytest.mark.skipif(torch.cuda.is_available() and torch.cuda.device_count() < 2, reason="cuda:1 cannot be named beside one GPU")
def test_tensors_of_two_devices(fake):
    """One tensor of another device among a call's: refused by its name."""
    other = dict(kc=(8, 2, 16, 64), vc=(8, 2, 16, 64), ks=(8, 2), vs=(8, 2), table=(2, 4), kv=(2,), cu=(3,))
    for name, shape in other.items():
        c = cache(fake)
        c[name] = fake(*shape, dt=c[name].dtype, dev="cuda:1")
        for call in calls(fake, c):
            with pytest.raises(ValueError, match="device is expected"):
                call()
    x, far = fake(3, 8), fake(3, 8, dev="cuda:1")
    a = dict(x=x, gamma=fake(8), eps=1e-5, residual=x, residual_out=x, mode=capi.SCALE_ROW, scale=fake(3), out=fake(3, 8, dt=U8))
    reaches_the_library(lambda: capi.rms_norm(**a, stream=0))
    for name in ("gamma", "residual", "residual_out", "scale", "out"):
        with pytest.raises(ValueError, match="device is expected"):
            capi.rms_norm(**(a | {name: fake(*a[name].shape, dt=a[name].dtype, dev="cuda:1")}), stream=0)
    with pytest.raises(ValueError, match="workspace: the other"):
        capi.rms_norm(**a | dict(mode=capi.SCALE_TENSOR), workspace=far, stream=0)
    q = fake(2, 4, 64)
    with pytest.raises(ValueError, match="workspace: the other"):
        capi.attention(q, *cache(fake).values(), 1, 64, 0.1, out=q, workspace=far, stream=0)


def test_current_stream_is_of_the_tensors_device(fake, monkeypatch):
    """Without a stream, a call goes to the current device's: tensors of another
    one are refused."""
    monkeypatch.setattr(capi, "_device", lambda: 1)
    monkeypatch.setattr(capi, "_raw_stream", lambda device: 0)
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    c = cache(fake).values()
    k, x, y = fake(2, 2, 64), fake(3, 8), fake(3, 8, dt=U8)
    for call in (lambda: capi.kv_cache_write(k, k, *c, 1), lambda: capi.kv_cache_read(*c, 1, k, k),
                 lambda: capi.attention(k, *c, 1, 64, 0.1, out=k, workspace=k),
                 lambda: capi.rms_norm(x, fake(8), 1e-5, mode=capi.SCALE_ROW, scale=fake(3), out=y)):
        with pytest.raises(ValueError, match="current device cuda:1"):
            call()


def test_one_row_of_any_stride(fake):
    """The row stride of a matrix of one row means nothing (an expanded vector's
    is 0); that of more rows does."""
    def norm(x, res, y, s):
        return lambda: capi.rms_norm(x, fake(8), 1e-5, residual=res, residual_out=res, mode=capi.SCALE_ROW, scale=s, out=y, stream=0)
    row = fake(8).expand(1, 8)
    reaches_the_library(norm(row, row, fake(8, dt=U8).expand(1, 8), fake(1)))
    for x, y in ((fake(8).expand(2, 8), fake(2, 8, dt=U8)), (fake(2, 8), fake(8, dt=U8).expand(2, 8))):
        with pytest.raises(capi.LcmlError, match="pitch"):
            norm(x, fake(2, 8), y, fake(2))()
