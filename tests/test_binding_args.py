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
