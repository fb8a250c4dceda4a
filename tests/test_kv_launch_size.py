"""The bound of a cache write's and read's launch: 2^32 work items, counted as
the kernels start them."""
import pytest

from luisaml_amd import capi
from tests.test_serving_cpu import read, write


def threads_of_write(page, dim, mq):
    """A thread for each 4 tokens x 8 elements that can hold a new token, up to
    the next size of workgroup."""
    units = min((mq + 2) // 4 + 1, page // 4) * dim // 8
    return next((t for t in (64, 128, 256, 512) if units <= t), 1024)


@pytest.mark.parametrize("page,dim,mq", [(256, 80, 256), (128, 80, 128), (128, 144, 100), (256, 48, 256), (256, 256, 256)])
def test_write_rounded_up_to_a_workgroup(page, dim, mq):
    """More sequences than the launch holds, but for threads counted unit by
    unit: refused before the device is touched."""
    pages_each, heads = (mq - 2 + page) // page + 1, 8
    spots = (1 << 32) // threads_of_write(page, dim, mq) + 1
    seqs = -(-spots // (2 * heads * pages_each))
    assert write(page=page, dim=dim, mq=mq, heads=heads, seqs=seqs) == capi.ERR_UNSUPPORTED, capi.last_error()
    assert "exceeds one launch" in capi.last_error()


@pytest.mark.parametrize("page,dim", [(256, 80), (16, 16), (128, 256)])
def test_read_counts_its_units(page, dim):
    pages_each, heads = (page - 2 + page) // page + 1, 8
    spots = (1 << 32) // (page // 4 * dim // 8) + 1
    seqs = -(-spots // (2 * heads * pages_each))
    assert read(page=page, dim=dim, mq=page, heads=heads, seqs=seqs) == capi.ERR_UNSUPPORTED, capi.last_error()
    assert "exceeds one launch" in capi.last_error()
