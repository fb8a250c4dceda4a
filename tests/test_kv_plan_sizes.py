"""The step plan at the ends of its sizes: how many sequences a call takes."""
import pytest

from luisaml_amd import capi

P = 0x1000


def plan(seqs, tokens=0):
    return capi.lib().lcml_fp8_kv_cache_plan(P, P, P, P, seqs, P, P, 8, 16, P, 4, 4, P, P, P, P, P, tokens, None, 0, None)


@pytest.mark.parametrize("seqs", [2 ** 30 + 1, 2 ** 31 - 1025, 2 ** 31 - 2, 2 ** 31 - 1])
def test_more_sequences_than_32_bits_index(seqs):
    assert plan(seqs) == capi.ERR_UNSUPPORTED and "seqs" in capi.last_error()


def test_the_most_sequences():
    """Up to the check of the workspace, which comes last."""
    assert plan(2 ** 30) == capi.ERR_INVALID_ARG and "workspace of 8589934608 bytes" in capi.last_error()
