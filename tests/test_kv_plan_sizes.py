"""The step plan at the ends of its sizes: how many sequences a call takes,
and lengths and row offsets at the end of int32."""
import numpy as np
import pytest
import torch

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


MOST = 2 ** 31 - 1
# tokens held and brought: offsets that stop at MOST in a sequence, before and
# after others, and with its length
CUT = [([0, 0], [5, MOST - 2]), ([0, 1], [3, MOST - 1]), ([40, 1000, 7], [20, MOST - 1000, 9]), ([0], [MOST]), ([17, 0, 3], [MOST, 5, 5]),
       ([0, 0, 33], [MOST - 30, 31, 2]), ([0, 300, 20], [5, MOST - 300, MOST])]


def expected(held, n, tokens):
    """(kv, cu, positions of the first `tokens` rows), one sequence after the other."""
    kv, cu, pos, rows = [], [0], np.full(tokens, -1), 0
    for a, b in zip(held, n):
        kv.append(min(a + b, MOST))
        k = kv[-1] - a
        if rows < tokens:
            pos[rows:min(rows + k, tokens)] = a + np.arange(min(k, tokens - rows))
        rows += k
        cu.append(min(rows, MOST))
    return kv, cu, pos


@pytest.mark.gpu
@pytest.mark.parametrize("held,n", CUT)
@pytest.mark.parametrize("tokens", [100, 1500, 40000])
@pytest.mark.parametrize("more", [0, 100, 3000])
def test_offsets_that_stop_at_the_end_of_int32(dev, held, n, tokens, more):
    """One launch and two, with and without the sums in LDS (`more` sequences
    that have no tokens, before the others)."""
    held, n = [0] * more + held, [0] * more + n
    i32 = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device=dev)  # noqa: E731
    cols, T = 30, 16
    has = [min(-(-x // T), cols) for x in held]
    pages = sum(has) + cols * len(CUT[0][0]) * 2
    table = np.full((len(held), cols), -1, np.int32)
    for b, k in enumerate(has):
        table[b, :k] = np.arange(k) + sum(has[:b])
    free = list(range(sum(has), pages))
    stack = i32(free + [-7] * (pages - len(free)))
    got = i32(table)
    kv, cu, left, pos, slots = capi.kv_cache_plan(i32(n), i32(held), got, stack, i32([len(free)]), T, tokens=tokens)
    torch.cuda.synchronize()
    want_kv, want_cu, want_pos = expected(held, n, tokens)
    for b, (a, e) in enumerate(zip(has, want_kv)):
        for c in range(a, min(-(-e // T), cols)):
            table[b, c] = free.pop() if free else -1
    assert kv.tolist() == want_kv and cu.tolist() == want_cu and np.array_equal(got.cpu().numpy(), table)
    assert np.array_equal(pos.cpu().numpy(), want_pos)
    of = np.searchsorted(np.array(want_cu[1:]), np.arange(tokens), side="right").clip(0, len(n) - 1)
    page = np.where((want_pos >= 0) & (want_pos // T < cols), table[of, (want_pos // T).clip(0, cols - 1)], -1).astype(np.int64)
    assert np.array_equal(slots.cpu().numpy(), np.where(page >= 0, page * T + want_pos % T, -1))
