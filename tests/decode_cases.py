"""Plain implementations of the step plan, the norm with rotation, and of
attention with sinks or behind shared prefixes, in 64 bits and one element after
the other, for the GPU tests to compare with."""
import numpy as np

from tests import kv_cases as kc

U = 2.0 ** -24  # of an fp32 rounding


# ------------------------------------------------------------------- plan --

def plan(n, held, table, stack, free, T, ended=None, own=None, tokens=None):
    """(kv, cu, left, positions, slots, table, stack), lists and arrays."""
    table, stack, pages = np.array(table), list(stack), len(stack)
    seqs, cols = table.shape
    ended = [0] * seqs if ended is None else ended
    own = [0] * seqs if own is None else own
    top = min(max(int(free), 0), pages)
    for b in range(seqs):
        if ended[b]:
            for c in range(max(own[b], 0), min(-(-max(held[b], 0) // T), cols)):
                if 0 <= table[b, c] < pages and top < pages:
                    stack[top] = int(table[b, c])
                    top += 1
    kv, cu, pos, slots = [], [0], [], []
    for b in range(seqs):
        old, new = (0 if ended[b] else max(held[b], 0)), max(n[b], 0)
        kv.append(old + new)
        cu.append(cu[-1] + new)
        for c in range(-(-old // T), min(-(-kv[b] // T), cols)):
            top -= 1
            table[b, c] = stack[top] if top >= 0 else -1
        for p in range(old, kv[b]):
            page = table[b, p // T] if p // T < cols else -1
            pos.append(p)
            slots.append(int(page) * T + p % T if 0 <= page < pages else -1)
    tokens = len(pos) if tokens is None else tokens
    spare = [-1] * max(0, tokens - len(pos))
    return kv, cu, top, (pos + spare)[:tokens], (slots + spare)[:tokens], table, stack


def pool(held, T, cols, pages, rng):
    """A table of pages in any order for sequences of these lengths, and a stack
    of the rest."""
    need = [min(-(-max(x, 0) // T), cols) for x in held]
    order = rng.permutation(pages)
    table, at = np.full((len(held), cols), -1, np.int32), 0
    for b, k in enumerate(need):
        table[b, :k] = order[at:at + k]
        at += k
    stack = np.full(pages, -9, np.int32)
    stack[:pages - at] = order[at:]
    return table, stack, pages - at


# --------------------------------------------------------- norm, rotation --

def norm_rope(x, gamma, eps, turn, positions, rot, interleaved):
    """x [tokens, heads, D] -> (result, bound of an fp32 evaluation's error).

    The bound: a sum of D <= 256 squares by 16 fused steps and 4 additions, the
    mean's two roundings, eps's, a root (which halves what was before it), a
    division and two products leave less than 18 roundings of v; each product
    with a cosine or sine and the sum of two add one each."""
    v = x.astype(np.float64)
    mass = np.abs(v)
    count = 0
    if gamma is not None:
        v = v / np.sqrt((v ** 2).mean(axis=2, keepdims=True) + eps) * gamma.astype(np.float64)
        count = 18
    mass, out = np.abs(v), v.copy()
    half = rot // 2
    if half:
        row = turn.astype(np.float64)[np.clip(positions, 0, len(turn) - 1)][:, None]
        c, s = row[..., :half], row[..., half:]
        i = np.arange(half)
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        out[..., a], out[..., b] = v[..., a] * c - v[..., b] * s, v[..., b] * c + v[..., a] * s
        m = mass.copy()
        mass[..., a], mass[..., b] = m[..., a] * abs(c) + m[..., b] * abs(s), m[..., b] * abs(c) + m[..., a] * abs(s)
        count += 2
    return out, mass * count * U + 1e-37


def turns(rows, rot, base=10000.0):
    a = np.arange(rows)[:, None] * base ** (-np.arange(rot // 2) / max(rot // 2, 1))
    return np.concatenate([np.cos(a), np.sin(a)], axis=1).astype(np.float32)


# How far two such tables of up to 2^18 positions may be apart.  A power in 64
# bits is within two steps of 2^-52 of itself, so an angle within 2^18 * 2^-51 +
# 2^-35 < 2^-32 of its value, and so are its cosine and sine; those are rounded
# to fp32 by 2^-25 at most.  Two libraries' 64-bit functions may differ by all of
# that on either side.
TURNS_APART = 2 * (2.0 ** -32 + 2.0 ** -25)


# --------------------------------------------------------------- attention --

def attention(q, cache, table, kv_len, cu, heads, scale, causal=True, window=0, sinks=0, shared=None):
    """o, and for tolerances the sums and reach of kv_cases.attention.  shared:
    (group_seq, prefix_table, prefix_len): positions of a prefix are read there
    by sequences whose rows all lie behind it."""
    tokens, q_heads, D = q.shape
    o = np.zeros((tokens, q_heads, D))
    mass, reach = np.zeros_like(o), np.zeros((tokens, q_heads, 1))
    grp = q_heads // heads
    for b in range(len(kv_len)):
        n, L = cu[b + 1] - cu[b], max(int(kv_len[b]), 0)
        if n <= 0:
            continue
        k, there = cache.values(0, table[b], L)
        v, _ = cache.values(1, table[b], L)
        if shared is not None:
            for g in range(len(shared[2])):
                P = int(shared[2][g])
                if shared[0][g] <= b < shared[0][g + 1] and 0 < P <= L - n:
                    k[:, :P], there[:P] = cache.values(0, shared[1][g], P)
                    v[:, :P] = cache.values(1, shared[1][g], P)[0]
        v = np.where(there[None, :, None], v, 0.0)
        j = np.arange(L)
        for i in range(n):
            p = L - n + i
            sees = there & (j <= p) if causal else there.copy()
            if window:
                sees &= (j > p - window) | (j < sinks)
            if not sees.any():
                continue
            r = cu[b] + i
            for h in range(q_heads):
                kk, vv = k[h // grp][sees], v[h // grp][sees]
                with np.errstate(invalid="ignore", over="ignore"):
                    s = scale * (kk @ q[r, h].astype(np.float64))
                    if s.max() == -np.inf:
                        continue
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    o[r, h] = w @ vv
                    mass[r, h] = w @ np.abs(vv)
                    reach[r, h] = scale * (np.abs(kk) @ np.abs(q[r, h].astype(np.float64))).max()
    return o, mass, reach


def check_attention(got, q, cache, table, kv_len, cu, heads, scale, out_bf16, **kw):
    """got against the definition, within the bound that kv_cases derives (parts
    and their join are among its roundings)."""
    o, mass, reach = attention(q, cache, table, kv_len, cu, heads, float(np.float32(scale)), **kw)
    bound = kc.attention_bound(mass, reach, q.shape[2], max(list(kv_len) + [1]), out_bf16)
    assert np.array_equal(np.isnan(got), np.isnan(o))
    bad = kc.outside(got, o, bound, out_bf16)
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], o[bad][:5], bound[bad][:5])
