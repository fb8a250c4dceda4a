"""Plain 64-bit implementations of the norm, the E4M3 KV cache and attention
over it, token by token on the CPU, for the GPU tests to compare with.

The E4M3 encoder is the oracle's; everything else is numpy."""
import numpy as np
import torch

import oracle

NAN_CODE = 0x7F


def bf16(a):
    """fp32 values rounded to bf16 values (nearest even), as fp32."""
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.float32)).bfloat16().float().numpy()


def encode(v):
    """fp32 array -> E4M3 codes, the oracle's encoder."""
    v = np.ascontiguousarray(v, dtype=np.float32)
    return oracle.quantize(v.reshape(-1), np.float32(1.0)).reshape(v.shape)


_TABLE = None


def decode(c):
    global _TABLE
    if _TABLE is None:
        _TABLE = oracle.dequantize(np.arange(256, dtype=np.uint8), np.float32(1.0)).astype(np.float64)
    return _TABLE[c]


def page_scale(x):
    """The smallest power of two s >= 2^-126 with |x| <= 448 s, x finite."""
    a = np.abs(x[np.isfinite(x)]).astype(np.float64)
    a = float(a.max()) if a.size else 0.0
    s = 2.0 ** -126
    while a > 448.0 * s:
        s *= 2.0
    return s


class Cache:
    """A KV cache of dense pages on the CPU: codes [pages, heads, T, D]."""

    def __init__(self, pages, heads, T, D, rng):
        self.shape = (pages, heads, T, D)
        # what earlier users left: any byte, NaN codes among them
        self.codes = [rng.integers(0, 256, self.shape, dtype=np.uint8) for _ in range(2)]
        self.scale = [np.exp2(rng.integers(-3, 4, (pages, heads))).astype(np.float32) for _ in range(2)]

    def page(self, table, pos):
        c = pos // self.shape[2]
        if pos < 0 or c >= table.shape[0]:
            return -1
        p = int(table[c])
        return p if 0 <= p < self.shape[0] else -1

    def write(self, k, v, table, kv_len, cu):
        """Rows of k, v [tokens, heads, D] fp32, page by page."""
        pages, heads, T, D = self.shape
        for b in range(len(kv_len)):
            n = cu[b + 1] - cu[b]
            rows = {}  # page place -> [(slot, row)]
            for i in range(n):
                pos = kv_len[b] - n + i
                if self.page(table[b], pos) >= 0:
                    rows.setdefault(pos // T, []).append((pos % T, cu[b] + i))
            for c, entries in rows.items():
                p, lo = self.page(table[b], c * T), entries[0][0]
                for which, x in enumerate((k, v)):
                    for h in range(heads):
                        new = np.stack([x[r, h] for _, r in entries])
                        s = page_scale(new)
                        if lo > 0:
                            old = float(self.scale[which][p, h])
                            s = max(s, old)
                            if s > old:
                                kept = decode(self.codes[which][p, h, :lo]) * (old / s)
                                self.codes[which][p, h, :lo] = encode(kept)
                        for (slot, _), row in zip(entries, new):
                            self.codes[which][p, h, slot] = encode(row.astype(np.float64) / s)
                        self.scale[which][p, h] = s

    def values(self, which, table, length):
        """[heads, length, D] in 64 bits, and which positions have a token."""
        pages, heads, T, D = self.shape
        out, there = np.zeros((heads, length, D)), np.zeros(length, bool)
        for pos in range(0, length, T):
            p, m = self.page(table, pos), min(T, length - pos)
            if p >= 0:
                out[:, pos:pos + m] = decode(self.codes[which][p, :, :m]) * self.scale[which][p].astype(np.float64)[:, None, None]
                there[pos:pos + m] = True
        return out, there

    def packed(self, which):
        """The codes in the cache's byte order."""
        P, H, T, D = self.shape
        c = self.codes[which]
        if which == 0:
            c = c.reshape(P, H, T // 16, 16, D // 16, 16).transpose(0, 1, 2, 4, 3, 5)
        else:
            c = c.reshape(P, H, T // 4, 4, D).transpose(0, 1, 2, 4, 3)
        return np.ascontiguousarray(c).reshape(P, H, T, D)

    def to(self, dev):
        """(k_cache, v_cache, k_scale, v_scale) on the device."""
        return tuple(torch.from_numpy(self.packed(w)).to(dev) for w in (0, 1)) + \
            tuple(torch.from_numpy(self.scale[w].copy()).to(dev) for w in (0, 1))


def tables(kv_len, T, rng, spare=2):
    """A block table over pages in any order, -1 past a sequence's pages."""
    need = [-(-x // T) for x in kv_len]
    order = rng.permutation(sum(need) + spare)
    table = np.full((len(kv_len), max(need + [1])), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, sum(need) + spare


def same_codes(got, want):
    """Codes equal; NaN codes may differ in their sign, zeros in theirs."""
    g, w = decode(got), decode(want)
    return np.array_equal(np.nan_to_num(g, nan=1e9), np.nan_to_num(w, nan=1e9))


def attention(q, cache, table, kv_len, cu, heads, scale, causal=True, window=0):
    """o, and for tolerances: the sums of w|v| / sum w, and the largest
    scale * sum |q||k| of the row, both [tokens, q_heads, ...]."""
    tokens, q_heads, D = q.shape
    o = np.zeros((tokens, q_heads, D))
    mass, reach = np.zeros_like(o), np.zeros((tokens, q_heads, 1))
    grp = q_heads // heads
    for b in range(len(kv_len)):
        n, L = cu[b + 1] - cu[b], int(kv_len[b])
        if n <= 0:
            continue
        k, there = cache.values(0, table[b], L)
        v, _ = cache.values(1, table[b], L)
        v = np.where(there[None, :, None], v, 0.0)
        j = np.arange(L)
        for i in range(n):
            p = L - n + i
            sees = there & (j <= p) if causal else there.copy()
            if window:
                sees &= j > p - window
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


def attention_bound(mass, reach, D, L, out_bf16):
    """|error| of an fp32 evaluation before its result is rounded, element by
    element: scores are sums of D products (D + 8 roundings of their absolute
    sum, which the exponential turns into a relative error of each weight, in
    numerator and denominator), the sums over tokens add a rounding for each 16
    of them and a few for the exponential, the split and the division.  With
    bf16 outputs each weight may be rounded to 11 bits (2^-11)."""
    u = 2.0 ** -24
    rel = 2 * (D + 8) * u * reach + 2 * (L / 16 + 64) * u
    return mass * (rel + 2.0 ** -11 if out_bf16 else rel) + 1e-37


def outside(got, o, bound, out_bf16):
    """Where got is not the rounding of a value within the bound of o (rounding
    is monotone: it lies between the ends' roundings)."""
    lo, hi = o - bound, o + bound
    if out_bf16:
        lo, hi = bf16(lo).astype(np.float64), bf16(hi).astype(np.float64)
    else:
        lo, hi = lo.astype(np.float32).astype(np.float64), hi.astype(np.float32).astype(np.float64)
    return (got < lo) | (got > hi)
