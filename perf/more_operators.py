"""A decode loop's other operators around the E4M3 KV cache, as measurable
cases.

A case is a dict of plain values; its "kind" names the operator:

  plan    from the tokens that each request brings: lengths, row offsets,
          pages from a free list (and back to it from requests that ended),
          every row's position and cache slot
  rope    RMS norms of the heads of queries and keys and the rotation by
          position, in one pass over columns of the QKV projection
  sinks   attention over the cache through a sliding window, with a few first
          tokens that stay visible
  shared  attention over the cache for groups of sequences that share their
          first tokens' pages

`own` says whether run() computes the operator in plain torch operations or
calls this framework.  Sequences are ragged; sequence b brings n[b] tokens,
which are the last ones of its kv[b].
"""
import math

import torch

own = False

DEV = "cuda:0"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "bf16": 2}
F8 = torch.float8_e4m3fn
EPS = 1e-6


def listed():
    return [
        # page bookkeeping of a decode step: few sequences cross into a page
        {"name": "plan_decode_b64", "kind": "plan", "seqs": 64, "q": 1, "kv": 4000, "ragged": True, "page": 16, "ended": 3,
         "room": 1.5},
        # a batch of long prompts and chunks of prompts comes in, others have
        # ended, and the last ones' pages run out
        {"name": "plan_prompts_b48", "kind": "plan", "seqs": 48, "q": 8192, "kv": 12000, "ragged": True, "page": 16,
         "ended": 9, "room": 0.95},
        # a decode step of 64 sequences: latency
        {"name": "rope_decode_b64", "kind": "rope", "rows": 64, "far": 8000, "heads": 32, "kv_heads": 8, "dim": 128,
         "rot": 128, "interleaved": False, "norm": True, "dtype": "bf16", "out": "bf16"},
        # prompts of 8192 tokens in all: bytes
        {"name": "rope_prompt_8192", "kind": "rope", "rows": 8192, "far": 8192, "heads": 32, "kv_heads": 8, "dim": 128,
         "rot": 128, "interleaved": False, "norm": True, "dtype": "bf16", "out": "bf16"},
        # chunks far into long sequences, fp32, neighbouring pairs, a part of
        # each head rotated, an odd number of rows
        {"name": "rope_chunk_fp32", "kind": "rope", "rows": 1333, "far": 120000, "heads": 28, "kv_heads": 4, "dim": 96,
         "rot": 64, "interleaved": True, "norm": True, "dtype": "fp32", "out": "fp32"},
        # one decode step of one sequence: latency
        {"name": "sinks_b1", "kind": "sinks", "seqs": 1, "q": 1, "kv": 5000, "ragged": False, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "window": 1024, "sinks": 4, "dtype": "bf16", "out": "bf16"},
        # one decode step of 32 long sequences: the bytes of their windows
        {"name": "sinks_b32_32k", "kind": "sinks", "seqs": 32, "q": 1, "kv": 32768, "ragged": True, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "window": 8192, "sinks": 64, "dtype": "bf16", "out": "bf16"},
        # a long prompt: the matrix cores
        {"name": "sinks_prompt_8192", "kind": "sinks", "seqs": 1, "q": 8192, "kv": 8192, "ragged": False, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "window": 2048, "sinks": 4, "dtype": "bf16", "out": "bf16"},
        # chunks of prompts behind a history, fp32, a head group and a head
        # size off the powers of two, more sinks than a page or two
        {"name": "sinks_chunk_fp32", "kind": "sinks", "seqs": 4, "q": 300, "kv": 4000, "ragged": True, "heads": 28,
         "kv_heads": 4, "dim": 96, "page": 16, "window": 700, "sinks": 100, "dtype": "fp32", "out": "fp32"},
        # a few requests behind a short system prompt: latency
        {"name": "shared_b8_1k", "kind": "shared", "groups": 1, "seqs": 8, "q": 1, "prefix": 1024, "kv": 200, "ragged": True,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "dtype": "bf16", "out": "bf16"},
        # a decode step of 64 requests behind a long one
        {"name": "shared_b64_16k", "kind": "shared", "groups": 1, "seqs": 64, "q": 1, "prefix": 16384, "kv": 800,
         "ragged": True, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "dtype": "bf16", "out": "bf16"},
        # three documents, several questions about each: their prefill
        {"name": "shared_chunk_fp32", "kind": "shared", "groups": 3, "seqs": 5, "q": 60, "prefix": 6000, "kv": 200,
         "ragged": True, "heads": 16, "kv_heads": 2, "dim": 64, "page": 32, "dtype": "fp32", "out": "fp32"},
    ]


def _log(rng, lo, hi):
    """An integer in [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


HEADS = [(32, 8, 128), (32, 8, 128), (32, 32, 128), (28, 4, 128), (16, 2, 64), (12, 4, 96), (20, 20, 80), (8, 1, 256)]


def draw(rng):
    kind = rng.choice(["plan", "rope", "rope", "sinks", "sinks", "shared", "shared"])
    if kind == "plan":
        seqs = _log(rng, 1, 512)
        q = 1 if rng.random() < 0.4 else _log(rng, 1, min(8192, 200_000 // seqs))
        return {"kind": kind, "seqs": seqs, "q": q, "kv": q + _log(rng, 1, min(12000, 2_000_000 // seqs)),
                "ragged": rng.random() < 0.7, "page": rng.choice([16, 16, 32, 64, 128, 256]),
                "ended": rng.choice([0, 0, seqs // 8, seqs // 3]), "room": rng.choice([1.2, 2.0, 0.9])}
    heads, kv_heads, dim = rng.choice(HEADS)
    case = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": rng.choice(["bf16", "bf16", "fp32"])}
    case["out"] = "fp32" if case["dtype"] == "fp32" else rng.choice(["bf16", "bf16", "fp32"])
    if kind == "rope":
        case["rows"] = _log(rng, 1, 8192 * 40 * 128 * 2 // ((heads + kv_heads) * dim * SIZE[case["out"]]))
        case["rows"] = min(case["rows"], 8192)
        case["far"] = case["rows"] + _log(rng, 1, 120000)
        case["rot"] = dim if rng.random() < 0.6 else 2 * rng.randint(1, dim // 2)
        case["interleaved"], case["norm"] = rng.random() < 0.4, rng.random() < 0.7
        return case
    case["page"], case["ragged"] = rng.choice([16, 16, 32, 64, 128]), rng.random() < 0.7
    most = 40_000_000 // (kv_heads * dim)  # tokens of all sequences
    if kind == "sinks":
        case["window"], case["sinks"] = _log(rng, 16, 6000), _log(rng, 1, 300)
        if rng.random() < 0.6:  # decode, of one token or a few
            case["seqs"], case["q"] = _log(rng, 1, 32), rng.choice([1, 1, 1, 2, 5])
            case["kv"] = max(case["q"], _log(rng, 16, min(32768, 4 * most // case["seqs"])))
        else:
            case["seqs"] = _log(rng, 1, 8)
            case["q"] = _log(rng, 7, 2000 // case["seqs"])
            case["kv"] = case["q"] if rng.random() < 0.5 else _log(rng, case["q"], 4500)
        return case
    case["groups"] = rng.choice([1, 1, 1, 2, 4])
    case["seqs"] = _log(rng, 2, 64 // case["groups"])  # of each group
    total = case["seqs"] * case["groups"]
    case["prefix"] = _log(rng, 64, min(12000, 28 * most // total))
    case["q"] = rng.choice([1, 1, 1, 4, _log(rng, 5, max(5, min(1000, 8_000_000 // case["prefix"]) // total))])
    case["kv"] = case["q"] + _log(rng, 1, 1000)  # tokens of its own that a sequence has
    return case


def _spread(top, b, least=8):
    """Lengths of a ragged batch: from a `least`-th of the top to the top."""
    lo = max(1, top // least)
    return lo + int((top - lo) * (1.0 - (b * 0.6180339887) % 1.0))


def _prefix(case):
    """Tokens that each group shares: whole pages."""
    T = case["page"]
    return [max(1, (_spread(case["prefix"], g, 2) if case["ragged"] else case["prefix"]) // T) * T for g in range(case["groups"])]


def _lengths(case):
    """(n, kv) of every sequence: new tokens, and all tokens with them."""
    seqs = case["seqs"] * case.get("groups", 1)
    kv = [_spread(case["kv"], b) if case["ragged"] else case["kv"] for b in range(seqs)]
    n = [_spread(case["q"], b + 3, 4) if case["ragged"] else case["q"] for b in range(seqs)]
    n = [min(a, b) for a, b in zip(n, kv)]
    if case["kind"] == "shared":
        kv = [x + _prefix(case)[b // case["seqs"]] for b, x in enumerate(kv)]
    return n, kv


def _gone(case):
    """The sequences that have ended before a plan: spread over the batch."""
    return [b * case["ended"] // case["seqs"] != (b + 1) * case["ended"] // case["seqs"] for b in range(case["seqs"])]


# ------------------------------------------------------------ plain pieces --

def _e4m3(v):
    """fp32 values to the E4M3 values nearest to them, saturating."""
    return v.clamp(-448.0, 448.0).to(F8)


def _page_scale(a):
    """The smallest power of two s >= 2^-126 with a <= 448 s."""
    m, e = torch.frexp(a)  # a = m 2^e, 1/2 <= m < 1; 448 = 7/8 2^9
    e = torch.where(m > 0.875, e - 8, e - 9).clamp_min(-126)
    return torch.ldexp(torch.ones_like(a), torch.where(a > 0, e, torch.full_like(e, -126)))


# A page's tokens lie in blocks of 16.  K: by 16-byte pieces of a token,
# [dim / 16][16 tokens][16]; V: by groups of four tokens, [4 groups][dim][4].

def _pack_k(x):
    *o, t, d = x.shape
    return x.reshape(*o, t // 16, 16, d // 16, 16).transpose(-3, -2).reshape(*o, t, d)


def _unpack_k(x):
    *o, t, d = x.shape
    return x.reshape(*o, t // 16, d // 16, 16, 16).transpose(-3, -2).reshape(*o, t, d)


def _pack_v(x):
    *o, t, d = x.shape
    return x.reshape(*o, t // 4, 4, d).transpose(-2, -1).reshape(*o, t, d)


def _unpack_v(x):
    *o, t, d = x.shape
    return x.reshape(*o, t // 4, d, 4).transpose(-2, -1).reshape(*o, t, d)


# ------------------------------------------------------------------ inputs --

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 7919 + 29)
    return g


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _activations(g, *shape):
    """N(0, 1) with a few large channels, as activations and keys have them."""
    gain = torch.exp(0.5 * torch.randn(shape[-1], device=DEV, generator=g))
    return torch.randn(*shape, device=DEV, generator=g).mul_(gain)


def _prepare_plan(case, st, g):
    T, (n, kv), gone = case["page"], _lengths(case), _gone(case)
    n = [0 if e else x for x, e in zip(n, gone)]
    held = [x - y for x, y in zip(kv, n)]  # before this step
    has = [-(-x // T) for x in held]
    need = [0 if e else -(-x // T) - h for x, h, e in zip(kv, has, gone)]
    back = sum(h for h, e in zip(has, gone) if e)
    free = max(0, int(sum(need) * case["room"]) - back) + 1
    pages = sum(has) + free
    order = torch.randperm(pages, device=DEV, generator=g).to(torch.int32)
    cols = max(h + x for h, x in zip(has, need)) + 2
    col = torch.arange(cols, device=DEV)
    first = _ints([sum(has[:b]) for b in range(len(has))])
    at = (first[:, None] + col[None]).clamp_max(pages - 1)
    st["block_table"] = torch.where(col[None] < _ints(has)[:, None], order[at.long()], torch.full_like(at, -1, dtype=torch.int32))
    st["free_pages"] = torch.full((pages,), -7, dtype=torch.int32, device=DEV)
    st["free_pages"][:free] = order[sum(has):]
    st["free_count"] = _ints([free])
    st["new_tokens"], st["kv_len"], st["ended"] = _ints(n), _ints(held), _ints([int(e) for e in gone])
    # the first page of every other ended sequence is one that others share
    st["first_own"] = _ints([b % 2 if e else 0 for b, e in enumerate(gone)])
    st["tokens"] = (sum(n) // 16 + 1) * 16  # a padded batch
    st["kv_out"], st["cu_q"], st["left"] = _ints([0] * len(n)), _ints([0] * (len(n) + 1)), _ints([0])
    st["positions"] = torch.empty(st["tokens"], dtype=torch.int32, device=DEV)
    st["slots"] = torch.empty(st["tokens"], dtype=torch.int64, device=DEV)


def _prepare_rope(case, st, g):
    d, rows, half = case["dim"], case["rows"], case["rot"] // 2
    st["qkv"] = _activations(g, rows, (case["heads"] + 2 * case["kv_heads"]) * d).to(DTYPES[case["dtype"]])
    if case["norm"]:
        st["q_gamma"], st["k_gamma"] = (1.0 + 0.1 * torch.randn(d, device=DEV, generator=g) for _ in range(2))
    # a few sequences' rows one after another, the longest ending at the last position
    cuts = [0, rows // 5, rows // 2, rows]
    pos = torch.arange(rows, device=DEV)
    for i, (a, b) in enumerate(zip(cuts, cuts[1:])):
        pos[a:b] += (case["far"] - (b - a)) * (i + 1) // 3 - a
    st["positions"] = pos.to(torch.int32)
    angle = torch.arange(case["far"], device=DEV, dtype=torch.float64)[:, None] * \
        10000.0 ** (-torch.arange(half, device=DEV, dtype=torch.float64) / max(half, 1))
    st["table"] = torch.cat([angle.cos(), angle.sin()], dim=1).float()  # of all positions, as a model holds it
    st["q"] = torch.empty(rows, case["heads"], d, dtype=DTYPES[case["out"]], device=DEV)
    st["k"] = torch.empty(rows, case["kv_heads"], d, dtype=DTYPES[case["out"]], device=DEV)


def prepare(case, seed):
    g = _gen(seed)
    st = {"case": case}
    if case["kind"] in ("plan", "rope"):
        (_prepare_plan if case["kind"] == "plan" else _prepare_rope)(case, st, g)
        return st
    n, kv = _lengths(case)
    T, hk, d = case["page"], case["kv_heads"], case["dim"]
    cu = [sum(n[:b]) for b in range(len(n) + 1)]
    shared = [_prefix(case)[b // case["seqs"]] // T for b in range(len(n))] if case["kind"] == "shared" else [0] * len(n)
    need = [-(-x // T) - s for x, s in zip(kv, shared)]
    prefix = [p // T for p in _prefix(case)] if case["kind"] == "shared" else []
    pages = sum(need) + sum(prefix) + 3  # a pool with room left; pages come in any order
    order = torch.randperm(pages, device=DEV, generator=g).to(torch.int32)
    cols = max(x + s for x, s in zip(need, shared))
    table = torch.full((len(n), cols), -1, dtype=torch.int32, device=DEV)
    at = sum(prefix)
    for b, (x, s) in enumerate(zip(need, shared)):
        if s:
            p0 = sum(prefix[:b // case["seqs"]])
            table[b, :s] = order[p0:p0 + s]
        table[b, s:s + x] = order[at:at + x]
        at += x
    st["block_table"], st["kv_len"], st["cu_q"] = table, _ints(kv), _ints(cu)
    st["max_q"], st["max_kv"], st["tokens"] = max(n), max(kv), cu[-1]
    if case["kind"] == "shared":
        st["group_seq"] = _ints([g * case["seqs"] for g in range(case["groups"] + 1)])
        st["prefix_len"] = _ints(_prefix(case))
        st["prefix_table"] = table[::case["seqs"], :max(prefix)]
        st["max_prefix"], st["max_own"] = max(_prefix(case)), max(x - s * T for x, s in zip(kv, shared))
        st["max_group_q"] = max(cu[(g + 1) * case["seqs"]] - cu[g * case["seqs"]] for g in range(case["groups"]))
    for name in ("k", "v"):
        # a cache in use: pages of E4M3 values with the scale of their largest
        x = _activations(g, pages, hk, T, d)
        x.mul_(torch.exp(torch.randn(pages, hk, 1, 1, device=DEV, generator=g) * 0.3))
        s = _page_scale(x.abs().amax(dim=(2, 3)))
        codes = _e4m3(x.div_(s[:, :, None, None])).view(torch.uint8)
        del x
        # what tokens that have gone left behind in a page's last slots
        last = torch.full((pages,), T, device=DEV, dtype=torch.int64)
        row = _ints([-(-x // T) - 1 for x in kv]).long()
        last[table[torch.arange(len(kv), device=DEV), row].long()] = _ints([(x - 1) % T + 1 for x in kv]).long()
        gone = torch.arange(T, device=DEV)[None] >= last[:, None]
        codes.masked_fill_(gone[:, None, :, None], 0x7F)
        st[name + "_cache"] = (_pack_k if name == "k" else _pack_v)(codes)
        st[name + "_scale"] = s
    st["q"] = _activations(g, cu[-1], case["heads"], d).to(DTYPES[case["dtype"]])
    st["o"] = torch.empty(cu[-1], case["heads"], d, dtype=DTYPES[case["out"]], device=DEV)
    st["sm_scale"] = d ** -0.5
    return st


def _columns(st):
    """Queries and keys: columns of the QKV projection."""
    c, x = st["case"], st["qkv"]
    x = x.view(x.shape[0], -1, c["dim"])
    return x[:, :c["heads"]], x[:, c["heads"]:c["heads"] + c["kv_heads"]]


# ------------------------------------------------------------- plain forms --

def _plain_plan(st):
    T, table, pages = st["case"]["page"], st["block_table"], st["free_pages"].shape[0]
    held, n, ended = st["kv_len"].long(), st["new_tokens"].long(), st["ended"] != 0
    old = torch.where(ended, torch.zeros_like(held), held)
    kv = old + n
    cu = torch.cat([torch.zeros_like(n[:1]), torch.cumsum(n, 0)])
    col = torch.arange(table.shape[1], device=DEV)[None]
    # pages that come back, in order of sequence and column, on top of the free ones
    back = ended[:, None] & (col >= st["first_own"][:, None]) & (col < ((held + T - 1) // T)[:, None]) & (table >= 0) & (table < pages)
    place = st["free_count"].long() + torch.cumsum(back.reshape(-1), 0) - 1
    stack = torch.cat([st["free_pages"], st["free_pages"][:1]])  # with a place for what stays
    stack.scatter_(0, torch.where(back.reshape(-1), place, torch.full_like(place, pages)), table.reshape(-1))
    st["free_pages"].copy_(stack[:-1])
    top = st["free_count"].long() + back.sum()
    # pages that are taken, in the same order, from the top
    first, end = (old + T - 1) // T, ((kv + T - 1) // T).clamp_max(table.shape[1])
    need = (end - first).clamp_min(0)
    rank = (torch.cumsum(need, 0) - need)[:, None] + col - first[:, None]
    at = top - 1 - rank
    page = torch.where(at >= 0, st["free_pages"][at.clamp(0, pages - 1)], torch.full_like(at, -1, dtype=torch.int32))
    table.copy_(torch.where((col >= first[:, None]) & (col < end[:, None]), page, table))
    st["kv_out"].copy_(kv)
    st["cu_q"].copy_(cu)
    st["left"].copy_(top - need.sum())
    t = torch.arange(st["tokens"], device=DEV)
    b = torch.searchsorted(cu[1:], t, right=True).clamp_max(len(n) - 1)
    pos = torch.where(t < cu[-1], kv[b] - (cu[b + 1] - t), torch.full_like(t, -1))
    page = table[b, (pos // T).clamp(0, table.shape[1] - 1)].long()
    there = (pos >= 0) & (pos // T < table.shape[1]) & (page >= 0) & (page < pages)
    st["positions"].copy_(pos)
    st["slots"].copy_(torch.where(there, page * T + pos % T, torch.full_like(pos, -1)))


def _plain_rope(st):
    c = st["case"]
    half, rot = c["rot"] // 2, c["rot"]
    cs = st["table"][st["positions"].long()][:, None]
    cos, sin = cs[..., :half], cs[..., half:]
    for x, gamma, out in zip(_columns(st), ("q_gamma", "k_gamma"), ("q", "k")):
        v = x.float()
        if c["norm"]:
            v = v * (1.0 / torch.sqrt((v * v).mean(dim=2, keepdim=True) + EPS)) * st[gamma]
        if c["interleaved"]:
            a, b = v[..., 0:rot:2], v[..., 1:rot:2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(2)
        else:
            a, b = v[..., :half], v[..., half:rot]
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
        st[out].copy_(torch.cat([turned, v[..., rot:]], dim=-1))


def _plain_attend(st):
    c = st["case"]
    T, hk, d = c["page"], c["kv_heads"], c["dim"]
    grp, nq = c["heads"] // hk, st["max_q"]
    cu, kv = st["cu_q"].long(), st["kv_len"].long()
    table = st["block_table"].long().clamp_min(0)
    j = torch.arange(table.shape[1] * T, device=DEV)
    there = j[None] < kv[:, None]  # [seqs, L]

    def dense(cache, scale, unpack):
        x = unpack(st[cache][table]).view(F8).float() * st[scale][table][..., None, None]
        x = x.transpose(1, 2).reshape(len(kv), hk, -1, d)
        return torch.where(there[:, None, :, None], x, torch.zeros((), device=DEV))

    i = torch.arange(nq, device=DEV)
    n = cu[1:] - cu[:-1]
    row = (cu[:-1, None] + i[None]).clamp_max(st["tokens"] - 1)  # [seqs, nq]
    q = st["q"].float()[row].reshape(len(kv), nq, hk, grp, d).permute(0, 2, 3, 1, 4).reshape(len(kv), hk, grp * nq, d)
    s = torch.matmul(q, dense("k_cache", "k_scale", _unpack_k).transpose(2, 3)) * st["sm_scale"]
    at = (kv - n)[:, None] + i[None]  # the queries' positions
    sees = there[:, None, :] & (j[None, None] <= at[:, :, None])
    if c["kind"] == "sinks":
        sees &= (j[None, None] > at[:, :, None] - c["window"]) | (j < c["sinks"])
    sees = sees[:, None, None].expand(-1, 1, grp, -1, -1).reshape(len(kv), 1, grp * nq, -1)
    s = s.masked_fill_(~sees, -math.inf)
    top = s.amax(dim=-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    del s
    total = p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p, dense("v_cache", "v_scale", _unpack_v))
    o = torch.where(total == 0, torch.zeros_like(o), o / total)
    o = o.reshape(len(kv), hk, grp, nq, d).permute(0, 3, 1, 2, 4).reshape(len(kv), nq, c["heads"], d)
    t = torch.arange(st["tokens"], device=DEV)
    b = torch.searchsorted(cu[1:], t, right=True)
    st["o"].copy_(o[b, t - cu[b]])


# ------------------------------------------------------------------- a pass --

def _pass_own(st):
    from luisaml_amd import capi
    c = st["case"]
    if c["kind"] == "plan":
        capi.kv_cache_plan(st["new_tokens"], st["kv_len"], st["block_table"], st["free_pages"], st["free_count"], c["page"],
                           ended=st["ended"], first_own=st["first_own"], kv_len_out=st["kv_out"], cu_q=st["cu_q"],
                           left=st["left"], positions=st["positions"], slots=st["slots"])
        return
    if c["kind"] == "rope":
        q, k = _columns(st)
        capi.qk_norm_rope(q, k, st["positions"], st["table"], q_gamma=st.get("q_gamma"), k_gamma=st.get("k_gamma"), eps=EPS,
                          interleaved=c["interleaved"], q_out=st["q"], k_out=st["k"])
        return
    cache = (st["k_cache"], st["v_cache"], st["k_scale"], st["v_scale"], st["block_table"], st["kv_len"], st["cu_q"])
    if c["kind"] == "sinks":
        capi.attention(st["q"], *cache, st["max_q"], st["max_kv"], st["sm_scale"], window=c["window"], sinks=c["sinks"],
                       out=st["o"])
    else:
        capi.attention_shared(st["q"], *cache, st["group_seq"], st["prefix_table"], st["prefix_len"], st["max_q"],
                              st["max_own"], st["max_group_q"], st["max_prefix"], st["sm_scale"], out=st["o"])


PLAIN = {"plan": _plain_plan, "rope": _plain_rope, "sinks": _plain_attend, "shared": _plain_attend}


def run(state):
    kind = state["case"]["kind"]
    (_pass_own if own else PLAIN[kind])(state)
    if kind == "plan":
        return {k: state[k] for k in ("kv_out", "cu_q", "left", "positions", "slots", "block_table", "free_pages")}
    if kind == "rope":
        return {"q": state["q"], "k": state["k"]}
    return state["o"]


# ------------------------------------------------------- 64-bit expectation --

def _exact_plan(st):
    T = st["case"]["page"]
    table, stack = st["block_table"].tolist(), st["free_pages"].tolist()
    n, held, gone, own_from = (st[k].tolist() for k in ("new_tokens", "kv_len", "ended", "first_own"))
    pages, top = len(stack), st["free_count"].item()
    for b, e in enumerate(gone):
        for p in table[b][own_from[b]:-(-held[b] // T)] if e else []:
            if 0 <= p < pages:
                stack[top] = p
                top += 1
    kv, cu, positions, slots = [], [0], [], []
    for b, e in enumerate(gone):
        start = 0 if e else held[b]
        kv.append(start + n[b])
        cu.append(cu[-1] + n[b])
        for c in range(-(-start // T), min(-(-kv[b] // T), len(table[b]))):
            top -= 1
            table[b][c] = stack[top] if top >= 0 else -1
        for p in range(start, kv[b]):
            page = table[b][p // T] if p // T < len(table[b]) else -1
            positions.append(p)
            slots.append(page * T + p % T if 0 <= page < pages else -1)
    spare = [-1] * (st["tokens"] - len(positions))
    out = {"kv_out": kv, "cu_q": cu, "left": [top], "positions": positions + spare, "slots": slots + spare,
           "block_table": table, "free_pages": stack}
    return {k: torch.tensor(v, dtype=torch.int64, device=DEV) for k, v in out.items()}


def _exact_rope(st):
    c = st["case"]
    out = {}
    turn = st["table"].double()[st["positions"].long()]
    turn = torch.complex(turn[:, :c["rot"] // 2], turn[:, c["rot"] // 2:])[:, None]
    for x, gamma, name in zip(_columns(st), ("q_gamma", "k_gamma"), ("q", "k")):
        v = x.double()
        if c["norm"]:
            v = v / torch.sqrt(v.square().sum(dim=2, keepdim=True) / c["dim"] + EPS) * st[gamma].double()
        r = v[..., :c["rot"]]
        if c["interleaved"]:
            pairs = torch.view_as_complex(r.reshape(*r.shape[:2], -1, 2).contiguous()) * turn
            r = torch.view_as_real(pairs).reshape(r.shape)
        else:
            pairs = torch.complex(*r.reshape(*r.shape[:2], 2, -1).unbind(2)) * turn
            r = torch.cat([pairs.real, pairs.imag], dim=2)
        out[name] = torch.cat([r, v[..., c["rot"]:]], dim=2)
    return out


def _order_k(T, d):
    """Where element (token, d) of a page lies, as a [T, d] table."""
    t, e = torch.arange(T, device=DEV)[:, None], torch.arange(d, device=DEV)[None]
    return (t // 16) * (16 * d) + (e // 16) * 256 + (t % 16) * 16 + e % 16


def _order_v(T, d):
    t, e = torch.arange(T, device=DEV)[:, None], torch.arange(d, device=DEV)[None]
    return (t // 4) * (4 * d) + e * 4 + t % 4


def _sequence(st, name, order, b, upto):
    """The first `upto` tokens of sequence b in 64 bits, [kv heads, upto, d]."""
    c = st["case"]
    T, d, hk = c["page"], c["dim"], c["kv_heads"]
    pages = st["block_table"][b, :-(-upto // T)].long()
    x = st[name + "_cache"].reshape(-1, hk, T * d)[pages][:, :, order.reshape(-1)].view(F8).double()
    x = x * st[name + "_scale"].double()[pages][:, :, None]
    return x.reshape(len(pages), hk, T, d).transpose(0, 1).reshape(hk, -1, d)[:, :upto]


def _exact_attend(st):
    c = st["case"]
    n, kv = _lengths(c)
    d, hk = c["dim"], c["kv_heads"]
    grp = c["heads"] // hk
    o = torch.zeros(st["tokens"], c["heads"], d, dtype=torch.float64, device=DEV)
    t0 = 0
    for b in range(len(kv)):
        k = _sequence(st, "k", _order_k(c["page"], d), b, kv[b])
        v = _sequence(st, "v", _order_v(c["page"], d), b, kv[b])
        for i0 in range(0, n[b], 1024):
            i1 = min(n[b], i0 + 1024)
            at = torch.arange(kv[b] - n[b] + i0, kv[b] - n[b] + i1, device=DEV)[:, None]
            j = torch.arange(kv[b], device=DEV)[None]
            hidden = j > at
            if c["kind"] == "sinks":
                hidden = hidden | ((j <= at - c["window"]) & (j >= c["sinks"]))
            for h in range(hk):
                heads = slice(h * grp, (h + 1) * grp)
                q = st["q"][t0 + i0:t0 + i1, heads].double().transpose(0, 1).reshape(-1, d)
                s = (q @ k[h].t().contiguous() * st["sm_scale"]).reshape(grp, i1 - i0, -1)
                w = torch.softmax(s.masked_fill(hidden[None], -math.inf), dim=2).reshape(grp * (i1 - i0), -1)
                o[t0 + i0:t0 + i1, heads] = (w @ v[h]).reshape(grp, i1 - i0, d).transpose(0, 1)
        t0 += n[b]
    return o


def exact(case, seed):
    st = prepare(case, seed)
    return {"plan": _exact_plan, "rope": _exact_rope, "sinks": _exact_attend, "shared": _exact_attend}[case["kind"]](st)


# -------------------------------------------------------------------- work --

def _pairs(case):
    """Of all queries of one head: tokens seen; and the tokens that any sees."""
    pairs = seen = 0
    w, sinks = case.get("window", 10 ** 9), case.get("sinks", 0)
    for n, kv in zip(*_lengths(case)):
        pairs += sum(min(p + 1, w + min(sinks, max(0, p + 1 - w))) for p in range(kv - n, kv))
        lo = max(0, kv - n - w + 1)
        seen += kv - lo + min(sinks, lo)
    if case["kind"] == "shared":  # a prefix once for its group
        seen -= (case["seqs"] - 1) * sum(_prefix(case))
    return pairs, seen


def work(case):
    """Bytes read once and written once, and operations (a multiply-add is two)."""
    if case["kind"] == "plan":
        T, gone, (n, kv) = case["page"], _gone(case), _lengths(case)
        n = [0 if e else x for x, e in zip(n, gone)]
        held = [x - y for x, y in zip(kv, n)]
        taken = sum(-(-x // T) - -(-h // T) for x, h, e in zip(kv, held, gone) if not e)
        back = sum(-(-h // T) for h, e in zip(held, gone) if e)
        return {"bytes": 24 * len(n) + 8 * (taken + back) + 12 * sum(n), "flops": 4 * sum(n)}
    if case["kind"] == "rope":
        elements = case["rows"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": elements * (SIZE[case["dtype"]] + SIZE[case["out"]]) + case["rows"] * (4 + 4 * case["rot"]),
                "flops": 6 * elements}
    pairs, seen = _pairs(case)
    qo = sum(_lengths(case)[0]) * case["heads"] * case["dim"] * (SIZE[case["dtype"]] + SIZE[case["out"]])
    return {"bytes": qo + seen * 2 * case["kv_heads"] * case["dim"] + 8 * case["kv_heads"] * -(-seen // case["page"]),
            "flops": 4 * pairs * case["heads"] * case["dim"]}
