"""The serving operators of a transformer layer around the FP8 linears, as
measurable cases.

A case is a dict of plain values; its "kind" names the operator:

  norm    h = x + residual, root-mean-square norm of h, E4M3 codes of it with
          a given scale, one dynamic scale, or a dynamic scale for each row:
          what feeds the next FP8 linear
  write   new tokens' K and V into an E4M3 cache of pages, a power-of-two
          scale for each page and head
  read    tokens of the cache back, as fp32 or bf16
  attend  attention over that cache, for prompts and for single tokens

`own` says whether run() computes the operator in plain torch operations or
calls this framework.  Sequences are ragged; sequence b brings n[b] tokens,
which are the last ones of its kv[b].
"""
import math

import torch

own = False

DEV = "cuda:0"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
F8 = torch.float8_e4m3fn
EPS = 1e-5
FLOOR_EXP = -126  # the smallest scale of a page, 2^-126


def listed():
    return [
        # the norm before a linear in one decode step of one sequence
        {"name": "norm_m1", "kind": "norm", "m": 1, "h": 4096, "x": "bf16", "res": "bf16", "scale": "row"},
        # prefill of 8 x 512 tokens: one scale for the whole activation, as
        # the FP8 linears take it, and an fp32 residual stream
        {"name": "norm_m4096", "kind": "norm", "m": 4096, "h": 4096, "x": "bf16", "res": "fp32", "scale": "tensor"},
        # a static scale, no residual, and rows of an odd length
        {"name": "norm_odd", "kind": "norm", "m": 777, "h": 5003, "x": "fp32", "res": "none", "scale": "static"},
        # one decode step of 64 sequences
        {"name": "write_decode_b64", "kind": "write", "seqs": 64, "q": 1, "kv": 2000, "ragged": True, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "dtype": "bf16"},
        # eight whole prompts, K and V as slices of the QKV projection
        {"name": "write_prompt_8x512", "kind": "write", "seqs": 8, "q": 512, "kv": 512, "ragged": False, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16"},
        # chunks of prompts that start and end inside pages
        {"name": "write_chunk", "kind": "write", "seqs": 5, "q": 300, "kv": 1500, "ragged": True, "heads": 16,
         "kv_heads": 2, "dim": 64, "page": 32, "dtype": "fp32"},
        # the caches of 16 long sequences, read back for another program
        {"name": "read_16x8192", "kind": "read", "seqs": 16, "q": 8192, "kv": 8192, "ragged": True, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "dtype": "bf16"},
        # the last tokens of three short sequences
        {"name": "read_tail", "kind": "read", "seqs": 3, "q": 100, "kv": 333, "ragged": True, "heads": 20,
         "kv_heads": 20, "dim": 80, "page": 16, "dtype": "fp32"},
        # one decode step of one short sequence: latency
        {"name": "attend_b1", "kind": "attend", "seqs": 1, "q": 1, "kv": 500, "ragged": False, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "window": 0, "dtype": "bf16", "out": "bf16"},
        # one decode step of 32 long sequences: the cache's bytes
        {"name": "attend_b32_16k", "kind": "attend", "seqs": 32, "q": 1, "kv": 16384, "ragged": True, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "window": 0, "dtype": "bf16", "out": "bf16"},
        # a long prompt: the matrix cores
        {"name": "attend_prompt_8192", "kind": "attend", "seqs": 1, "q": 8192, "kv": 8192, "ragged": False, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "window": 0, "dtype": "bf16", "out": "bf16"},
        # chunks of prompts behind a history, a sliding window, fp32 queries
        # and outputs, a head group and a head size off the powers of two
        {"name": "attend_chunk_fp32", "kind": "attend", "seqs": 4, "q": 333, "kv": 4000, "ragged": True, "heads": 28,
         "kv_heads": 4, "dim": 96, "page": 16, "window": 1024, "dtype": "fp32", "out": "fp32"},
    ]


def _log(rng, lo, hi):
    """An integer in [lo, hi], spread over its logarithm."""
    v = min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))
    return v + 1 if v == 3072 else v


HEADS = [(32, 8, 128), (32, 8, 128), (32, 32, 128), (28, 4, 128), (16, 2, 64), (12, 4, 96), (20, 20, 80), (8, 1, 256)]


def draw(rng):
    kind = rng.choice(["norm", "norm", "write", "write", "read", "attend", "attend", "attend"])
    if kind == "norm":
        h = _log(rng, 64, 8192)
        h = h if rng.random() < 0.3 else h // 16 * 16 + (16 if h // 16 == 192 else 0)
        return {"kind": kind, "m": _log(rng, 1, 4096), "h": h, "x": rng.choice(["bf16", "fp32"]),
                "res": rng.choice(["bf16", "fp32", "none"]), "scale": rng.choice(["row", "tensor", "static"])}
    heads, kv_heads, dim = rng.choice(HEADS)
    case = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": rng.choice([16, 16, 32, 64, 128]),
            "ragged": rng.random() < 0.7, "dtype": rng.choice(["bf16", "bf16", "fp32"])}
    most = 40_000_000 // (kv_heads * dim)  # tokens of all sequences
    if kind == "attend":
        case["out"] = "fp32" if case["dtype"] == "fp32" else rng.choice(["bf16", "fp32"])
        case["window"] = 0 if rng.random() < 0.7 else _log(rng, 16, 4096)
        if rng.random() < 0.6:  # decode, of one token or a few
            case["seqs"] = _log(rng, 1, 64)
            case["q"] = rng.choice([1, 1, 1, 2, 4, 5])
            case["kv"] = max(case["q"], _log(rng, 1, min(32768, 4 * most // case["seqs"])))
        else:
            case["seqs"] = _log(rng, 1, 8)
            case["q"] = _log(rng, 7, 6000 // case["seqs"])
            case["kv"] = case["q"] if rng.random() < 0.5 else _log(rng, case["q"], 6000)
        return case
    case["seqs"] = _log(rng, 1, 64)
    case["kv"] = _log(rng, 1, min(16384, most // case["seqs"]))
    how = rng.random()
    case["q"] = 1 if how < 0.3 else case["kv"] if how < 0.6 else _log(rng, 1, case["kv"])
    return case


def _spread(top, b, least=8):
    """Lengths of a ragged batch: from a `least`-th of the top to the top."""
    lo = max(1, top // least)
    return lo + int((top - lo) * (1.0 - (b * 0.6180339887) % 1.0))


def _lengths(case):
    """(n, kv) of every sequence: new tokens, and all tokens with them."""
    kv = [_spread(case["kv"], b) if case["ragged"] else case["kv"] for b in range(case["seqs"])]
    n = [_spread(case["q"], b + 3, 4) if case["ragged"] else case["q"] for b in range(case["seqs"])]
    return [min(a, b) for a, b in zip(n, kv)], kv


def _touched(case):
    """Pages that hold a new token."""
    T = case["page"]
    return sum((kv - 1) // T - (kv - n) // T + 1 for n, kv in zip(*_lengths(case)))


# ------------------------------------------------------------ plain pieces --

def _e4m3(v):
    """fp32 values to the E4M3 values nearest to them, saturating."""
    return v.clamp(-448.0, 448.0).to(F8)


def _amax_scale(a):
    s = a / torch.full_like(a, 448.0)  # a division by a number would be a product with its reciprocal
    return torch.where((s > 0) & torch.isfinite(s), s, torch.ones_like(s))


def _page_scale(a):
    """The smallest power of two s >= 2^-126 with a <= 448 s."""
    m, e = torch.frexp(a)  # a = m 2^e, 1/2 <= m < 1; 448 = 7/8 2^9
    e = torch.where(m > 0.875, e - 8, e - 9).clamp_min(FLOOR_EXP)
    return torch.ldexp(torch.ones_like(a), torch.where(a > 0, e, torch.full_like(e, FLOOR_EXP)))


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
    g.manual_seed(int(seed) * 7919 + 17)
    return g


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _activations(g, *shape):
    """N(0, 1) with a few large channels, as activations and keys have them."""
    gain = torch.exp(0.5 * torch.randn(shape[-1], device=DEV, generator=g))
    return torch.randn(*shape, device=DEV, generator=g).mul_(gain)


def prepare(case, seed):
    g = _gen(seed)
    st = {"case": case}
    if case["kind"] == "norm":
        m, h = case["m"], case["h"]
        st["x"] = _activations(g, m, h).to(DTYPES[case["x"]])
        st["gamma"] = 1.0 + 0.1 * torch.randn(h, device=DEV, generator=g)
        if case["res"] != "none":
            st["res"] = _activations(g, m, h).mul_(3.0).to(DTYPES[case["res"]])
            st["res_out"] = torch.empty_like(st["res"])
        st["y"] = torch.empty(m, h, dtype=torch.uint8, device=DEV)
        # the static scale of a calibrated model
        st["scale"] = (torch.full((1,), 6.0 / 448.0, device=DEV) if case["scale"] == "static" else
                       torch.empty(m if case["scale"] == "row" else 1, device=DEV))
        return st
    n, kv = _lengths(case)
    T, hk, d = case["page"], case["kv_heads"], case["dim"]
    cu = [sum(n[:b]) for b in range(len(n) + 1)]
    need = [-(-x // T) for x in kv]
    pages = sum(need) + 3  # a pool with room left; pages come in any order
    order = torch.randperm(pages, device=DEV, generator=g).to(torch.int32)
    first = _ints([sum(need[:b]) for b in range(len(need))])
    col = torch.arange(max(need), device=DEV)
    at = (first[:, None] + col[None]).clamp_max(pages - 1)
    used = col[None] < _ints(need)[:, None]
    st["block_table"] = torch.where(used, order[at.long()], torch.full_like(at, -1, dtype=torch.int32))
    st["kv_len"], st["cu_q"] = _ints(kv), _ints(cu)
    st["max_q"], st["max_kv"], st["tokens"] = max(n), max(kv), cu[-1]
    st["touched"] = _touched(case)
    for name in ("k", "v"):
        # a cache in use: pages of E4M3 values with the scale of their largest
        x = _activations(g, pages, hk, T, d)
        x.mul_(torch.exp(torch.randn(pages, hk, 1, 1, device=DEV, generator=g) * 0.3))
        s = _page_scale(x.abs().amax(dim=(2, 3)))
        codes = _e4m3(x.div_(s[:, :, None, None])).view(torch.uint8)
        del x
        # what tokens that have gone left behind in a page's last slots
        slot = torch.arange(T, device=DEV)
        last = torch.full((pages,), T, device=DEV, dtype=torch.int64)
        filled = [x if case["kind"] != "write" else x - y for x, y in zip(kv, n)]  # before this call
        row = _ints([max(0, -(-f // T) - 1) for f in filled])
        has = _ints([f % T if f % T or not f else T for f in filled]).long()
        last[st["block_table"][torch.arange(len(kv), device=DEV), row.long()].long()] = has
        gone = slot[None] >= last[:, None]
        codes.masked_fill_(gone[:, None, :, None], 0x7F)
        st[name + "_cache"] = (_pack_k if name == "k" else _pack_v)(codes)
        st[name + "_scale"] = s
    dt = DTYPES[case["dtype"]]
    if case["kind"] == "attend":
        st["q"] = _activations(g, cu[-1], case["heads"], d).to(dt)
        st["o"] = torch.empty(cu[-1], case["heads"], d, dtype=DTYPES[case["out"]], device=DEV)
        st["sm_scale"] = d ** -0.5
    elif case["kind"] == "write":
        # rows of the QKV projection; K and V are columns of it
        st["qkv"] = _activations(g, cu[-1], (case["heads"] + 2 * hk) * d).to(dt)
    else:
        st["k_out"] = torch.empty(cu[-1], hk, d, dtype=dt, device=DEV)
        st["v_out"] = torch.empty_like(st["k_out"])
    return st


def _kv_columns(st):
    c, x = st["case"], st["qkv"]
    x = x.view(x.shape[0], -1, c["dim"])
    return x[:, c["heads"]:c["heads"] + c["kv_heads"]], x[:, c["heads"] + c["kv_heads"]:]


# ------------------------------------------------------------- plain forms --

def _plain_norm(st):
    c = st["case"]
    if "res" in st:
        st["res_out"].copy_(st["x"].float() + st["res"].float())
        h = st["res_out"].float()
    else:
        h = st["x"].float()
    v = h * (1.0 / torch.sqrt((h * h).mean(dim=1, keepdim=True) + EPS)) * st["gamma"]
    if c["scale"] != "static":
        a = torch.where(torch.isnan(v), torch.zeros_like(v), v.abs())
        st["scale"].copy_(_amax_scale(a.amax(dim=1) if c["scale"] == "row" else a.amax().reshape(1)))
    s = st["scale"][:, None] if c["scale"] == "row" else st["scale"]
    st["y"].copy_(_e4m3(v / s).view(torch.uint8))


def _places(st):
    """Of each of the call's tokens: its sequence, and its position there."""
    cu, kv = st["cu_q"].long(), st["kv_len"].long()
    t = torch.arange(st["tokens"], device=DEV)
    b = torch.searchsorted(cu[1:], t, right=True)
    return b, kv[b] - (cu[b + 1] - t)


def _write_half(st, x, cache, scale, pack, unpack, places):
    """K's or V's half of a write; only the pages that it touches are read."""
    page, slot, begin, touched, mine = places
    x = x.float()
    a = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(dim=2)
    amax = torch.zeros_like(scale).scatter_reduce(0, page[:, None].expand_as(a), a, "amax")[touched]
    old, begin = scale[touched], begin[touched][:, None]
    new = torch.where(begin > 0, torch.maximum(old, _page_scale(amax)), _page_scale(amax))
    grown = (old / new)[:, :, None, None]  # a power of two: where it is below 1, kept tokens are encoded again
    codes = unpack(cache[touched])
    kept = (torch.arange(codes.shape[2], device=DEV)[None] < begin)[:, None, :, None]
    codes = torch.where(kept & (grown < 1), _e4m3(codes.view(F8).float() * grown).view(torch.uint8), codes)
    codes[mine, :, slot] = _e4m3(x / new[mine][:, :, None]).view(torch.uint8)
    cache[touched] = pack(codes)
    scale[touched] = new


def _plain_write(st):
    T, cu, kv = st["case"]["page"], st["cu_q"].long(), st["kv_len"].long()
    b, pos = _places(st)
    page, slot = st["block_table"][b, pos // T].long(), pos % T
    # the first new slot of every page
    begin = torch.full((st["k_scale"].shape[0],), T, device=DEV).scatter_reduce(0, page, slot, "amin")
    # the touched pages, sequence by sequence, and each token's among them
    first = (kv - (cu[1:] - cu[:-1])) // T
    count = (kv - 1) // T - first + 1
    mine = (torch.cumsum(count, 0) - count - first)[b] + pos // T
    touched = torch.empty(st["touched"], dtype=torch.int64, device=DEV).scatter_(0, mine, page)
    places = (page, slot, begin, touched, mine)
    k, v = _kv_columns(st)
    _write_half(st, k, st["k_cache"], st["k_scale"], _pack_k, _unpack_k, places)
    _write_half(st, v, st["v_cache"], st["v_scale"], _pack_v, _unpack_v, places)


def _plain_read(st):
    T = st["case"]["page"]
    b, pos = _places(st)
    page, slot = st["block_table"][b, pos // T].long(), pos % T
    d = torch.arange(st["case"]["dim"], device=DEV)
    hk, D = st["case"]["kv_heads"], st["case"]["dim"]
    head = torch.arange(hk, device=DEV)[None, :, None]
    # where element d of a token lies in its (page, head)'s T * D bytes
    at_k = (slot // 16 * 16 * D + slot % 16 * 16)[:, None, None] + (d // 16 * 256 + d % 16)
    at_v = (slot // 4 * 4 * D + slot % 4)[:, None, None] + d * 4
    k = st["k_cache"].reshape(-1, hk, T * D)[page[:, None, None], head, at_k]
    v = st["v_cache"].reshape(-1, hk, T * D)[page[:, None, None], head, at_v]
    st["k_out"].copy_(k.view(F8).float() * st["k_scale"][page][:, :, None])
    st["v_out"].copy_(v.view(F8).float() * st["v_scale"][page][:, :, None])


def _plain_attend(st):
    c = st["case"]
    T, hk, d, L = c["page"], c["kv_heads"], c["dim"], st["max_kv"]
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
    if c["window"]:
        sees &= j[None, None] > at[:, :, None] - c["window"]
    sees = sees[:, None, None].expand(-1, 1, grp, -1, -1).reshape(len(kv), 1, grp * nq, -1)
    s = s.masked_fill_(~sees, -math.inf)
    top = s.amax(dim=-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    del s
    total = p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p, dense("v_cache", "v_scale", _unpack_v))
    o = torch.where(total == 0, torch.zeros_like(o), o / total)
    o = o.reshape(len(kv), hk, grp, nq, d).permute(0, 3, 1, 2, 4).reshape(len(kv), nq, c["heads"], d)
    b = _places(st)[0]
    st["o"].copy_(o[b, torch.arange(st["tokens"], device=DEV) - cu[b]])


# ------------------------------------------------------------------- a pass --

def _pass_own(st):
    from luisaml_amd import capi
    c = st["case"]
    if c["kind"] == "norm":
        capi.rms_norm(st["x"], st["gamma"], EPS, residual=st.get("res"), residual_out=st.get("res_out"),
                      mode={"static": capi.SCALE_STATIC, "tensor": capi.SCALE_TENSOR, "row": capi.SCALE_ROW}[c["scale"]],
                      scale=st["scale"], out=st["y"])
        return
    cache = (st["k_cache"], st["v_cache"], st["k_scale"], st["v_scale"], st["block_table"], st["kv_len"], st["cu_q"])
    if c["kind"] == "write":
        k, v = _kv_columns(st)
        capi.kv_cache_write(k, v, *cache, st["max_q"])
    elif c["kind"] == "read":
        capi.kv_cache_read(*cache, st["max_q"], st["k_out"], st["v_out"])
    else:
        capi.attention(st["q"], *cache, st["max_q"], st["max_kv"], st["sm_scale"], window=c["window"], out=st["o"])


PLAIN = {"norm": _plain_norm, "write": _plain_write, "read": _plain_read, "attend": _plain_attend}


def run(state):
    kind = state["case"]["kind"]
    (_pass_own if own else PLAIN[kind])(state)
    if kind == "norm":
        out = {"y": state["y"].view(F8), "scale": state["scale"]}
        return dict(out, h=state["res_out"]) if "res" in state else out
    if kind == "write":
        return {"k": state["k_cache"].view(F8), "v": state["v_cache"].view(F8), "k_scale": state["k_scale"],
                "v_scale": state["v_scale"]}
    if kind == "read":
        return {"k": state["k_out"], "v": state["v_out"]}
    return state["o"]


# ------------------------------------------------------- 64-bit expectation --

def _exact_norm(st):
    c = st["case"]
    h = st["x"].double()
    out = {}
    if "res" in st:
        out["h"] = h + st["res"].double()
        h = out["h"].float().to(st["res"].dtype).double()  # the norm is of what is stored
    v = h / torch.sqrt(h.square().sum(dim=1, keepdim=True) / c["h"] + EPS) * st["gamma"].double()
    if c["scale"] == "static":
        s = st["scale"].double()
    else:
        s = v.abs().max(dim=1).values / 448.0 if c["scale"] == "row" else (v.abs().max() / 448.0).reshape(1)
    # the quotients that the codes are the rounding of
    out["y"] = (v / (s[:, None] if c["scale"] == "row" else s)).clamp(-448.0, 448.0)
    out["scale"] = s
    return out


def _order_k(T, d):
    """Where element (token, d) of a page lies, as a [T, d] table."""
    t, e = torch.arange(T, device=DEV)[:, None], torch.arange(d, device=DEV)[None]
    return (t // 16) * (16 * d) + (e // 16) * 256 + (t % 16) * 16 + e % 16


def _order_v(T, d):
    t, e = torch.arange(T, device=DEV)[:, None], torch.arange(d, device=DEV)[None]
    return (t // 4) * (4 * d) + e * 4 + t % 4


def _exact_write(st):
    c = st["case"]
    n, kv = _lengths(c)
    T, d, hk = c["page"], c["dim"], c["kv_heads"]
    table, out = st["block_table"].tolist(), {}
    x = st["qkv"].double().reshape(st["tokens"], -1, d)
    for name, order, lo in (("k", _order_k(T, d), c["heads"]), ("v", _order_v(T, d), c["heads"] + hk)):
        values = st[name + "_cache"].view(F8).double().reshape(-1, hk, T * d)
        scales = st[name + "_scale"].double()
        t0 = 0
        for b in range(c["seqs"]):
            pos, end = kv[b] - n[b], kv[b]
            while pos < end:
                page, lo_slot = table[b][pos // T], pos % T
                k = min(T - lo_slot, end - pos)
                new = x[t0:t0 + k, lo:lo + hk].transpose(0, 1)  # [hk, k, d]
                a = new.abs().amax(dim=(1, 2)) / 448.0
                s = torch.exp2(torch.ceil(torch.log2(a.clamp_min(2.0 ** FLOOR_EXP))))
                if lo_slot:
                    s = torch.maximum(s, scales[page])
                    old = order[:lo_slot].reshape(-1)
                    values[page][:, old] = values[page][:, old] * (scales[page] / s)[:, None]
                values[page][:, order[lo_slot:lo_slot + k].reshape(-1)] = (new / s[:, None, None]).reshape(hk, -1)
                scales[page] = s
                pos, t0 = pos + k, t0 + k
        out[name], out[name + "_scale"] = values.reshape(-1, hk, T, d), scales
    return out


def _sequence(st, name, order, b, upto):
    """The first `upto` tokens of sequence b in 64 bits, [kv heads, upto, d]."""
    c = st["case"]
    T, d, hk = c["page"], c["dim"], c["kv_heads"]
    pages = st["block_table"][b, :-(-upto // T)].long()
    x = st[name + "_cache"].reshape(-1, hk, T * d)[pages][:, :, order.reshape(-1)].view(F8).double()
    x = x * st[name + "_scale"].double()[pages][:, :, None]
    return x.reshape(len(pages), hk, T, d).transpose(0, 1).reshape(hk, -1, d)[:, :upto]


def _exact_read(st):
    c = st["case"]
    n, kv = _lengths(c)
    out = {}
    for name, order in (("k", _order_k(c["page"], c["dim"])), ("v", _order_v(c["page"], c["dim"]))):
        parts = [_sequence(st, name, order, b, kv[b])[:, kv[b] - n[b]:].transpose(0, 1) for b in range(c["seqs"])]
        out[name] = torch.cat(parts)
    return out


def _exact_attend(st):
    c = st["case"]
    n, kv = _lengths(c)
    d, hk = c["dim"], c["kv_heads"]
    grp = c["heads"] // hk
    o = torch.zeros(st["tokens"], c["heads"], d, dtype=torch.float64, device=DEV)
    t0 = 0
    for b in range(c["seqs"]):
        k = _sequence(st, "k", _order_k(c["page"], d), b, kv[b])
        v = _sequence(st, "v", _order_v(c["page"], d), b, kv[b])
        for i0 in range(0, n[b], 1024):
            i1 = min(n[b], i0 + 1024)
            at = torch.arange(kv[b] - n[b] + i0, kv[b] - n[b] + i1, device=DEV)[:, None]
            j = torch.arange(kv[b], device=DEV)[None]
            hidden = (j > at) | (j <= at - c["window"] if c["window"] else j < 0)
            for h in range(c["heads"]):
                s = st["q"][t0 + i0:t0 + i1, h].double() @ k[h // grp].t().contiguous() * st["sm_scale"]
                s = torch.softmax(s.masked_fill(hidden, -math.inf), dim=1)
                o[t0 + i0:t0 + i1, h] = s @ v[h // grp]
        t0 += n[b]
    return o


def exact(case, seed):
    st = prepare(case, seed)
    return {"norm": _exact_norm, "write": _exact_write, "read": _exact_read, "attend": _exact_attend}[case["kind"]](st)


# -------------------------------------------------------------------- work --

SIZE = {"fp32": 4, "bf16": 2, "none": 0}


def _pairs(case):
    """Of all queries of one head: tokens seen; and the tokens that any sees."""
    w = case.get("window") or 10 ** 9
    both = list(zip(*_lengths(case)))
    return (sum(min(w, p + 1) for n, kv in both for p in range(kv - n, kv)),
            sum(kv - max(0, kv - n - w + 1) for n, kv in both))


def work(case):
    """Bytes read once and written once, and operations (a multiply-add is two)."""
    if case["kind"] == "norm":
        mh = case["m"] * case["h"]
        scales = 4 * (case["m"] if case["scale"] == "row" else 1)
        return {"bytes": mh * (SIZE[case["x"]] + 2 * SIZE[case["res"]] + 1) + 4 * case["h"] + scales, "flops": 6 * mh}
    n, kv = _lengths(case)
    T, row = case["page"], case["kv_heads"] * case["dim"]
    size = SIZE[case["dtype"]]
    if case["kind"] == "attend":
        pairs, seen = _pairs(case)
        qo = sum(n) * case["heads"] * case["dim"] * (size + SIZE[case["out"]])
        return {"bytes": qo + seen * 2 * row + 8 * case["kv_heads"] * -(-seen // T),
                "flops": 4 * pairs * case["heads"] * case["dim"]}
    return {"bytes": sum(n) * 2 * row * (size + 1) + 8 * case["kv_heads"] * _touched(case), "flops": 4 * sum(n) * row}
