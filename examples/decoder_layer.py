"""One layer of a decoder on E4M3, from the prompt to single tokens.

    h  = x + (what the layer before left to add)
    a  = attention(norm(h) Wqkv, cache) Wo
    h' = h + a;  y = gelu(norm(h') Wup) Wdown

No positions are encoded.  Every step is a call of luisaml_amd.capi: the norms
add the residual and emit the E4M3 codes and the scale that the QKV and up
projections take, K and V go from columns of the QKV projection's output into a
paged E4M3 cache, attention reads them there, and the output and down
projections quantise their fp32 inputs as they run.  Sequences of any lengths
share the pages; a step of single tokens needs no host value that changes, so
that it can be captured in a HIP graph and replayed while the sequences grow.

    python examples/decoder_layer.py [--graph]
"""
from __future__ import annotations

import argparse
import math
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from luisaml_amd import capi  # noqa: E402


class Linear:
    """An E4M3 weight [K, N] with a scale per column, packed once."""

    def __init__(self, w: torch.Tensor, bias: torch.Tensor | None = None):
        self.K, self.N = w.shape
        s = w.abs().amax(dim=0) / 448.0
        self.scale = torch.where(s > 0, s, torch.ones_like(s))
        codes = capi.quantize(w.contiguous(), self.scale, axis=1)
        self.packed, self.bias = capi.pack_weight(codes, w_is_nk=False), bias
        self.values = capi.dequantize(codes, self.scale, axis=1)  # for checks

    def codes(self, a, a_scale, out_dtype, act=capi.ACT_NONE):
        return capi.gemm(a, a_scale, self.packed, self.scale, self.N, self.K, c=self.bias, act=act, out_dtype=out_dtype)

    def dynamic(self, x, out_dtype):
        return capi.gemm_dynamic(x, self.packed, self.scale, self.N, self.K, c=self.bias, out_dtype=out_dtype)


class Cache:
    """Pages of one layer, and each sequence's place in them."""

    def __init__(self, seqs, pages_each, kv_heads, page_tokens, head_dim, device):
        self.tensors = capi.kv_cache(seqs * pages_each, kv_heads, page_tokens, head_dim, device)
        self.block_table = torch.arange(seqs * pages_each, dtype=torch.int32, device=device).view(seqs, pages_each)
        self.kv_len = torch.zeros(seqs, dtype=torch.int32, device=device)
        self.most = pages_each * page_tokens  # tokens of a sequence

    def args(self, cu_q):
        return (*self.tensors, self.block_table, self.kv_len, cu_q)


class DecoderLayer:
    def __init__(self, hidden, heads, kv_heads, head_dim, ffn, device, seed=0, eps=1e-5):
        g = torch.Generator(device=device).manual_seed(seed)
        rand = lambda *s, std=1.0: torch.randn(*s, device=device, generator=g) * std  # noqa: E731
        self.heads, self.kv_heads, self.dim, self.eps = heads, kv_heads, head_dim, eps
        width = (heads + 2 * kv_heads) * head_dim
        self.gamma1, self.gamma2 = 1 + rand(hidden, std=0.1), 1 + rand(hidden, std=0.1)
        self.qkv = Linear(rand(hidden, width, std=hidden ** -0.5))
        self.o = Linear(rand(heads * head_dim, hidden, std=(heads * head_dim) ** -0.5))
        self.up = Linear(rand(hidden, ffn, std=hidden ** -0.5), rand(ffn, std=0.01))
        self.down = Linear(rand(ffn, hidden, std=ffn ** -0.5), rand(hidden, std=0.01))

    def __call__(self, x, add, cache: Cache, cu_q, max_q):
        """x: the residual stream [tokens, hidden] fp32, add: what the layer
        before adds to it (bf16).  The rows are the last tokens of the cache's
        sequences, whose lengths count them.  Returns the same two for the next
        layer."""
        a, s, h = capi.rms_norm(add, self.gamma1, self.eps, residual=x)
        qkv = self.qkv.codes(a, s, torch.bfloat16).view(len(a), -1, self.dim)
        q, k, v = qkv.split((self.heads, self.kv_heads, self.kv_heads), dim=1)
        capi.kv_cache_write(k, v, *cache.args(cu_q), max_q)
        o = capi.attention(q, *cache.args(cu_q), max_q, cache.most, self.dim ** -0.5, out_dtype=torch.float32)
        o = self.o.dynamic(o.view(len(a), -1), torch.bfloat16)
        a, s, h = capi.rms_norm(o, self.gamma2, self.eps, residual=h)
        y = self.up.codes(a, s, torch.float32, act=capi.ACT_GELU_ERF)
        return h, self.down.dynamic(y, torch.bfloat16)

    def plain(self, x, add, lengths, history):
        """The layer in fp64 on the same weights, nothing else rounded; history:
        the K and V of each sequence's earlier tokens, which it extends."""
        def norm(h, gamma):
            return h / (h.square().mean(dim=1, keepdim=True) + self.eps).sqrt() * gamma.double()
        h = x.double() + add.double()
        qkv = (norm(h, self.gamma1) @ self.qkv.values.double()).view(len(x), -1, self.dim)
        q, k, v = qkv.split((self.heads, self.kv_heads, self.kv_heads), dim=1)
        out, at = [], 0
        for b, n in enumerate(lengths):
            K = torch.cat([history[b][0], k[at:at + n]]) if history[b] else k[at:at + n]
            V = torch.cat([history[b][1], v[at:at + n]]) if history[b] else v[at:at + n]
            history[b] = (K, V)
            L, grp = len(K), self.heads // self.kv_heads
            sc = torch.einsum("ihd,jhd->hij", q[at:at + n].cpu(), K.repeat_interleave(grp, 1).cpu()) * self.dim ** -0.5
            hidden = torch.arange(L)[None] > torch.arange(L - n, L)[:, None]
            w = torch.softmax(sc.masked_fill(hidden, -math.inf), dim=2)
            out.append(torch.einsum("hij,jhd->ihd", w, V.repeat_interleave(grp, 1).cpu()).reshape(n, -1).to(x.device))
            at += n
        h = h + torch.cat(out) @ self.o.values.double()
        y = norm(h, self.gamma2) @ self.up.values.double() + self.up.bias.double()
        y = 0.5 * y * (1 + torch.erf(y * 0.5 ** 0.5))
        return h, y @ self.down.values.double() + self.down.bias.double()


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--graph", action="store_true", help="replay the single tokens from a HIP graph")
    ap.add_argument("--steps", type=int, default=64)
    args = ap.parse_args()
    dev = torch.device("cuda:0")
    hidden, lengths = 4096, [512, 100, 1, 300]
    layer = DecoderLayer(hidden, 32, 8, 128, 11008, dev)
    seqs = len(lengths)
    cache = Cache(seqs, (max(lengths) + args.steps + 63) // 64, 8, 64, 128, dev)
    g = torch.Generator(device=dev).manual_seed(1)
    x = torch.randn(sum(lengths), hidden, device=dev, generator=g)
    cu = torch.tensor([0] + lengths, device=dev).cumsum(0).int()
    cache.kv_len.copy_(torch.tensor(lengths))
    h, add = layer(x, torch.zeros_like(x, dtype=torch.bfloat16), cache, cu, max(lengths))
    torch.cuda.synchronize()
    print(f"prompts of {lengths} tokens: |y| = {(h + add).norm().item():.1f}")

    one = torch.arange(seqs + 1, dtype=torch.int32, device=dev)
    x1, add1 = torch.randn(seqs, hidden, device=dev, generator=g), torch.zeros(seqs, hidden, device=dev, dtype=torch.bfloat16)

    def step():
        cache.kv_len.add_(1)
        return layer(x1, add1, cache, one, 1)
    if args.graph:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):  # once eagerly, so that the capture loads nothing
            step()
        torch.cuda.current_stream().wait_stream(side)
        cache.kv_len.sub_(1)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
    torch.cuda.synchronize()
    t = time.perf_counter()
    for _ in range(args.steps):
        if args.graph:
            graph.replay()
        else:
            out = step()
    torch.cuda.synchronize()
    us = (time.perf_counter() - t) / args.steps * 1e6
    print(f"{args.steps} single-token steps of {seqs} sequences{' (graph)' if args.graph else ''}: {us:.1f} us a step, "
          f"|y| = {(out[0] + out[1]).norm().item():.1f}")


if __name__ == "__main__":
    main()
