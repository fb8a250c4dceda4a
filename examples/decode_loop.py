"""Requests that come and go behind one system prompt, on the E4M3 decoder layer.

    plan: lengths, pages and positions on the GPU  ->  norm, QKV  ->  norms and
    rotation of queries and keys  ->  cache write  ->  attention  ->  the rest

The system prompt is prefilled once, as a sequence of its own; every request's
row of the page table begins with its pages, and attention reads them once for
all requests.  Without one, attention may instead look through a window beside
which the first tokens stay visible: a step then reads no more than these, while
the pages that the window has passed stay with their request until it ends.  A
request ends at --most tokens, as many as the page table and the table of
rotations are made for.  What a step needs from the host is how many tokens each
request brings; a step of single tokens is captured in a HIP graph and replayed
on a batch that is padded to the graph's rows, and between replays requests end
(a plan of its own, which takes their pages back) and start (their slot's first
pages and length are written).

    python examples/decode_loop.py [--window 512 --sinks 4] [--steps 200] [--most 8192]
"""
from __future__ import annotations

import argparse
import math
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from decoder_layer import DecoderLayer  # noqa: E402
from luisaml_amd import capi  # noqa: E402


class RotaryLayer(DecoderLayer):
    """The decoder layer with norms and rotation of queries and keys."""

    def __init__(self, hidden, heads, kv_heads, head_dim, ffn, device, positions, window=0, sinks=0, seed=0):
        super().__init__(hidden, heads, kv_heads, head_dim, ffn, device, seed=seed)
        g = torch.Generator(device=device).manual_seed(seed + 1000)
        self.q_gamma, self.k_gamma = (1 + 0.1 * torch.randn(head_dim, device=device, generator=g) for _ in range(2))
        self.turns = capi.rope_table(positions, head_dim, device=device)
        self.window, self.sinks = window, sinks

    def __call__(self, x, add, batch: "Requests", max_q):
        rows = len(x)
        (q, k, v), h = self.project(x, add)
        # (in place: rows that the batch is padded with keep the projection's values)
        q, k = capi.qk_norm_rope(q, k, batch.positions[:rows], self.turns, self.q_gamma, self.k_gamma, self.eps, q_out=q, k_out=k)
        capi.kv_cache_write(k, v, *batch.cache_args(), max_q)
        o = torch.zeros(rows, self.heads, self.dim, device=x.device)  # rows that the batch is padded with stay 0
        if batch.prefix:
            capi.attention_shared(q, *batch.cache_args(), *batch.group_args(), max_q, batch.most - batch.prefix, batch.prefix,
                                  self.dim ** -0.5, out=o)
        else:
            capi.attention(q, *batch.cache_args(), max_q, batch.most, self.dim ** -0.5, window=self.window, sinks=self.sinks,
                           out=o)
        return self.finish(o, h)

    def plain(self, x, add, which, starts, history):
        """The layer in fp64 on the same weights, nothing else rounded: rows of
        sequences `which` (one for each run of rows) from positions `starts` on;
        history: keys and values by sequence, which it extends."""
        (q, k, v), h = self.plain_project(x, add)
        q, k = self.plain_norm(q, self.q_gamma), self.plain_norm(k, self.k_gamma)
        out, at = [], 0
        for b, (n, p) in zip(which, starts):
            pos = torch.arange(p, p + n, device=x.device, dtype=torch.float64)
            angle = pos[:, None] * 10000.0 ** (-torch.arange(self.dim // 2, device=x.device, dtype=torch.float64) / (self.dim // 2))
            c, s = angle.cos()[:, None], angle.sin()[:, None]

            def turn(y):
                a, d = y[at:at + n].chunk(2, dim=2)
                return torch.cat([a * c - d * s, d * c + a * s], dim=2)
            K, V = (torch.cat([old[:p], new]) for old, new in zip(history[b], (turn(k), v[at:at + n])))
            history[b] = (K, V)
            grp, j, i = self.heads // self.kv_heads, torch.arange(len(K))[None], torch.arange(p, p + n)[:, None]
            sc = torch.einsum("ihd,jhd->hij", turn(q).cpu(), K.repeat_interleave(grp, 1).cpu()) * self.dim ** -0.5
            hidden = j > i
            if self.window:
                hidden |= (j <= i - self.window) & (j >= self.sinks)
            w = torch.softmax(sc.masked_fill(hidden, -math.inf), dim=2)
            out.append(torch.einsum("hij,jhd->ihd", w, V.repeat_interleave(grp, 1).cpu()).reshape(n, -1).to(x.device))
            at += n
        return self.plain_finish(torch.cat(out), h[:at])


class Requests:
    """A layer's cache and the requests in it: a slot each, and one more sequence
    for the system prompt.  All of it lives on the device; the host only says
    what each slot brings, and counts along, as a request ends at `most` tokens."""

    def __init__(self, slots, prefix, most, pages, kv_heads, page_tokens, head_dim, rows, device):
        ints = lambda n, v=0: torch.full((n,), v, dtype=torch.int32, device=device)  # noqa: E731
        if prefix % page_tokens:
            raise ValueError("the system prompt fills whole pages")
        self.slots, self.prefix, self.most, self.T = slots, prefix, most, page_tokens
        self.cache = capi.kv_cache(pages, kv_heads, page_tokens, head_dim, device)
        cols = -(-most // page_tokens)
        self.block_table = torch.full((slots + 1, cols), -1, dtype=torch.int32, device=device)
        self.kv_len, self.new, self.ended = ints(slots + 1), ints(slots + 1), ints(slots + 1)
        self.first_own = ints(slots + 1, prefix // page_tokens)  # columns before it are the system prompt's
        self.free_pages, self.left = torch.arange(pages, dtype=torch.int32, device=device), ints(1, pages)
        self.cu_q, self.positions = ints(slots + 2), ints(rows, -1)
        self.group_seq = torch.tensor([0, slots], dtype=torch.int32, device=device)
        self.prefix_len = ints(1, prefix)
        self.held, self.bringing = [0] * (slots + 1), {}  # the host's count

    def cache_args(self):
        return (*self.cache, self.block_table, self.kv_len, self.cu_q)

    def group_args(self):
        return self.group_seq, self.block_table[self.slots:, :self.prefix // self.T], self.prefix_len

    def brings(self, tokens: dict):
        """How many tokens each slot brings to the next steps."""
        new = [0] * (self.slots + 1)
        for b, n in tokens.items():
            new[b] = n
        self.bringing = dict(tokens)
        self.new.copy_(torch.tensor(new, dtype=torch.int32), non_blocking=True)

    def grow(self):
        """The host's count of a step: of each plan, and before each replay of a
        captured one."""
        for b, n in self.bringing.items():
            if self.held[b] + n > self.most:
                raise ValueError(f"slot {b} holds {self.held[b]} tokens and brings {n}: {self.most} at most")
        for b, n in self.bringing.items():
            self.held[b] += n

    def plan(self, rows):
        if not torch.cuda.is_current_stream_capturing():
            self.grow()
        capi.kv_cache_plan(self.new, self.kv_len, self.block_table, self.free_pages, self.left, self.T, ended=self.ended,
                           first_own=self.first_own, kv_len_out=self.kv_len, cu_q=self.cu_q, left=self.left,
                           positions=self.positions[:rows])

    def end(self, slots):
        """The slots' own pages go back."""
        self.brings({})
        self.ended[slots] = 1
        self.plan(0)
        self.ended.zero_()
        for b in slots:
            self.held[b] = 0

    def start(self, slots):
        """Empty slots begin behind the system prompt."""
        cols = self.prefix // self.T
        self.block_table[slots, :cols] = self.block_table[self.slots, :cols]
        self.kv_len[slots] = self.prefix
        for b in slots:
            self.held[b] = self.prefix


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--prefix", type=int, default=2048, help="tokens of the system prompt")
    ap.add_argument("--window", type=int, default=0)
    ap.add_argument("--sinks", type=int, default=4)
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--most", type=int, default=8192, help="tokens at which a request ends")
    args = ap.parse_args()
    dev = torch.device("cuda:0")
    hidden, slots, T, most = 4096, 16, 64, args.most
    prefix = 0 if args.window else args.prefix
    layer = RotaryLayer(hidden, 32, 8, 128, 11008, dev, most, args.window, args.sinks)
    first = {b: 50 + 37 * b for b in range(slots)}
    batch = Requests(slots, prefix, most, 2048, 8, T, 128, max(prefix, sum(first.values())), dev)
    g = torch.Generator(device=dev).manual_seed(1)
    tokens = lambda n: (torch.randn(n, hidden, device=dev, generator=g),  # noqa: E731
                        torch.zeros(n, hidden, device=dev, dtype=torch.bfloat16))

    def prompt(lengths):
        rows = sum(lengths.values())
        batch.brings(lengths)
        batch.plan(rows)
        return layer(*tokens(rows), batch, max(lengths.values()))
    if prefix:
        prompt({slots: prefix})
    for b in range(slots):
        batch.start([b])
    prompt(first)

    x, add = tokens(slots)
    batch.brings(dict.fromkeys(range(slots), 1))

    def step():
        batch.plan(slots)
        return layer(x, add, batch, 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # once eagerly, so that the capture loads nothing
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    torch.cuda.synchronize()
    spent = 0.0
    for i in range(args.steps):
        gone = {b for b in range(slots) if batch.held[b] == most}
        if i % 20 == 10:
            gone.add(i // 20 % slots)
        if gone:  # requests end, and others take their slots
            batch.end(sorted(gone))
            batch.start(sorted(gone))
            prompt(dict.fromkeys(gone, 100))
            batch.brings(dict.fromkeys(range(slots), 1))
        batch.grow()
        torch.cuda.synchronize()
        t = time.perf_counter()
        graph.replay()
        torch.cuda.synchronize()
        spent += time.perf_counter() - t
    print(f"{args.steps} steps of {slots} requests: {spent / args.steps * 1e6:.1f} us a step, {batch.left.item()} of "
          f"{len(batch.free_pages)} pages free, lengths {batch.kv_len[:slots].tolist()}, |y| = {(out[0] + out[1]).norm().item():.1f}")


if __name__ == "__main__":
    main()
