"""Serving several sequences over one paged cache with xpose_b200.serving.

One attention layer of the 4-head, 256-wide model (one kv head, rotary base
10^6), with random projections in place of trained weights:

1. four prompts of different lengths arrive together: rotary positions,
   attention over the packed prompts, keys and values into 8-bit pages;
2. a fifth, longer prompt arrives in chunks, each attending to its own pages,
   while the first four go on decoding in the same step;
3. all five decode, one token a sequence and step, captured in one CUDA graph.

Every sequence's outputs are compared at the end with attention over its whole
text in one packed call on unquantised keys and values.

    python examples/paged_serving.py [--steps 32] [--cache int8|fp8|bf16]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from xpose_b200 import serving as S  # noqa: E402

HEADS, KV_HEADS, DIM, HIDDEN, PAGE = 4, 1, 256, 1152, 16
TYPES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn, "bf16": torch.bfloat16}


def ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


class Server:
    """Pages, the sequences' page lists, and one layer's step over any mix of new tokens."""

    def __init__(self, pages, width, cache):
        g = torch.Generator(device="cuda").manual_seed(0)
        rows = (HEADS + 2 * KV_HEADS) * DIM
        self.qkv = (torch.randn(HIDDEN, rows, generator=g, device="cuda") * HIDDEN ** -0.5).bfloat16()
        self.turns, _ = S.rope_turns(DIM, 1e6)
        self.pages = S.new_pages(pages, PAGE, KV_HEADS, DIM, cache)
        self.free = list(range(pages))
        self.width, self.tables, self.lens = width, [], []
        self.scratch = S.new_scratch()

    def add(self):
        self.tables.append([])
        self.lens.append(0)
        return len(self.lens) - 1

    def plan(self, new):
        """What a step with new[i] tokens of sequence i needs: positions, slots, table, lengths, starts."""
        pos, slots, starts = [], [], [0]
        for i, n in enumerate(new):
            while len(self.tables[i]) * PAGE < self.lens[i] + n:
                self.tables[i].append(self.free.pop())
            for p in range(self.lens[i], self.lens[i] + n):
                pos.append(p)
                slots.append(self.tables[i][p // PAGE] * PAGE + p % PAGE)
            self.lens[i] += n
            starts.append(len(pos))
        table = [t + [-1] * (self.width - len(t)) for t in self.tables]
        return {"pos": ints(pos), "slots": ints(slots, torch.int64), "table": ints(table), "lens": ints(self.lens),
                "starts": ints(starts), "most": max(new)}

    def project(self, x):
        y = (x @ self.qkv).view(-1, HEADS + 2 * KV_HEADS, DIM)
        return y[:, :HEADS], y[:, HEADS:HEADS + KV_HEADS], y[:, HEADS + KV_HEADS:]

    def step(self, x, p, prompts=False):
        """x [tokens, hidden] -> attention output [tokens, heads, dim]. Prompts that start now need no pages to
        attend to: their own rows are enough."""
        q, k, v = self.project(x)
        out = torch.empty(q.shape, dtype=q.dtype, device="cuda")
        S.rope_rows(q, q, p["pos"], self.turns)
        S.kv_write(*self.pages, k, v, p["slots"], positions=p["pos"], turns=self.turns)
        if prompts:
            S.rope_rows(k, k, p["pos"], self.turns)
            S.attention_packed(out, q, k, v, p["starts"], self.scratch)
        else:
            S.attention_paged(out, q, *self.pages, p["table"], p["lens"], p["starts"], p["most"], self.scratch)
        return out


def main(steps=32, cache="int8", chunk=100):
    g = torch.Generator(device="cuda").manual_seed(1)
    lens = [5, 130, 517, 64]
    late = 3 * chunk + 17
    server = Server(pages=512, width=128, cache=TYPES[cache])
    texts = [torch.randn(n + steps + 8, HIDDEN, generator=g, device="cuda").bfloat16() for n in lens + [late]]
    outs = [[] for _ in texts]

    def feed(new, prompts=False):
        x = torch.cat([texts[i][server.lens[i]:server.lens[i] + n] for i, n in enumerate(new)])
        p = server.plan(new)
        y = server.step(x, p, prompts)
        for i, part in enumerate(y.split(new)):
            outs[i].append(part)

    for _ in lens:
        server.add()
    feed(lens, prompts=True)
    server.add()
    left = late
    while left:  # the late prompt's chunks ride along with the others' next tokens
        n = min(chunk, left)
        feed([1, 1, 1, 1, n])
        left -= n

    # decoding: one captured step, its inputs refilled between replays
    p = server.plan([1] * 5)
    x = torch.stack([texts[i][server.lens[i] - 1] for i in range(5)])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        server.step(x, p)  # loads the library's kernels before the capture; the capture repeats the same writes
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = server.step(x, p)
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    spent = 0.0
    for s in range(steps):
        if s:
            q = server.plan([1] * 5)
            for name in ("pos", "slots", "table", "lens"):
                p[name].copy_(q[name])
            x.copy_(torch.stack([texts[i][server.lens[i] - 1] for i in range(5)]))
        begin.record()
        graph.replay()
        end.record()
        for i in range(5):
            outs[i].append(y[i:i + 1].clone())
        end.synchronize()
        spent += begin.elapsed_time(end)
    assert S.error_word(server.scratch) == 0

    # each sequence again, whole, on unquantised keys and values
    worst = 0.0
    for i, text in enumerate(texts):
        got = torch.cat(outs[i])
        n = server.lens[i]
        q, k, v = server.project(text[:n])
        pos = torch.arange(n, device="cuda", dtype=torch.int32)
        S.rope_rows(q, q, pos, server.turns)
        S.rope_rows(k, k, pos, server.turns)
        want = torch.empty(q.shape, dtype=q.dtype, device="cuda")
        S.attention_packed(want, q, k, v, ints([0, n]), server.scratch)
        off = float((got.float() - want.float()).norm() / want.float().norm())
        worst = max(worst, off)
        print(f"sequence {i}: {n} tokens, relative difference to the whole text unquantised {off:.2e}")
    print(f"{steps} decode steps of 5 sequences: {spent / steps * 1e3:.1f} us a step (projection, rotation, cache, attention)")
    return worst


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=32)
    ap.add_argument("--cache", choices=sorted(TYPES), default="int8")
    a = ap.parse_args()
    main(a.steps, a.cache)
