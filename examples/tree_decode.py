"""Greedy decoding with drafted trees over an 8-bit paged cache.

A small random Llama-shaped model, every layer through the operator library.
The same prompts are continued twice: one token per step, and with a tree of
drafted tokens per sequence and step. The trees come from a stand-in for a draft
model that is right four times in five; what the model itself answers decides,
so both ways give the same tokens, the second in fewer steps.

    python examples/tree_decode.py [--format int8|e4m3|f32] [--tokens 40]
"""

import argparse
import os
import random
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch  # noqa: E402

import opworks_b200  # noqa: E402
from opworks_b200.tree import PagedCache, Rows  # noqa: E402

LAYERS, HIDDEN, Q_HEADS, KV_HEADS, DIM, INTER, VOCAB = 2, 256, 8, 2, 64, 512, 1000
# node 0 is the last token of the context; two children a level, drafts go on below the first
PARENTS = [-1, 0, 0, 1, 1, 3, 3]


class Model:
    def __init__(self, seed=0):
        g = torch.Generator().manual_seed(seed)
        w = lambda *s: (torch.randn(*s, generator=g) / s[-1] ** 0.5).cuda()  # noqa: E731
        self.ops = opworks_b200.ops_lib()
        self.embed, self.head = w(VOCAB, HIDDEN) * 8, w(VOCAB, HIDDEN)
        self.ones = torch.ones(HIDDEN, device="cuda")
        self.inv_freq = (10000.0 ** (-torch.arange(0, DIM, 2).float() / DIM)).cuda()
        self.layers = [dict(q=w(Q_HEADS * DIM, HIDDEN), k=w(KV_HEADS * DIM, HIDDEN), v=w(KV_HEADS * DIM, HIDDEN),
                            o=w(HIDDEN, Q_HEADS * DIM), gate=w(INTER, HIDDEN), up=w(INTER, HIDDEN), down=w(HIDDEN, INTER))
                       for _ in range(LAYERS)]

    def linear(self, x, w, s):
        y = torch.empty(x.shape[0], w.shape[0], device="cuda")
        self.ops.linear_f32(x, w, y, x.shape[0], w.shape[1], w.shape[0], s)
        return y

    def norm(self, x, s):
        y = torch.empty_like(x)
        self.ops.rms_norm(x, self.ones, y, x.shape[0], HIDDEN, 1e-5, s)
        return y

    def step(self, cache, tokens, positions, rows):
        """The model's greedy token after each row. positions: of each row, on the host."""
        n, s = len(tokens), torch.cuda.current_stream().cuda_stream
        x = torch.empty(n, HIDDEN, device="cuda")
        ids = torch.tensor(tokens, dtype=torch.int32).cuda()
        self.ops.embedding_f32(self.embed, ids, x, n, HIDDEN, s)
        for i, w in enumerate(self.layers):
            h = self.norm(x, s)
            q, k, v = (self.linear(h, w[name], s) for name in "qkv")
            for r, pos in enumerate(positions):
                self.ops.rope(q[r], self.inv_freq, 1, Q_HEADS, DIM, pos, s)
                self.ops.rope(k[r], self.inv_freq, 1, KV_HEADS, DIM, pos, s)
            cache.write(i, k, v, rows)
            out = torch.empty_like(q)
            cache.attend(i, q.view(n, Q_HEADS, DIM), rows, out.view(n, Q_HEADS, DIM), DIM**-0.5)
            x = x + self.linear(out, w["o"], s)
            h = self.norm(x, s)
            act = torch.empty(n, INTER, device="cuda")
            self.ops.swiglu(self.linear(h, w["gate"], s), self.linear(h, w["up"], s), act, n * INTER, s)
            x = x + self.linear(act, w["down"], s)
        logits = self.linear(self.norm(x, s), self.head, s)
        target = torch.empty(n, dtype=torch.int32, device="cuda")
        greedy = torch.zeros(n, device="cuda")
        self.ops.sample(logits, n, VOCAB, greedy, greedy + 1, greedy.double(), target, s)
        return ids, target


def generate(model, prompts, tokens, format, draft=None, seed=0):
    """Continues the prompts by at least `tokens` tokens. draft: None for one token per step, else the continuations that
    the stand-in for a draft model knows. Returns (tokens of each sequence, steps)."""
    rng, batch = random.Random(seed), len(prompts)
    room = max(map(len, prompts)) + tokens + 2 * len(PARENTS)  # what is kept (a path may end past `tokens`), and a tree
    cache = PagedCache(LAYERS, batch, room, KV_HEADS, DIM, format)
    rows = Rows([len(p) for p in prompts])
    _, target = model.step(cache, sum(prompts, []), [i for p in prompts for i in range(len(p))], rows)
    cache.advance(rows)
    out = [[t] for t in target[rows.start[1:].long() - 1].tolist()]
    lens, steps = [len(p) for p in prompts], 0
    depth = [0] * len(PARENTS)
    for i, p in enumerate(PARENTS[1:], 1):
        depth[i] = depth[p] + 1
    while min(map(len, out)) <= tokens:
        steps += 1
        parents = [[] if len(o) > tokens else PARENTS if draft else [-1] for o in out]  # a sequence that is done has no rows
        rows = Rows([len(p) for p in parents], parents)
        given, positions = [], []
        for b in range(batch):
            for i in range(len(parents[b])):
                positions.append(lens[b] + depth[i])
                if i == 0:
                    given.append(out[b][-1])
                else:
                    at = len(out[b]) - 1 + depth[i]
                    right = at < len(draft[b]) and rng.random() < 0.8
                    given.append(draft[b][at] if right else rng.randrange(VOCAB))
        ids, target = model.step(cache, given, positions, rows)
        path, count, nxt = cache.commit(ids, target, rows)
        path, count, nxt, start = path.tolist(), count.tolist(), nxt.tolist(), rows.start.tolist()
        cache.kept(count)
        for b in range(batch):
            if count[b] == 0:
                continue
            kept = [given[start[b] + path[start[b] + i]] for i in range(1, count[b])]
            out[b] += kept + [nxt[b]]
            lens[b] += count[b]
    return [o[: tokens + 1] for o in out], steps


def main(format="int8", tokens=40, quiet=False):
    model = Model()
    rng = random.Random(1)
    prompts = [[rng.randrange(VOCAB) for _ in range(n)] for n in (5, 17, 40)]
    plain, steps = generate(model, prompts, tokens, format)
    drafted, fewer = generate(model, prompts, tokens, format, draft=plain)
    if not quiet:
        print(f"{format}: {tokens} tokens of {len(prompts)} sequences in {steps} steps one by one, {fewer} with drafted trees; "
              f"the same tokens: {plain == drafted}")
    return plain, steps, drafted, fewer


if __name__ == "__main__":
    p = argparse.ArgumentParser()
    p.add_argument("--format", default="int8", choices=["int8", "e4m3", "f32"])
    p.add_argument("--tokens", type=int, default=40)
    a = p.parse_args()
    main(a.format, a.tokens)
