"""Plain forms, in 64 bits on the CPU, of the 8-bit paged KV cache and the
drafted-token step (include/ops/kv_quant.cuh, tree_attention.cuh,
tree_commit.cuh), and the random caches and trees that their tests use."""

import numpy as np
import torch

PAGE = 16
TOP = {1: 127.0, 2: 448.0}
KIND = {1: torch.int8, 2: torch.float8_e4m3fn}


def views(pool, dim, fmt):
    """K codes, V codes [..., 16, D] and K, V scales [..., 16] of a pool [..., record]."""
    n = PAGE * dim
    k, v = (pool[..., i * n : (i + 1) * n].unflatten(-1, (PAGE, dim)).view(KIND[fmt]) for i in (0, 1))
    s = pool[..., 2 * n :].view(torch.float32)
    return k, v, s[..., :PAGE], s[..., PAGE:]


def quantise(x, fmt):
    """fp32 rows [..., D] -> (codes, scales), by the format's definition in fp32."""
    x = x.float()
    top = x.abs().amax(-1)
    bad = ~torch.isfinite(x).all(-1)
    s = top * torch.tensor(np.float32(1) / np.float32(TOP[fmt]))
    s = torch.where(bad, torch.tensor(float("nan")), s)
    y = torch.where((s > 0)[..., None], x / s[..., None], torch.zeros(()))
    codes = y.round().clamp(-127, 127).to(torch.int8) if fmt == 1 else y.clamp(-448, 448).to(torch.float8_e4m3fn)
    return codes, s


def dequantise(codes, s):
    return codes.double() * s.double()[..., None]


class Cache:
    """A random paged cache of several sequences: lens[b] tokens each, block ids shuffled, more table columns than
    needed. `kv(b)` gives the K, V rows [len, kvh, D] in 64 bits."""

    def __init__(self, lens, kvh, dim, fmt, seed, spare_columns=2, junk=True):
        rng = np.random.default_rng(seed)
        self.fmt, self.kvh, self.dim, self.lens = fmt, kvh, dim, list(lens)
        pages = [-(-n // PAGE) for n in lens]
        self.stride = max(pages + [1]) + spare_columns
        blocks = sum(pages) + 3
        self.table = np.full((len(lens), self.stride), 0, np.int32)
        order, at = rng.permutation(blocks - 1) + 1, 0  # block 0 is what unused entries point at
        for b, n in enumerate(pages):
            self.table[b, :n] = order[at : at + n]
            at += n
        self.blocks = blocks
        g = torch.Generator().manual_seed(seed)
        x = torch.randn(2, blocks, kvh, PAGE, dim, generator=g) * torch.exp(0.5 * torch.randn(dim, generator=g))
        if fmt == 0:
            self.k, self.v = x[0].clone(), x[1].clone()
            if junk:
                self._each_unused(lambda blk, lo: (self.k[blk, :, lo:].fill_(float("nan")), self.v[blk, :, lo:].fill_(float("inf"))))
        else:
            self.pool = torch.zeros(blocks, kvh, 2 * PAGE * dim + 8 * PAGE, dtype=torch.uint8)
            kc, vc, ks, vs = views(self.pool, dim, fmt)
            for codes, scales, rows in ((kc, ks, x[0]), (vc, vs, x[1])):
                c, s = quantise(rows, fmt)
                codes.view(torch.uint8).copy_(c.view(torch.uint8))
                scales.copy_(s)
            if junk:  # codes and scales of slots that hold no token: NaN patterns
                self._each_unused(lambda blk, lo: (kc.view(torch.uint8)[blk, :, lo:].fill_(0x7F), vc.view(torch.uint8)[blk, :, lo:].fill_(0xFF),
                                                   ks[blk, :, lo:].fill_(float("nan")), vs[blk, :, lo:].fill_(float("inf"))))

    def _each_unused(self, f):
        for blk in set(range(self.blocks)) - {int(x) for b, n in enumerate(self.lens) for x in self.table[b, : -(-n // PAGE)]}:
            f(blk, 0)
        for b, n in enumerate(self.lens):
            if n % PAGE:
                f(int(self.table[b, n // PAGE]), n % PAGE)

    def rows(self, b, first=0, last=None):
        last = self.lens[b] if last is None else last
        pos = np.arange(first, last)
        blk, slot = torch.from_numpy(self.table[b, pos // PAGE].astype(np.int64)), torch.from_numpy(pos % PAGE)
        if self.fmt == 0:
            return self.k[blk, :, slot].double(), self.v[blk, :, slot].double()
        kc, vc, ks, vs = views(self.pool, self.dim, self.fmt)
        pick = lambda c: c.view(torch.uint8)[blk, :, slot].view(c.dtype)  # noqa: E731
        return dequantise(pick(kc), ks[blk, :, slot]), dequantise(pick(vc), vs[blk, :, slot])

    def spoil(self, b, pos):
        """Makes the token at `pos` of sequence b a NaN (K) and an infinity (V)."""
        blk, slot = int(self.table[b, pos // PAGE]), pos % PAGE
        if self.fmt == 0:
            self.k[blk, :, slot] = float("nan")
            self.v[blk, :, slot] = float("inf")
        else:
            kc, vc, ks, vs = views(self.pool, self.dim, self.fmt)
            kc.view(torch.uint8)[blk, :, slot] = 0x7F
            vc.view(torch.uint8)[blk, :, slot] = 0xFF
            ks[blk, :, slot] = float("nan")
            vs[blk, :, slot] = float("inf")


def attention(cache, q, ctx, start, sees, scale):
    """Returns (out, tol1): out [rows, qh, D] in 64 bits and, per row and head, the largest sum_d |q_d k_d| * |scale| and
    the largest |v| among the visible keys (what rounding errors are proportional to)."""
    rows, qh, dim = q.shape
    rep = qh // cache.kvh
    out = torch.zeros(rows, qh, dim, dtype=torch.float64)
    mass, top = torch.zeros(rows, qh, dtype=torch.float64), torch.zeros(rows, qh, dtype=torch.float64)
    for b in range(len(ctx)):
        n = start[b + 1] - start[b]
        k, v = cache.rows(b, 0, ctx[b] + n)
        for i in range(n):
            seen = torch.cat([torch.ones(ctx[b], dtype=torch.bool), torch.as_tensor(sees[b][i])])
            if not seen.any():
                continue
            for h in range(qh):
                kk, vv, x = k[seen, h // rep], v[seen, h // rep], q[start[b] + i, h].double()
                out[start[b] + i, h] = torch.softmax(scale * (kk @ x), 0) @ vv
                mass[start[b] + i, h] = abs(scale) * (kk.abs() @ x.abs()).max()
                top[start[b] + i, h] = vv.abs().max()
    return out, mass, top


def tree(rng, n, shape="tree"):
    """Parents and the rows of visible nodes of a random tree; a node comes after its parent."""
    parent, sees = np.full(n, -1, np.int32), np.zeros((n, n), bool)
    for i in range(n):
        if i:
            parent[i] = i - 1 if shape == "chain" else rng.integers(0, i)
            sees[i] = sees[parent[i]]
        sees[i, i] = True
    return parent, sees


def pack_mask(sees, words):
    out = np.zeros((len(sees), words * 32), np.uint32)
    if len(sees):
        out[:, : sees.shape[1]] = sees
    return (out.reshape(-1, words, 32) << np.arange(32, dtype=np.uint32)).sum(-1, dtype=np.uint32).view(np.int32)


def commit(draft, target, parent):
    """The accepted path of one tree."""
    path = [0] if len(draft) else []
    while path:
        cur = path[-1]
        below = [j for j in range(cur + 1, len(draft)) if parent[j] == cur and draft[j] == target[cur]]
        if not below:
            break
        path.append(below[0])
    return path
