"""Plain forms, in 64 bits or with whole numbers on the CPU, of the 4-bit paged cache, of pages and slots, and of norm and
rotation of heads (include/ops/kv4.cuh, pages.cuh, qk_norm_rope.cuh)."""

import numpy as np
import torch

import tree_cache_plain as plain

PAGE, GROUP = 16, 32
MOST = 7936.0  # the largest scale


def views(pool, dim):
    """K, V codes [..., G, 16, 16] and K, V scales [..., G, 16] of a pool [..., record]."""
    g = dim // GROUP
    n = g * 256
    k, v = (pool[..., i * n : (i + 1) * n].unflatten(-1, (g, PAGE, 16)) for i in (0, 1))
    s = pool[..., 2 * n :].view(torch.float16)
    return k, v, s[..., : g * PAGE].unflatten(-1, (g, PAGE)), s[..., g * PAGE :].unflatten(-1, (g, PAGE))


def round5(t):
    """fp32 numbers to 5 significant bits, ties to even, and no finer than fp16's smallest step."""
    t = t.double()
    m, e = torch.frexp(t)  # t = m 2^e, m in [0.5, 1)
    unit = torch.exp2((e - 5).clamp_min(-24).double())
    return torch.round(t / unit) * unit


def quantise(x):
    """fp32 rows [..., D] -> (packed codes [..., G, 16] uint8, scales [..., G] fp16)."""
    g = x.float().unflatten(-1, (-1, GROUP))
    top = g.abs().amax(-1)
    scale = round5(top * torch.tensor(np.float32(1) / np.float32(7)))
    bad = ~torch.isfinite(g).all(-1) | (scale > MOST)
    scale = torch.where(bad, torch.tensor(float("nan"), dtype=torch.float64), scale)
    good = (scale > 0)[..., None]
    code = torch.where(good, torch.round(g.double() / torch.where(good, scale[..., None], torch.ones(()).double())), torch.zeros(()).double())
    code = (code.clamp(-7, 7) + 8).to(torch.uint8).unflatten(-1, (16, 2))
    return code[..., 0] | (code[..., 1] << 4), scale.to(torch.float16)


def dequantise(packed, scales):
    """[..., G, 16] and [..., G] -> [..., D] in 64 bits."""
    c = torch.stack([packed & 15, packed >> 4], -1).flatten(-2).double() - 8
    return (c * scales.double()[..., None]).flatten(-2)


class Cache4(plain.Cache):
    """A random 4-bit cache of several sequences, as plain.Cache; slots that hold no token hold NaN patterns."""

    def __init__(self, lens, kvh, dim, seed, spare_columns=2, gain=1.0):
        super().__init__(lens, kvh, dim, 0, seed, spare_columns, junk=False)
        self.fmt = 4
        self.pool = torch.zeros(self.blocks, kvh, 18 * dim, dtype=torch.uint8)
        kc, vc, ks, vs = views(self.pool, dim)
        for codes, scales, rows in ((kc, ks, self.k), (vc, vs, self.v)):  # rows [blocks, kvh, 16, D]
            c, s = quantise(rows * gain)
            codes.copy_(c.transpose(2, 3))
            scales.copy_(s.transpose(2, 3))
        self._each_unused(lambda blk, lo: (kc[blk, :, :, lo:].fill_(0x00), vc[blk, :, :, lo:].fill_(0x0F),
                                           ks[blk, :, :, lo:].fill_(float("nan")), vs[blk, :, :, lo:].fill_(float("inf"))))

    def at(self, blk, slot):
        kc, vc, ks, vs = views(self.pool, self.dim)
        pick = lambda x: x[blk, :, :, slot]  # noqa: E731
        return dequantise(pick(kc), pick(ks)), dequantise(pick(vc), pick(vs))

    def rows(self, b, first=0, last=None):
        pos = np.arange(first, self.lens[b] if last is None else last)
        return self.at(torch.from_numpy(self.table[b, pos // PAGE].astype(np.int64)), torch.from_numpy(pos % PAGE))

    def spoil(self, b, pos):
        blk, slot = int(self.table[b, pos // PAGE]), pos % PAGE
        kc, vc, ks, vs = views(self.pool, self.dim)
        kc[blk, :, :, slot], vc[blk, :, :, slot] = 0, 0xFF
        ks[blk, :, :, slot], vs[blk, :, :, slot] = float("nan"), float("inf")


def take(lens, starts, rows, table, free, count):
    """(status, table, positions, slots, left) by a host's loop. free None: the table is complete."""
    table, before = table.copy(), table
    batch, stride = table.shape
    positions, slots = np.zeros(rows, np.int64), np.full(rows, -1, np.int64)
    need, bad = 0, False
    for b in range(batch):
        n = starts[b + 1] - starts[b]
        have, want = -(-lens[b] // PAGE), -(-(lens[b] + n) // PAGE)
        if lens[b] < 0 or n < 0 or want > stride or starts[b] < 0 or starts[b + 1] > rows:
            bad = True
        elif free is not None:
            need += want - have
    if bad or need > max(0, count):
        return -1 if bad else need - max(0, count), before, None, slots, max(0, count)
    for b in range(batch):
        end = lens[b] + starts[b + 1] - starts[b]
        if free is not None:
            for page in range(-(-lens[b] // PAGE), -(-end // PAGE)):
                count -= 1
                table[b, page] = free[count]
        for i, pos in enumerate(range(lens[b], end)):
            positions[starts[b] + i] = pos
            slots[starts[b] + i] = int(table[b, pos // PAGE]) * PAGE + pos % PAGE
    return 0, table, positions, slots, count


def give(old, new, table, free, count):
    free = free.copy()
    for b in range(len(old)):
        for page in range(-(-new[b] // PAGE), -(-old[b] // PAGE)):
            free[count] = table[b, page]
            count += 1
    return free, count


def norm_rope(x, weight, eps, positions, inv_freq, rot):
    """x [rows, heads, D] -> the same in 64 bits."""
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * weight.double()
    else:
        y = y.clone()
    if rot:
        angle = positions.double()[:, None, None] * inv_freq.double()
        a, b = y[..., : rot // 2].clone(), y[..., rot // 2 : rot].clone()
        y[..., : rot // 2] = a * torch.cos(angle) - b * torch.sin(angle)
        y[..., rot // 2 : rot] = b * torch.cos(angle) + a * torch.sin(angle)
    return y
