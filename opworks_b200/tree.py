"""Drafted-token decoding over a paged cache: the torch-side wrapper of
``kv_quant_*``, ``tree_attention*`` and ``tree_commit*`` (include/opworks_ops.h).

``PagedCache`` owns the pools of all layers and the block table of a batch, in
fp32 or in 8 bits; a step writes the new tokens' K and V, attends, and commits::

    cache = PagedCache(layers=2, batch=4, max_tokens=512, kv_heads=2, head_dim=64, format="int8")
    rows = Rows([len(p) for p in prompts])                 # ragged: a chain per sequence
    for layer in ...:
        cache.write(layer, k, v, rows)                      # at cache.lens + 0, 1, ...
        cache.attend(layer, q, rows, out, scale)            # q, out [rows, q_heads, head_dim]
    cache.advance(rows)                                     # a prompt: all of it stays
    ...
    rows = Rows([n] * 4, parents)                           # a drafted tree per sequence
    path, count, next = cache.commit(draft, target, rows)   # only the accepted path stays
    cache.kept(count.tolist())                              # once the host has read it: how full the cache is

Everything runs on torch's current stream; nothing here waits for the device.
"""

from __future__ import annotations

import numpy as np
import torch

from . import ops_lib

FORMATS = {"f32": 0, "int8": 1, "e4m3": 2}
TYPES = {torch.float32: 0, torch.bfloat16: 1}
INTEGERS = (torch.int32, torch.int64, torch.int16, torch.uint8, torch.int8)


def tree_mask(parents, words):
    """Rows of bits, one per node: its ancestors and itself. parents: of one tree, -1 for the root."""
    sees = np.zeros((len(parents), words * 32), np.uint32)
    for i, p in enumerate(parents):
        if p >= i or p < -1:
            raise ValueError("a node comes after its parent")
        if p >= 0:
            sees[i] = sees[p]
        sees[i, i] = 1
    return (sees.reshape(len(parents), words, 32) << np.arange(32, dtype=np.uint32)).sum(-1, dtype=np.uint32).view(np.int32)


def deepest(parents):
    """Nodes on the longest path of a tree from node 0 on, which is all that can be accepted."""
    depth = []
    for i, p in enumerate(parents):
        depth.append(1 if i == 0 else depth[p] + 1 if p >= 0 and depth[p] else 0)
    return max(depth, default=0)


def to_device(device, *arrays):
    """int32 arrays as tensors, in one copy that the host does not wait for (from pinned memory, which torch keeps until
    the copy is done)."""
    both = torch.from_numpy(np.concatenate([a.ravel() for a in arrays]))
    if torch.device(device).type == "cuda":
        both = both.pin_memory().to(device, non_blocking=True)
    out, at = [], 0
    for a in arrays:
        out.append(both[at : at + a.size].view(a.shape))
        at += a.size
    return out


class Rows:
    """The new tokens of a step: ``counts[b]`` rows of each sequence, one after another. With ``parents`` (a list per
    sequence) they are trees, else chains."""

    def __init__(self, counts, parents=None, device="cuda"):
        start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.counts, self.total, self.most = list(counts), int(start[-1]), max(counts, default=0)
        self.depths = list(counts)  # the most nodes on a path
        self.mask, self.words, self._parents = None, 0, None
        if parents is None:
            (self.start,) = to_device(device, start)
            return
        if [len(p) for p in parents] != self.counts:
            raise ValueError("parents: one list per sequence, as long as its rows")
        self.words = max(1, -(-self.most // 32))
        mask = np.concatenate([tree_mask(p, self.words) for p in parents])
        self.depths = [deepest(p) for p in parents]
        self.start, self.mask, self._parents = to_device(device, start, mask, np.concatenate(parents).astype(np.int32))

    @property
    def parents(self):
        """The node that each row follows, int32 on the device: in a chain the one before it."""
        if self._parents is None:
            owner = np.repeat(np.arange(len(self.counts)), self.counts)
            node = np.arange(self.total) - np.concatenate([[0], np.cumsum(self.counts)])[owner]
            (self._parents,) = to_device(self.start.device, (node - 1).astype(np.int32))
        return self._parents


class PagedCache:
    PAGE = 16

    def __init__(self, layers, batch, max_tokens, kv_heads, head_dim, format="int8", device="cuda"):
        self.ops, self.format = ops_lib(), FORMATS[format]
        self.layers, self.batch, self.kv_heads, self.head_dim = layers, batch, kv_heads, head_dim
        self.stride = -(-max_tokens // self.PAGE)
        blocks = batch * self.stride
        if self.format:
            record = self.ops.kv_quant_record_bytes(head_dim)
            self.pool = torch.zeros(layers, blocks, kv_heads, record, dtype=torch.uint8, device=device)
        else:
            self.k = torch.zeros(layers, blocks, kv_heads, self.PAGE, head_dim, device=device)
            self.v = torch.zeros_like(self.k)
        # each sequence's pages spread over the pool, as an allocator would leave them
        self.table = torch.arange(blocks, dtype=torch.int32, device=device).view(self.stride, batch).t().contiguous()
        self.lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self.bounds = [0] * batch  # upper bounds of lens that the host knows
        self._before = None        # those before the last commit

    @property
    def max_len(self):
        return max(self.bounds, default=0)

    def _stream(self):
        """torch's current stream, where it is one of this cache's device: an operator launches on the current device."""
        if self.lens.device.type != "cuda" or self.lens.device.index != torch.cuda.current_device():
            raise ValueError(f"the cache is on {self.lens.device}, which is not the current CUDA device")
        return torch.cuda.current_stream().cuda_stream

    def _belongs(self, rows):
        if len(rows.counts) != self.batch or rows.start.device != self.lens.device:
            raise ValueError("rows: counts of this cache's sequences, on its device")

    def _takes(self, name, t, shape, dtypes):
        """Refuses a tensor that an operator, which gets its address only, would read or write wrongly."""
        if t.device != self.lens.device or tuple(t.shape) != tuple(shape) or t.dtype not in dtypes:
            raise ValueError(f"{name}: {list(shape)} of {' or '.join(str(d) for d in dtypes)} on {self.lens.device}, not "
                             f"{list(t.shape)} of {t.dtype} on {t.device}")

    def _room(self, rows):
        if any(n and b + n > self.stride * self.PAGE for b, n in zip(self.bounds, rows.counts)):
            raise ValueError("the cache has no room for these rows")

    def write(self, layer, k, v, rows):
        """K and V rows [total, kv_heads * head_dim] (any row stride) at positions lens + 0, 1, ... of their sequences."""
        self._belongs(rows)
        shape = (rows.total, self.kv_heads * self.head_dim)
        self._takes("k", k, shape, TYPES)
        self._takes("v", v, shape, (k.dtype,))
        self._room(rows)
        if k.stride() != v.stride() or k.stride(1) != 1:  # the operator takes one row stride
            k, v = k.contiguous(), v.contiguous()
        if self.format:
            self.ops.kv_quant_write(k, v, TYPES[k.dtype], k.stride(0), self.pool[layer], self.format, self.table, self.stride,
                                    self.lens, rows.start, self.batch, rows.total, self.kv_heads, self.head_dim, self._stream())
            return
        owner = torch.repeat_interleave(torch.arange(self.batch, device=k.device), rows.start.diff(), output_size=rows.total)
        pos = self.lens.long()[owner] + torch.arange(rows.total, device=k.device) - rows.start.long()[owner]
        block, slot = self.table.long()[owner, pos // self.PAGE], pos % self.PAGE
        shape = (rows.total, self.kv_heads, self.head_dim)
        self.k[layer][block, :, slot] = k.float().view(shape)
        self.v[layer][block, :, slot] = v.float().view(shape)

    def read(self, layer, rows, dtype=torch.float32):
        """The rows at positions lens + 0, 1, ... of an 8-bit cache, as [total, kv_heads, head_dim] K and V."""
        if not self.format:
            raise ValueError("read: of an 8-bit cache; the fp32 pools are plain tensors")
        self._belongs(rows)
        if dtype not in TYPES:
            raise ValueError(f"read: as {' or '.join(str(d) for d in TYPES)}, not {dtype}")
        k = torch.empty(rows.total, self.kv_heads, self.head_dim, dtype=dtype, device=self.lens.device)
        v = torch.empty_like(k)
        self.ops.kv_quant_read(self.pool[layer], self.format, self.table, self.stride, self.lens, rows.start, self.batch,
                               rows.total, self.kv_heads, self.head_dim, k, v, TYPES[dtype], self.kv_heads * self.head_dim,
                               self._stream())
        return k, v

    def attend(self, layer, q, rows, out, scale):
        """q, out [total, q_heads, head_dim], both fp32 or both bf16, rows contiguous; the rows' K and V are written already."""
        self._belongs(rows)
        heads = q.shape[1] if q.dim() == 3 else 0
        shape = (rows.total, heads, self.head_dim)
        self._takes("q", q, shape, TYPES)
        self._takes("out", out, shape, (q.dtype,))
        for name, t in (("q", q), ("out", out)):
            if rows.total and (t.stride(2) != 1 or (heads > 1 and t.stride(1) != self.head_dim)):
                raise ValueError(f"{name}: the heads of a row lie one after another")
        rest = (self.table, self.stride, self.lens, rows.start, rows.mask, rows.words, self.batch, rows.total, rows.most,
                self.max_len, heads, self.kv_heads, self.head_dim, scale, out, out.stride(0), self._stream())
        if self.format:
            self.ops.tree_attention_q8(q, TYPES[q.dtype], q.stride(0), self.pool[layer], self.format, *rest)
        else:
            self.ops.tree_attention(q, TYPES[q.dtype], q.stride(0), self.k[layer], self.v[layer], *rest)

    def advance(self, rows):
        """Keeps all rows (a prompt, or a chain that needs no verification)."""
        self._belongs(rows)
        self.lens = self.lens + rows.start.diff()
        self.bounds, self._before = [b + n for b, n in zip(self.bounds, rows.counts)], None

    def commit(self, draft, target, rows):
        """Keeps each tree's accepted path, each chain's accepted part (all layers). draft, target: whole numbers [total], any integer type. Returns
        (path, count, next), int32 on the device."""
        self._belongs(rows)
        for name, t in (("draft", draft), ("target", target)):
            self._takes(name, t, (rows.total,), INTEGERS)
        draft, target = draft.to(torch.int32).contiguous(), target.to(torch.int32).contiguous()
        new = lambda n: torch.empty(n, dtype=torch.int32, device=self.lens.device)  # noqa: E731
        path, count, nxt, lens = new(rows.total), new(self.batch), new(self.batch), new(self.batch)
        head = (draft, target, rows.parents, rows.start, self.lens, self.batch, rows.most)
        tail = (self.layers, self.table, self.stride, self.kv_heads, self.head_dim, path, count, nxt, lens, self._stream())
        if self.format:
            self.ops.tree_commit_q8(*head, self.pool, self.pool.stride(0), *tail)
        else:
            self.ops.tree_commit(*head, self.k, self.v, self.k.stride(0), *tail)
        self.lens = lens
        self._before, self.bounds = self.bounds, [b + n for b, n in zip(self.bounds, rows.depths)]
        return path, count, nxt

    def kept(self, counts):
        """Tells the host what the last commit kept: its count, which the caller has read. Without it a sequence is taken
        to have grown by its tree's deepest path, and the cache seems full before it is."""
        counts = [int(n) for n in counts]
        if self._before is None or len(counts) != self.batch:
            raise ValueError("kept: the counts of a commit, once after it")
        bounds = [b + n for b, n in zip(self._before, counts)]
        if any(n < 0 for n in counts) or any(b > most for b, most in zip(bounds, self.bounds)):
            raise ValueError("kept: no more than the deepest paths of the last commit's trees")
        self.bounds, self._before = bounds, None
