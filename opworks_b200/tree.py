"""Decoding over a paged cache, drafted tokens included: the torch-side wrapper of
``kv_quant_*``, ``kv4_*``, ``page_*``, ``qk_norm_rope``, ``tree_attention*`` and
``tree_commit*`` (include/opworks_ops.h).

``PagedCache`` owns the pools of all layers and the block table of a batch, in
fp32, in 8 bits or in 4; a step writes the new tokens' K and V, attends, and commits::

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

With ``blocks`` the sequences share that many pages: a step takes what its new
tokens need, a commit gives back what its drafts did not, and ``release`` all that
sequences hold. ``place`` says where the new tokens go, ``positions`` what
``qk_norm_rope`` rotates them by::

    cache = PagedCache(layers=2, batch=64, max_tokens=4096, kv_heads=2, head_dim=64, format="int4", blocks=1000)
    q, k = qk_norm_rope(q, k, cache.positions(rows), inv_freq, q_weight, k_weight)
    ...
    cache.release([3, 7])                                   # sequences that are done

Everything runs on torch's current stream; nothing here waits for the device.
"""

from __future__ import annotations

import ctypes
from typing import Any, NamedTuple

import numpy as np
import torch

from . import ops_lib

FORMATS = {"f32": 0, "int8": 1, "e4m3": 2, "int4": 4}
INT4 = FORMATS["int4"]
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


def depths(parents):
    """How far each node of a tree is from its root."""
    depth = []
    for p in parents:
        depth.append(depth[p] + 1 if p >= 0 else 0)
    return depth


def to_device(device, *arrays):
    """int32 arrays as tensors, in one copy that the host does not wait for (from pinned memory, which torch keeps until
    the copy is done)."""
    both = torch.from_numpy(np.concatenate([a.ravel() for a in arrays]))
    if torch.device(device).type == "cuda":
        if torch.cuda.is_current_stream_capturing():
            raise ValueError("rows and the numbers of sequences come from the host: not while a graph is captured (each replay would copy them again, "
                             "from memory that holds others by then)")
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
        self.lift = None  # of a tree: a node's depth less its number
        if parents is None:
            self.start, self.sizes = to_device(device, start, np.diff(start))
            return
        if [len(p) for p in parents] != self.counts:
            raise ValueError("parents: one list per sequence, as long as its rows")
        self.words = max(1, -(-self.most // 32))
        mask = np.concatenate([tree_mask(p, self.words) for p in parents])
        self.depths = [deepest(p) for p in parents]
        lift = np.concatenate([np.subtract(depths(p), range(len(p))) for p in parents]).astype(np.int32)
        self.start, self.sizes, self.mask, self._parents, self.lift = to_device(device, start, np.diff(start), mask, np.concatenate(parents).astype(np.int32), lift)

    @property
    def parents(self):
        """The node that each row follows, int32 on the device: in a chain the one before it."""
        if self._parents is not None:
            return self._parents
        device = self.start.device
        owner = torch.repeat_interleave(torch.arange(len(self.counts), device=device), self.sizes, output_size=self.total)
        parents = torch.arange(self.total, dtype=torch.int32, device=device) - self.start[owner] - 1
        if device.type != "cuda" or not torch.cuda.is_current_stream_capturing():  # (a graph's are there when it is replayed)
            self._parents = parents
        return parents


def _current(device):
    """torch's current stream, where it is one of `device`: an operator launches on the current device."""
    if device.type != "cuda" or device.index != torch.cuda.current_device():
        raise ValueError(f"these tensors are on {device}, which is not the current CUDA device")
    return torch.cuda.current_stream().cuda_stream


def _version(t):
    """The number of changes in place of a tensor; None where nothing counts them (made in inference mode)."""
    return None if t.is_inference() else t._version


def _plain(make):
    """A tensor whose changes in place are counted, in inference mode too."""
    if not torch.is_inference_mode_enabled():
        return make()
    with torch.inference_mode(False):
        return make()


def _lines(x, rows, width, elem):
    """x, or a copy of it, as operators take rows of `width` elements of `elem` bytes (apart, and beginning where 16 bytes are
    loaded at a time), and its row stride."""
    stride = x.stride(0) if rows > 1 else width
    if (x.data_ptr() | stride * elem) & 15 == 0 and stride >= width:
        return x, stride
    return x.clone(memory_format=torch.contiguous_format), width


def qk_norm_rope(q, k, positions, inv_freq=None, q_weight=None, k_weight=None, eps=1e-5, out=None):
    """Queries [rows, q_heads, D] and keys [rows, kv_heads, D] (fp32 or bf16, any row stride), each head normalised (root mean
    square, fp32 weights [D]; None: that side is not) and its first 2 * len(inv_freq) dims rotated by its row's position (int32;
    inv_freq None: no rotation). Returns new tensors, or writes into ``out`` = (q_out, k_out), which may be (q, k)."""
    rows, dim = (q.shape[0], q.shape[2]) if q.dim() == 3 else (-1, -1)
    if k.dim() != 3 or k.shape[0] != rows or k.shape[2] != dim or q.dtype not in TYPES or k.dtype != q.dtype or k.device != q.device:
        raise ValueError("q and k: [rows, heads, D], both fp32 or both bf16, on one device")
    new = (torch.empty(q.shape, dtype=q.dtype, device=q.device), torch.empty(k.shape, dtype=k.dtype, device=k.device)) if out is None else tuple(out)
    for name, t, like in (("q_out", new[0], q), ("k_out", new[1], k)):
        if t.shape != like.shape or t.dtype != like.dtype or t.device != like.device:
            raise ValueError(f"{name}: as its input, {list(like.shape)} of {like.dtype} on {like.device}")
    for name, t in (("q", q), ("k", k), ("q_out", new[0]), ("k_out", new[1])):
        if rows and t.shape[1] and (t.stride(2) != 1 or (t.shape[1] > 1 and t.stride(1) != dim)):
            raise ValueError(f"{name}: the heads of a row lie one after another")
    rot = 0 if inv_freq is None else 2 * inv_freq.numel()
    plain = [("q_weight", q_weight, torch.float32, dim), ("k_weight", k_weight, torch.float32, dim)]
    if rot:
        plain += [("inv_freq", inv_freq, torch.float32, rot // 2), ("positions", positions, torch.int32, rows)]
    for name, t, kind, n in plain:
        if t is not None and (t.dtype != kind or t.numel() != n or not t.is_contiguous() or t.device != q.device):
            raise ValueError(f"{name}: {n} of {kind} on {q.device}, one after another")
    if rot and positions is None:
        raise ValueError("positions: a rotation needs them")
    stride = lambda t: t.stride(0) if rows > 1 else t.shape[1] * dim  # noqa: E731
    (q, qs), (k, ks) = ((x, stride(x)) if x is y else _lines(x, rows, x.shape[1] * dim, x.element_size()) for x, y in zip((q, k), new))
    ops_lib().qk_norm_rope(q, qs, k, ks, TYPES[q.dtype], q_weight, k_weight, eps, positions if rot else None, inv_freq if rot else None,
                           rot, rows, q.shape[1], k.shape[1], dim, new[0], stride(new[0]), new[1], stride(new[1]), _current(q.device))
    return new


class _Places(NamedTuple):
    """Where the rows of a step go, and for which calls that holds."""

    rows: Rows
    lens: torch.Tensor
    table: torch.Tensor
    versions: Any  # of both
    capture: int  # the graph capture that they are part of; 0: none
    stream: Any  # that computes them
    positions: torch.Tensor
    slots: torch.Tensor


class _Step(NamedTuple):
    """A step that has taken its pages, where sequences share them."""

    rows: Rows
    after: torch.Tensor  # lens with all of its rows
    stream: Any  # that takes them


class PagedCache:
    PAGE = 16

    def __init__(self, layers, batch, max_tokens, kv_heads, head_dim, format="int8", device="cuda", blocks=None):
        self.ops, self.format = ops_lib(), FORMATS[format]
        self.layers, self.batch, self.kv_heads, self.head_dim = layers, batch, kv_heads, head_dim
        self.stride = -(-max_tokens // self.PAGE)
        self.shared = blocks is not None  # pages are taken as sequences grow, and given back
        blocks = batch * self.stride if blocks is None else blocks
        self.blocks = blocks
        if self.format:
            record = self.ops.kv4_record_bytes(head_dim) if self.format == INT4 else self.ops.kv_quant_record_bytes(head_dim)
            self.pool = torch.zeros(layers, blocks, kv_heads, record, dtype=torch.uint8, device=device)
        else:
            self.k = torch.zeros(layers, blocks, kv_heads, self.PAGE, head_dim, device=device)
            self.v = torch.zeros_like(self.k)
        # each sequence's pages spread over the pool, as an allocator would leave them
        if self.shared:
            self.table = _plain(lambda: torch.zeros(batch, self.stride, dtype=torch.int32, device=device))
            self.free = torch.arange(blocks - 1, -1, -1, dtype=torch.int32, device=device)
            self.free_count = torch.full((1,), blocks, dtype=torch.int32, device=device)
        else:
            self.table = _plain(lambda: torch.arange(blocks, dtype=torch.int32, device=device).view(self.stride, batch).t().contiguous())
        self.status = torch.zeros(1, dtype=torch.int32, device=device)  # of the last pages taken or given: 0
        self._placed = None        # the places of the last step that asked for them
        self._step = None          # with shared pages the step that has taken its own and is not ended
        self._set_lens(_plain(lambda: torch.zeros(batch, dtype=torch.int32, device=device)))
        self.bounds = [0] * batch  # upper bounds of lens that the host knows
        self._before = None        # those before the last commit; None in it: a sequence that has ended since

    @property
    def max_len(self):
        return max(self.bounds, default=0)

    def _stream(self):
        """torch's current stream, where it is one of this cache's device: an operator launches on the current device."""
        if self.lens.device.type != "cuda" or self.lens.device.index != torch.cuda.current_device():
            raise ValueError(f"the cache is on {self.lens.device}, which is not the current CUDA device")
        return torch.cuda.current_stream().cuda_stream

    def _capturing(self):
        return self.lens.device.type == "cuda" and torch.cuda.is_current_stream_capturing()

    def _capture(self, stream):
        """The number of the graph capture that the current stream takes part in; 0: none."""
        if not self._capturing():
            return 0
        number = ctypes.c_int64()
        self.ops.ops_capture_id(stream, ctypes.byref(number))
        return number.value

    def _no_graph(self, what):
        if self._capturing():
            raise ValueError(f"{what}: not while a graph is captured, where sequences share pages (each replay would take or give them again)")

    def _set_lens(self, lens):
        self.lens = lens
        self._own = (lens, lens._version)  # as this cache left it

    def _unmoved(self):
        return self.lens is self._own[0] and _version(self.lens) == self._own[1]

    def _pages(self, tokens):
        return sum(-(-n // self.PAGE) for n in tokens)

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
        if self.shared and self._pages(b + n for b, n in zip(self.bounds, rows.counts)) > self.blocks:
            raise ValueError("the cache has no pages for these rows")

    def _where(self, rows, take, stream):
        """Positions (int32) and slots (int64) of the rows; with ``take`` their pages come off the stack."""
        positions = torch.empty(rows.total, dtype=torch.int32, device=self.lens.device)
        slots = torch.empty(rows.total, dtype=torch.int64, device=self.lens.device)
        stack = (self.free, self.free_count) if take else (None, None)
        self.ops.page_take(self.lens, rows.start, self.batch, rows.total, self.table, self.stride, *stack, positions, slots, stack[1],
                           self.status, stream)
        return positions, slots

    def place(self, rows):
        """Where the rows of a step go: positions (int32, lens + 0, 1, ..., in a tree too: until commit every node has its own;
        ``positions`` is what rows are rotated by) and slots (int64, 16 * block + place in the page). With
        shared pages those that the step needs are taken, once, whoever asks first: this, or the step's first write; not while a
        graph is captured (write, read and attend may be captured once they are)."""
        self._belongs(rows)
        self._room(rows)
        return self._at(rows, self._stream())

    def _at(self, rows, stream):
        if self.shared:
            self._own_lens()
            if self._step is not None and self._step.rows is not rows:
                raise ValueError("place: the step before has been given its places and is neither kept nor dropped (advance, commit, drop)")
        at = self._places(rows, stream)
        if at is not None:
            return at
        capture, current = self._capture(stream), torch.cuda.current_stream() if self.lens.device.type == "cuda" else None
        take = self.shared and self._step is None
        if take:
            self._no_graph("place")
        elif self._step is not None and not capture:
            self._after(self._step.stream, stream, self._step.after)
        at = self._where(rows, take, stream)
        self._placed = _Places(rows, self.lens, self.table, (_version(self.lens), _version(self.table)), capture, current, *at)
        if take:
            self._step = _Step(rows, _plain(lambda: self.lens + rows.sizes), current)
        return at

    def _own_lens(self):
        if not self._unmoved():
            raise ValueError("lens has been moved: with shared pages it goes with the pages that sequences have (advance, commit, release; drop "
                             "sets it back to what it was before a step)")

    def positions(self, rows):
        """The positions that the rows are rotated by, int32: of a chain lens + 0, 1, ..., of a tree lens + the node's depth, so that
        siblings have one, and a path that commit keeps has those of the places that it moves to. Takes the step's pages as
        ``place`` does, which has one place for every node."""
        at, _ = self.place(rows)
        return at if rows.lift is None else at + rows.lift

    def _places(self, rows, stream):
        """Positions and slots of the rows that the step has already, None: they are to be asked for. A program that moves lens or
        changes the table has moved the rows; what a graph computes is there when it is replayed, and only in it. Another stream than
        theirs waits for them (and for the table, where pages were taken): the program does not know of them."""
        p = self._placed
        if p is None or p.rows is not rows or p.lens is not self.lens or p.table is not self.table:
            return None
        versions = (_version(self.lens), _version(self.table))
        if None in versions or p.versions != versions or p.capture != self._capture(stream):
            return None
        self._after(p.stream, stream, p.positions, p.slots, *([] if self._step is None else [self._step.after]))
        return p.positions, p.slots

    @staticmethod
    def _after(made, stream, *tensors):
        """Lets the current stream (its handle) use what another one computes."""
        if made is not None and made.cuda_stream != stream:
            current = torch.cuda.current_stream()
            current.wait_stream(made)
            for t in tensors:
                t.record_stream(current)

    def drop(self):
        """Forgets the rows of the step that was placed: their pages go back, and lens is what it was before it."""
        if self._step is not None:
            self._no_graph("drop")
            rows, after, made = self._step
            self._after(made, self._stream(), after)
            lens = _plain(lambda: after - rows.sizes)
            self._give(after, lens)
            if not self._unmoved():
                self._set_lens(lens)
        self._placed = self._step = None

    def _give(self, old, new):
        self.ops.page_give(old, new, self.batch, self.table, self.stride, self.free, self.blocks, self.free_count, self.free_count,
                           self.status, self._stream())

    def release(self, sequences):
        """Ends sequences (their numbers): their lengths become zero, and with shared pages their pages go back."""
        gone = np.zeros(self.batch, np.int32)
        for b in sequences:
            if not 0 <= int(b) < self.batch:
                raise ValueError(f"release: sequences 0 to {self.batch - 1}, not {b}")
            gone[int(b)] = 1
        if self._step is not None:
            raise ValueError("release: between steps, not within one (advance, commit, drop)")
        if self.shared:
            self._no_graph("release")
            self._own_lens()
        (mask,) = to_device(self.lens.device, gone)
        lens = _plain(lambda: torch.where(mask != 0, torch.zeros_like(self.lens), self.lens))
        if self.shared:
            self._give(self.lens, lens)
        self._set_lens(lens)
        self._placed = None
        self.bounds = [0 if g else n for n, g in zip(self.bounds, gone)]
        if self._before is not None:
            self._before = [None if g else n for n, g in zip(self._before, gone)]

    def write(self, layer, k, v, rows):
        """K and V rows [total, kv_heads * head_dim] (any row stride) at positions lens + 0, 1, ... of their sequences."""
        self._belongs(rows)
        shape = (rows.total, self.kv_heads * self.head_dim)
        self._takes("k", k, shape, TYPES)
        self._takes("v", v, shape, (k.dtype,))
        self._room(rows)
        if self.shared or self.format:
            stream = self._stream()
        if self.shared or self.format == INT4:
            _, slots = self._at(rows, stream)
        if self.format == INT4:
            elem = 4 if k.dtype is torch.float32 else 2
            k, ks = _lines(k if k.stride(1) == 1 else k.contiguous(), rows.total, shape[1], elem)
            v, vs = _lines(v if v.stride(1) == 1 else v.contiguous(), rows.total, shape[1], elem)
            self.ops.kv4_write(k, ks, v, vs, TYPES[k.dtype], self.pool[layer], self.blocks, slots, rows.total, self.kv_heads,
                               self.head_dim, stream)
            return
        if k.stride() != v.stride() or k.stride(1) != 1:  # the operator takes one row stride
            k, v = k.contiguous(), v.contiguous()
        if self.format:
            elem = 4 if k.dtype is torch.float32 else 2
            stride = k.stride(0) if rows.total > 1 else shape[1]
            if (k.data_ptr() | v.data_ptr() | stride * elem) & 15 or stride < shape[1]:
                k, v = (x.clone(memory_format=torch.contiguous_format) for x in (k, v))
                stride = shape[1]
            self.ops.kv_quant_write(k, v, TYPES[k.dtype], stride, self.pool[layer], self.format, self.table, self.stride,
                                    self.lens, rows.start, self.batch, rows.total, self.kv_heads, self.head_dim, stream)
            return
        owner = torch.repeat_interleave(torch.arange(self.batch, device=k.device), rows.sizes, output_size=rows.total)
        pos = self.lens.long()[owner] + torch.arange(rows.total, device=k.device) - rows.start.long()[owner]
        block, slot = self.table.long()[owner, pos // self.PAGE], pos % self.PAGE
        shape = (rows.total, self.kv_heads, self.head_dim)
        self.k[layer][block, :, slot] = k.float().view(shape)
        self.v[layer][block, :, slot] = v.float().view(shape)

    def read(self, layer, rows, dtype=torch.float32):
        """The rows at positions lens + 0, 1, ... of an 8-bit or 4-bit cache, as [total, kv_heads, head_dim] K and V."""
        if not self.format:
            raise ValueError("read: of an 8-bit or 4-bit cache; the fp32 pools are plain tensors")
        self._belongs(rows)
        if dtype not in TYPES:
            raise ValueError(f"read: as {' or '.join(str(d) for d in TYPES)}, not {dtype}")
        k = torch.empty(rows.total, self.kv_heads, self.head_dim, dtype=dtype, device=self.lens.device)
        v = torch.empty_like(k)
        if self.format == INT4:
            stream = self._stream()
            _, slots = self._places(rows, stream) or self._where(rows, False, stream)
            width = self.kv_heads * self.head_dim
            self.ops.kv4_read(self.pool[layer], self.blocks, slots, rows.total, self.kv_heads, self.head_dim, k, width, v, width, TYPES[dtype], stream)
            return k, v
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
        if self.format == INT4:
            self.ops.tree_attention_q4(q, TYPES[q.dtype], q.stride(0), self.pool[layer], *rest)
        elif self.format:
            self.ops.tree_attention_q8(q, TYPES[q.dtype], q.stride(0), self.pool[layer], self.format, *rest)
        else:
            self.ops.tree_attention(q, TYPES[q.dtype], q.stride(0), self.k[layer], self.v[layer], *rest)

    def advance(self, rows):
        """Keeps all rows (a prompt, or a chain that needs no verification)."""
        self._belongs(rows)
        if self.shared:
            self._no_graph("advance")
            self.place(rows)
        self._set_lens(self._step.after if self.shared else _plain(lambda: self.lens + rows.sizes))
        self._placed = self._step = None
        self.bounds, self._before = [b + n for b, n in zip(self.bounds, rows.counts)], None

    def commit(self, draft, target, rows):
        """Keeps each tree's accepted path, each chain's accepted part (all layers). draft, target: whole numbers [total], any integer type. Returns
        (path, count, next), int32 on the device."""
        self._belongs(rows)
        for name, t in (("draft", draft), ("target", target)):
            self._takes(name, t, (rows.total,), INTEGERS)
        draft, target = draft.to(torch.int32).contiguous(), target.to(torch.int32).contiguous()
        new = lambda n: torch.empty(n, dtype=torch.int32, device=self.lens.device)  # noqa: E731
        path, count, nxt = new(rows.total), new(self.batch), new(self.batch)
        lens = _plain(lambda: new(self.batch))
        head = (draft, target, rows.parents, rows.start, self.lens, self.batch, rows.most)
        tail = (self.layers, self.table, self.stride, self.kv_heads, self.head_dim, path, count, nxt, lens, self._stream())
        if self.shared:
            self._no_graph("commit")
            self.place(rows)
        if self.format:
            call = self.ops.tree_commit_q4 if self.format == INT4 else self.ops.tree_commit_q8
            call(*head, self.pool, self.pool.stride(0), *tail)
        else:
            self.ops.tree_commit(*head, self.k, self.v, self.k.stride(0), *tail)
        if self.shared:  # pages that the drafts had and the kept path does not need
            self._give(self._step.after, lens)
        self._set_lens(lens)
        self._placed = self._step = None
        self._before, self.bounds = self.bounds, [b + n for b, n in zip(self.bounds, rows.depths)]
        return path, count, nxt

    def kept(self, counts):
        """Tells the host what the last commit kept: its count, which the caller has read. Without it a sequence is taken
        to have grown by its tree's deepest path, and the cache seems full before it is. Sequences may have ended (release) in
        between: theirs are passed over."""
        counts = [int(n) for n in counts]
        if self._before is None or len(counts) != self.batch:
            raise ValueError("kept: the counts of a commit, once after it")
        bounds = [most if b is None else b + n for b, n, most in zip(self._before, counts, self.bounds)]
        if any(n < 0 for n in counts) or any(b > most for b, most in zip(bounds, self.bounds)):
            raise ValueError("kept: no more than the deepest paths of the last commit's trees")
        self.bounds, self._before = bounds, None
