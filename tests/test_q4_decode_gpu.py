"""Shared pages, norm and rotation, and the 4-bit cache as a program uses them: through opworks_b200/tree.py, through the example,
and as captured graphs. Tolerances of attention as in test_q4_gpu.py."""

import math
import os
import sys

import numpy as np
import pytest

import q4_plain

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("format,norm,shared", [("int4", False, False), ("int4", True, True), ("int8", True, True), ("f32", False, True), ("e4m3", True, False)])
def test_drafted_trees_give_the_tokens_of_single_steps(format, norm, shared):
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    try:
        import tree_decode
    finally:
        sys.path.pop(0)
    plain, steps, drafted, fewer = tree_decode.main(format, 24, quiet=True, norm=norm, shared=shared)
    assert plain == drafted
    assert fewer < steps
    assert len({tuple(p) for p in plain}) == 3 and len(set(sum(plain, []))) > 10


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_cache_gives_back_what_it_took(dtype):
    from opworks_b200.tree import PagedCache, Rows

    cache = PagedCache(2, 3, 100, 2, 64, "int4")
    rows = Rows([5, 0, 33])
    wide = torch.randn(rows.total, 384, device="cuda").to(dtype)
    k, v = wide[:, 128:256], wide[:, :128]
    cache.write(1, k, v, rows)
    cache.write(0, k.t().contiguous().t(), v, rows)  # inner stride rows.total
    for layer in (0, 1):
        for x, got in zip((k, v), cache.read(layer, rows)):
            want = q4_plain.dequantise(*q4_plain.quantise(x.float().cpu().view(-1, 2, 64)))
            assert torch.equal(got.cpu().double(), want)
    with pytest.raises(ValueError):
        cache.write(0, k, v, Rows([5, 0, 113]))
    with pytest.raises(ValueError, match="as"):
        cache.read(0, rows, torch.float16)


def held(cache, b, layer, n):
    """K and V rows [n, kvh, D] of a sequence, in 64 bits."""
    pos = np.arange(n)
    table = cache.table.cpu().numpy()
    blk, slot = torch.from_numpy(table[b, pos // 16].astype(np.int64)), torch.from_numpy(pos % 16)
    kc, vc, ks, vs = q4_plain.views(cache.pool[layer].cpu(), cache.head_dim)
    return (q4_plain.dequantise(c[blk, :, :, slot], s[blk, :, :, slot]) for c, s in ((kc, ks), (vc, vs)))


@pytest.mark.parametrize("format", ["int4", "int8"])
def test_sequences_that_come_and_go_share_the_pages(format):
    """40 steps of requests that begin, draft, and end, in a cache of fewer pages than they would reserve: no page has two owners,
    none is lost, lengths are what was kept, and every sequence's rows are those that it wrote."""
    from opworks_b200.tree import PagedCache, Rows

    rng, batch, kvh, dim = np.random.default_rng(5), 6, 2, 64
    cache = PagedCache(1, batch, 256, kvh, dim, format, blocks=40)
    wrote = [torch.zeros(0, kvh * dim) for _ in range(batch)]  # what each sequence should hold of K
    g = torch.Generator().manual_seed(1)
    refused = 0
    for step in range(40):
        counts = [int(rng.integers(1, 60)) if not len(w) else int(rng.integers(0, 9)) for w in wrote]
        trees = step % 3 == 2 and all(len(w) for w in wrote)
        parents = [[-1] + [int(rng.integers(0, i)) for i in range(1, n)] if n else [] for n in counts]
        rows = Rows(counts, parents if trees else None)
        try:
            positions, slots = cache.place(rows)
        except ValueError:  # no pages: the longest one ends
            refused += 1
            b = int(np.argmax([len(w) for w in wrote]))
            cache.release([b])
            wrote[b] = torch.zeros(0, kvh * dim)
            continue
        k = torch.randn(rows.total, kvh * dim, generator=g)
        cache.write(0, k.cuda(), k.cuda() * 2, rows)
        lens = [len(w) for w in wrote]
        assert positions.tolist() == [lens[b] + i for b in range(batch) for i in range(counts[b])]
        at = np.concatenate([[0], np.cumsum(counts)])
        if trees:
            draft = torch.arange(rows.total, dtype=torch.int32)
            target = torch.full((rows.total,), -5, dtype=torch.int32)
            for b in range(batch):
                for i in range(counts[b] - 1, 0, -1):
                    target[at[b] + parents[b][i]] = int(at[b]) + i
            path, count, _ = cache.commit(draft.cuda(), target.cuda(), rows)
            cache.kept(count.tolist())
            for b in range(batch):
                nodes = path[int(at[b]) : int(at[b]) + int(count[b])].cpu().long()
                wrote[b] = torch.cat([wrote[b], k[int(at[b]) + nodes]])
        elif rng.random() < 0.2:
            cache.drop()
        else:
            cache.advance(rows)
            for b in range(batch):
                wrote[b] = torch.cat([wrote[b], k[at[b] : at[b + 1]]])
        assert cache.status.item() == 0 and cache.lens.tolist() == [len(w) for w in wrote]
        pages = [-(-len(w) // 16) for w in wrote]
        owned = [int(x) for b in range(batch) for x in cache.table[b, : pages[b]].tolist()]
        free = cache.free[: cache.free_count.item()].tolist()
        assert sorted(owned + free) == list(range(40))
        if format == "int4":
            for b in range(batch):
                if len(wrote[b]):
                    got, _ = held(cache, b, 0, len(wrote[b]))
                    assert torch.equal(got.flatten(1), q4_plain.dequantise(*q4_plain.quantise(wrote[b].view(-1, kvh, dim))).flatten(1))
        if rng.random() < 0.15:
            gone = rng.permutation(batch)[:2].tolist()
            cache.release(gone)
            for b in gone:
                wrote[b] = torch.zeros(0, kvh * dim)
    cache.release(range(batch))
    assert cache.free_count.item() == 40 and sorted(cache.free.tolist()) == list(range(40)) and refused


def test_a_step_placed_twice_or_left_hanging_is_refused():
    from opworks_b200.tree import PagedCache, Rows

    cache = PagedCache(1, 2, 64, 2, 64, "int4", blocks=8)
    rows, other = Rows([3, 20]), Rows([1, 1])
    first = cache.place(rows)
    assert all(a is b for a, b in zip(first, cache.place(rows))) and cache.free_count.item() == 5
    with pytest.raises(ValueError, match="place"):
        cache.place(other)
    with pytest.raises(ValueError, match="release"):
        cache.release([0])
    cache.advance(rows)
    cache.place(rows)  # the same rows again: the next step's places
    assert cache.lens.tolist() == [3, 20] and cache.free_count.item() == 4
    cache.drop()
    assert cache.free_count.item() == 5


def test_rows_follow_a_length_that_the_program_sets():
    """Without shared pages a program may move lens itself: the same rows then have other places."""
    from opworks_b200.tree import PagedCache, Rows

    cache = PagedCache(1, 1, 64, 1, 64, "int4")
    rows = Rows([2])
    x = torch.randn(2, 64, device="cuda")
    cache.write(0, x, x, rows)
    cache.lens += 20
    cache.write(0, -x, -x, rows)
    got, _ = held(cache, 0, 0, 22)
    want = q4_plain.dequantise(*q4_plain.quantise(x.cpu().view(2, 1, 64)))
    assert torch.equal(got[:2], want) and torch.equal(got[20:], -want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_norm_and_rotation_of_slices_and_in_place(dtype):
    from opworks_b200.tree import qk_norm_rope

    g = torch.Generator().manual_seed(2)
    wide = torch.randn(7, 12, 64, generator=g).to(dtype)
    pos = torch.randint(0, 9000, (7,), generator=g, dtype=torch.int32)
    inv = 10000.0 ** (-torch.arange(0, 64, 2) / 64)
    w = torch.rand(2, 64, generator=g) + 0.5
    x = wide.cuda()
    for out in (None, (x[:, :8], x[:, 8:10])):
        q, k = qk_norm_rope(x[:, :8], x[:, 8:10], pos.cuda(), inv.cuda(), w[0].cuda(), w[1].cuda(), out=out)
        for got, lo, hi, wt in ((q, 0, 8, w[0]), (k, 8, 10, w[1])):
            want = q4_plain.norm_rope(wide[:, lo:hi], wt, 1e-5, pos, inv, 64)
            assert (got.cpu().double() - want).abs().max() <= (2.0**-7 if dtype == torch.bfloat16 else 2.0**-18) * want.abs().max()
        assert torch.equal(x[:, 10:].cpu(), wide[:, 10:])
    assert torch.equal(x[:, :8], q)
    q, k = qk_norm_rope(wide.cuda()[:, :8], wide.cuda()[:, 8:8], None)  # nothing to do: a copy
    assert torch.equal(q.cpu(), wide[:, :8])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows_each", [1, 40])
def test_a_captured_step_gives_what_an_eager_one_does(dtype, rows_each):
    """Pages, norm, store and attention in one graph, replayed with other contents and lengths, on a stream of its own, between
    replays of another graph over the same pool."""
    import opworks_b200

    ops = opworks_b200.ops_lib()
    batch, kvh, rep, dim, stride, blocks = 3, 2, 4, 64, 12, 40
    kind, total = int(dtype == torch.bfloat16), batch * rows_each + 2  # two rows of padding
    dev = dict(device="cuda")

    class Step:
        def __init__(self):
            self.lens = torch.zeros(batch, dtype=torch.int32, **dev)
            self.start = (torch.arange(batch + 1, dtype=torch.int32) * rows_each).cuda()
            self.table = torch.zeros(batch, stride, dtype=torch.int32, **dev)
            self.free = torch.arange(blocks, dtype=torch.int32, **dev)
            self.count = torch.tensor([blocks], dtype=torch.int32, **dev)
            self.pos, self.slots = torch.zeros(total, dtype=torch.int32, **dev), torch.zeros(total, dtype=torch.int64, **dev)
            self.status = torch.zeros(1, dtype=torch.int32, **dev)
            self.qkv = torch.zeros(total, (rep + 2) * kvh, dim, dtype=dtype, **dev)
            self.q, self.k = torch.zeros(total, rep * kvh, dim, dtype=dtype, **dev), torch.zeros(total, kvh, dim, dtype=dtype, **dev)
            self.out = torch.full((total, rep * kvh, dim), 7.0, dtype=dtype, **dev)
            self.pool = torch.zeros(blocks, kvh, 18 * dim, dtype=torch.uint8, **dev)
            self.inv = (10000.0 ** (-torch.arange(0, dim, 2) / dim)).cuda()
            self.w = torch.ones(dim, **dev)

        def run(self):
            s = torch.cuda.current_stream().cuda_stream
            wide, qw, kw = (rep + 2) * kvh * dim, rep * kvh * dim, kvh * dim
            ops.page_take(self.lens, self.start, batch, total, self.table, stride, self.free, self.count, self.pos, self.slots, self.count, self.status, s)
            ops.qk_norm_rope(self.qkv, wide, self.qkv[:, rep * kvh :], wide, kind, self.w, self.w, 1e-5, self.pos, self.inv, dim, total, rep * kvh, kvh, dim,
                             self.q, qw, self.k, kw, s)
            ops.kv4_write(self.k, kw, self.qkv[:, (rep + 1) * kvh :], wide, kind, self.pool, blocks, self.slots, total, kvh, dim, s)
            ops.tree_attention_q4(self.q, kind, qw, self.pool, self.table, stride, self.lens, self.start, None, 0, batch, total, rows_each, stride * 16, rep * kvh, kvh,
                                  dim, 0.125, self.out, qw, s)
            self.lens += rows_each

    eager, graphs = [Step(), Step()], [Step(), Step()]
    side = torch.cuda.Stream()
    for s in graphs:  # every kernel once, before it is captured
        s.run()
        s.__init__()
    torch.cuda.synchronize()
    captured = []
    with torch.cuda.stream(side):
        for s in graphs:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                s.run()
            captured.append(g)
    gen = torch.Generator().manual_seed(3)
    for step in range(4):
        x = [torch.randn(eager[0].qkv.shape, generator=gen).to(dtype).cuda() for _ in range(2)]
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for s, g, y in zip(graphs, captured, x):
                s.qkv.copy_(y)
                g.replay()
        for s, y in zip(eager, x):
            s.qkv.copy_(y)
            s.run()
        torch.cuda.synchronize()
        for a, b in zip(eager, graphs):
            assert a.status.item() == 0 and b.status.item() == 0
            for name in ("table", "count", "pos", "slots", "pool", "q", "k", "out", "lens"):
                assert torch.equal(getattr(a, name), getattr(b, name)), (step, name)
            assert (b.out[batch * rows_each :] == 7).all() and b.out[: batch * rows_each].isfinite().all()
    assert not torch.equal(graphs[0].out, graphs[1].out)


def test_a_sequence_of_the_cache_attends_to_what_it_wrote():
    """A prompt in two pieces, then single tokens: against 64 bits over the rows that the cache holds."""
    from opworks_b200.tree import PagedCache, Rows

    batch, kvh, rep, dim = 2, 2, 4, 128
    cache = PagedCache(2, batch, 200, kvh, dim, "int4", blocks=20)
    gen = torch.Generator().manual_seed(4)
    for counts in ([50, 7], [33, 40], [1, 1], [1, 0]):
        rows = Rows(counts)
        k, v = torch.randn(2, rows.total, kvh * dim, generator=gen).cuda()
        q = torch.randn(rows.total, kvh * rep, dim, generator=gen).cuda()
        out = torch.empty_like(q)
        before = cache.lens.tolist()
        cache.write(1, k, v, rows)
        cache.attend(1, q, rows, out, 1 / math.sqrt(dim))
        cache.advance(rows)
        lo = 0
        for b, n in enumerate(counts):
            kk, vv = held(cache, b, 1, before[b] + n)
            for i in range(n):
                for h in range(kvh * rep):
                    seen = before[b] + i + 1
                    p = torch.softmax(kk[:seen, h // rep] @ q[lo + i, h].cpu().double() / math.sqrt(dim), 0)
                    want = p @ vv[:seen, h // rep]
                    assert (out[lo + i, h].cpu().double() - want).abs().max() <= 2.0**-15 * vv.abs().max() * 8
            lo += n


def test_a_cache_that_is_not_on_the_current_device_is_refused():
    from opworks_b200 import tree

    with pytest.raises(ValueError, match="current"):
        tree._current(torch.device("cuda", torch.cuda.current_device() + 1))
