"""PagedCache (opworks_b200/tree.py) as programs run it, where the order and the place of the calls matter."""

import numpy as np
import pytest

import q4_plain

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def of(x):
    """What a 4-bit cache gives back of rows [n, 64]."""
    return q4_plain.dequantise(*q4_plain.quantise(x.float().cpu().view(-1, 1, 64)))


def held(cache, b, layer, first, n):
    """K rows [n, kvh, D] of a sequence of a 4-bit cache, in 64 bits."""
    pos = first + np.arange(n)
    table = cache.table.cpu().numpy()
    block, slot = torch.from_numpy(table[b, pos // 16].astype(np.int64)), torch.from_numpy(pos % 16)
    kc, _, ks, _ = q4_plain.views(cache.pool[layer].cpu(), cache.head_dim)
    return q4_plain.dequantise(kc[block, :, :, slot], ks[block, :, :, slot])


def sound(cache, lens):
    """Lengths are those expected, and every page has one owner."""
    assert cache.lens.tolist() == lens and cache.status.item() == 0
    owned = [int(x) for b, n in enumerate(lens) for x in cache.table[b, : -(-n // 16)].tolist()]
    return sorted(owned + cache.free[: cache.free_count.item()].tolist()) == list(range(cache.blocks))


@pytest.mark.parametrize("format,blocks", [("int4", None), ("int4", 12), ("int8", 12), ("int8", None), ("f32", 12)])
@pytest.mark.parametrize("whole", [True, False])
def test_steps_in_inference_mode(format, blocks, whole):
    """The cache made in that mode, or before it: the same steps as outside of it, to the bit."""
    from opworks_b200.tree import PagedCache, Rows

    def steps(made, run):
        with torch.inference_mode(made):
            cache = PagedCache(2, 2, 96, 1, 64, format, blocks=blocks)
        outs = []
        with torch.inference_mode(run):
            for counts, parents in (([20, 3], None), ([4, 3], [[-1, 0, 0, 1], [-1, 0, 1]]), ([1, 1], None), ([5, 0], None)):
                rows = Rows(counts, parents)
                g = torch.Generator().manual_seed(rows.total)
                k, v = torch.randn(2, rows.total, 64, generator=g).cuda()
                q = torch.randn(rows.total, 4, 64, generator=g).cuda()
                for layer in range(2):
                    out = torch.empty_like(q)
                    cache.write(layer, k + layer, v, rows)
                    cache.attend(layer, q, rows, out, 0.125)
                    outs.append(out)
                if parents:
                    ids = torch.arange(rows.total, device="cuda")
                    target = torch.tensor([1, 3, 0, 9, 5, 9, 9], device="cuda")
                    outs += cache.commit(ids, target, rows)
                    cache.kept(outs[-2].tolist())
                else:
                    cache.advance(rows)
            if blocks:
                cache.release([1])
            outs.append(cache.lens)
        return [x.tolist() for x in outs]

    assert steps(whole, True) == steps(False, False)


def test_a_length_moved_in_inference_mode_moves_the_rows():
    from opworks_b200.tree import PagedCache, Rows

    with torch.inference_mode():
        cache, rows = PagedCache(1, 1, 64, 1, 64, "int4"), Rows([2])
        x = torch.randn(2, 64, device="cuda")
        for way, at in (("in place", 20), ("another", 40)):
            cache.write(0, x, x, rows)
            if way == "in place":
                cache.lens += 20
            else:
                cache.lens = cache.lens + 20  # made in that mode: nothing counts its changes
            cache.write(0, -x, -x, rows)
            assert torch.equal(held(cache, 0, 0, at, 2), -of(x))
        cache.lens -= 30
        cache.write(0, x * 3, x, rows)
        assert torch.equal(held(cache, 0, 0, 10, 2), of(x * 3))


def test_drafted_rows_are_rotated_by_their_depth():
    """Siblings have one position; a kept path's rows then lie where their positions are."""
    from opworks_b200.tree import PagedCache, Rows

    for blocks in (None, 9):
        cache = PagedCache(1, 3, 64, 1, 64, "int4", blocks=blocks)
        prompt = Rows([7, 0, 20])
        assert cache.positions(prompt).tolist() == [*range(7), *range(20)]
        cache.advance(prompt)
        rows = Rows([7, 3, 1], [[-1, 0, 0, 1, 1, 3, 2], [-1, 0, -1], [-1]])
        positions = cache.positions(rows)
        assert positions.dtype == torch.int32
        assert positions.tolist() == [7, 8, 8, 9, 9, 10, 9, 0, 1, 0, 20]
        at, slots = cache.place(rows)  # where the rows lie until one path is kept
        assert at.tolist() == [*range(7, 14), 0, 1, 2, 20]
        table = cache.table.tolist()
        owner = [0] * 7 + [1] * 3 + [2]
        assert slots.tolist() == [table[b][p // 16] * 16 + p % 16 for b, p in zip(owner, at.tolist())]
        draft = torch.arange(11, device="cuda")
        target = torch.tensor([1, 3, 0, 5, 0, 99, 0, 99, 0, 0, 99], device="cuda")
        path, count, _ = cache.commit(draft, target, rows)
        assert count.tolist() == [4, 1, 1] and path[:4].tolist() == [0, 1, 3, 5]
        assert positions[path[:4].long()].tolist() == [7, 8, 9, 10]  # lens + 0, 1, ...: where commit moved them


@pytest.mark.parametrize("how", ["in place", "another"])
def test_a_length_moved_within_a_shared_step_gives_no_page_two_owners(how):
    from opworks_b200.tree import PagedCache, Rows

    cache = PagedCache(1, 3, 96, 1, 64, "int4", blocks=12)
    first = Rows([20, 40, 0])
    cache.place(first)
    cache.advance(first)
    assert sound(cache, [20, 40, 0])
    rows = Rows([30, 1, 9])
    cache.place(rows)
    if how == "in place":
        cache.lens += 33
    else:
        cache.lens = cache.lens + 33
    x = torch.randn(rows.total, 64, device="cuda")
    for call in (lambda: cache.place(rows), lambda: cache.write(0, x, x, rows), lambda: cache.advance(rows),
                 lambda: cache.commit(torch.zeros(40, dtype=torch.int32, device="cuda"), torch.zeros(40, dtype=torch.int32, device="cuda"), rows)):
        with pytest.raises(ValueError):
            call()
    cache.drop()  # the step is as if it had not been: its pages and the lengths
    assert sound(cache, [20, 40, 0])
    cache.place(rows)
    cache.advance(rows)
    assert sound(cache, [50, 41, 9])


@pytest.mark.parametrize("how", ["in place", "another"])
def test_a_length_moved_between_shared_steps_is_refused(how):
    """Its pages would not be those that the table has."""
    from opworks_b200.tree import PagedCache, Rows

    cache = PagedCache(1, 2, 96, 1, 64, "int8", blocks=12)
    rows = Rows([20, 40])
    cache.advance(rows)
    kept = cache.lens
    if how == "in place":
        cache.lens -= 10
    else:
        cache.lens = cache.lens + 40
    for call in (lambda: cache.place(rows), lambda: cache.advance(rows), lambda: cache.release([0])):
        with pytest.raises(ValueError, match="lens"):
            call()
    if how == "another":
        cache.lens = kept
        cache.release([0, 1])
        assert sound(cache, [0, 0]) and cache.free_count.item() == 12


def test_a_captured_write_follows_the_lengths_after_an_eager_one():
    from opworks_b200.tree import PagedCache, Rows

    cache, rows = PagedCache(2, 1, 64, 1, 64, "int4"), Rows([2])
    x = torch.randn(2, 64, device="cuda")
    for layer in range(2):
        cache.write(layer, x, x, rows)  # every kernel once, and the rows have places
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        for layer in range(2):
            cache.write(layer, x, x, rows)
    for at in (20, 33):
        cache.lens.fill_(at)
        x.normal_()
        graph.replay()
        for layer in range(2):
            assert torch.equal(held(cache, 0, layer, at, 2), of(x))


def test_an_eager_write_after_a_captured_one():
    from opworks_b200.tree import PagedCache, Rows

    cache, rows, other = PagedCache(1, 1, 640, 1, 64, "int4"), Rows([2]), Rows([2])
    x, y = torch.randn(2, 2, 64, device="cuda")
    cache.write(0, y, y, other)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):  # not replayed: its places are not there
        cache.write(0, x, x, rows)
    cache.write(0, x * 5, x, rows)
    assert torch.equal(held(cache, 0, 0, 0, 2), of(x * 5))


def test_two_graphs_have_places_of_their_own():
    from opworks_b200.tree import PagedCache, Rows

    cache, rows = PagedCache(1, 1, 640, 1, 64, "int4"), Rows([2])
    x = torch.randn(2, 64, device="cuda")
    cache.write(0, x, x, rows)
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for graph in graphs:
        with torch.cuda.graph(graph):
            cache.write(0, x, x, rows)
    for at, graph in ((30, graphs[1]), (50, graphs[0]), (70, graphs[1])):
        cache.lens.fill_(at)
        x.normal_()
        graph.replay()
        assert torch.equal(held(cache, 0, 0, at, 2), of(x))


def test_a_captured_write_takes_the_places_once():
    """One launch for the places of all layers, as outside of a graph."""
    from opworks_b200.tree import PagedCache, Rows

    cache, rows = PagedCache(3, 1, 64, 1, 64, "int4"), Rows([2])
    x = torch.randn(2, 64, device="cuda")
    cache.write(0, x, x, rows)
    torch.cuda.synchronize()
    graph, calls, take = torch.cuda.CUDAGraph(), [], cache._where
    cache._where = lambda *a: (calls.append(a), take(*a))[1]
    with torch.cuda.graph(graph):
        for layer in range(3):
            cache.write(layer, x, x, rows)
    assert len(calls) == 1


@pytest.mark.parametrize("format,blocks", [("int4", None), ("int4", 12), ("int8", 12)])
def test_a_step_placed_on_one_stream_and_written_on_another(format, blocks):
    """The program orders nothing but its own tensors: the places are the cache's."""
    from opworks_b200.tree import PagedCache, Rows

    cache = PagedCache(2, 2, 96, 1, 64, format, blocks=blocks)
    warm = Rows([1, 1])
    x = torch.randn(30, 64, device="cuda")
    cache.write(0, x[:2], x[:2], warm)
    cache.advance(warm)
    rows = Rows([25, 5])
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(a):
        torch.cuda._sleep(100_000_000)  # about 50 ms: the places come late
        cache.place(rows)
    with torch.cuda.stream(b):
        for layer in range(2):
            cache.write(layer, x, x, rows)
    torch.cuda.synchronize()
    if format == "int4":
        for layer in range(2):
            assert torch.equal(held(cache, 0, layer, 1, 25), of(x[:25])) and torch.equal(held(cache, 1, layer, 1, 5), of(x[25:]))
    else:
        for layer in range(2):
            k, v = cache.read(layer, rows)
            assert torch.equal(k, v) and (k.flatten(1) - x).abs().max() <= x.abs().max() / 126


@pytest.mark.parametrize("end", ["advance", "drop", "commit"])
def test_a_shared_step_ended_on_another_stream(end):
    from opworks_b200.tree import PagedCache, Rows

    cache, rows = PagedCache(1, 2, 96, 1, 64, "int4", blocks=12), Rows([25, 5])
    x, zeros = torch.randn(30, 64, device="cuda"), torch.zeros(30, dtype=torch.int32, device="cuda")
    rows.parents  # made before: a commit reads them
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(a):
        torch.cuda._sleep(100_000_000)
        cache.write(0, x, x, rows)
    with torch.cuda.stream(b):
        if end == "commit":
            cache.commit(zeros, zeros + 1, rows)
        else:
            cache.advance(rows) if end == "advance" else cache.drop()
    torch.cuda.synchronize()
    assert sound(cache, {"advance": [25, 5], "drop": [0, 0], "commit": [1, 1]}[end])



def test_shared_pages_are_not_taken_by_a_graph():
    """Each replay would take them again, and the host would not know. What was placed before may be written in one."""
    from opworks_b200.tree import PagedCache, Rows

    cache = PagedCache(1, 1, 64, 1, 64, "int4", blocks=4)
    rows, x = Rows([3]), torch.randn(3, 64, device="cuda")
    cache.write(0, x, x, rows)
    cache.advance(rows)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = x + 1
        for call in (lambda: cache.place(rows), lambda: cache.write(0, x, x, rows), lambda: cache.advance(rows), lambda: cache.release([0])):
            with pytest.raises(ValueError, match="graph"):
                call()
    cache.place(rows)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        cache.write(0, x, x, rows)
        for call in (lambda: cache.advance(rows), cache.drop):
            with pytest.raises(ValueError, match="graph"):
                call()
    x.normal_()
    graph.replay()
    assert torch.equal(held(cache, 0, 0, 3, 3), of(x))
    cache.write(0, x * 2, x, rows)
    assert torch.equal(held(cache, 0, 0, 3, 3), of(x * 2))
    cache.advance(rows)
    assert sound(cache, [6]) and y is not None


def test_kept_after_some_of_the_sequences_have_ended():
    from opworks_b200.tree import PagedCache, Rows

    cache = PagedCache(1, 3, 64, 1, 64, "int4", blocks=12)
    rows = Rows([4, 3, 2])
    x = torch.randn(9, 64, device="cuda")
    cache.write(0, x, x, rows)
    _, count, _ = cache.commit(torch.zeros(9, dtype=torch.int32, device="cuda"), torch.ones(9, dtype=torch.int32, device="cuda"), rows)
    cache.release([1])
    assert cache.bounds == [4, 0, 2]
    cache.kept(count.tolist())
    assert cache.bounds == [1, 0, 1] and cache.lens.tolist() == [1, 0, 1]
    with pytest.raises(ValueError, match="kept"):
        cache.kept(count.tolist())
