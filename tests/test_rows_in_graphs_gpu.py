"""Rows (opworks_b200/tree.py) and captured graphs: what comes from the host is there before."""

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def test_a_captured_commit_of_chains():
    """A chain's parents are asked for first inside the capture: every replay has them, and eager commits too."""
    from opworks_b200.tree import PagedCache, Rows

    cache = PagedCache(1, 2, 64, 1, 64, "int8")
    warm, rows = Rows([4, 3]), Rows([4, 3])
    x = torch.randn(7, 64, device="cuda")
    draft = torch.tensor([5, 6, 7, 8, 1, 2, 3], dtype=torch.int32, device="cuda")
    target = torch.tensor([6, 7, 1, 9, 2, 9, 9], dtype=torch.int32, device="cuda")
    cache.write(0, x, x, warm)
    cache.commit(draft, target, warm)
    lens = cache.lens
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        path, count, nxt = cache.commit(draft, target, rows)
    cache.lens = lens  # (the graph's is there when it has been replayed)
    eager = cache.commit(draft, target, rows)  # before any replay
    assert eager[1].tolist() == [3, 2] and eager[0].tolist() == [0, 1, 2, -1, 0, 1, -1]
    junk = [Rows([9, 9, 9, 9, 9]) for _ in range(50)]  # other small copies from pinned memory
    for _ in range(3):
        path.zero_(), count.zero_()
        graph.replay()
        assert count.tolist() == [3, 2] and path.tolist() == [0, 1, 2, -1, 0, 1, -1] and nxt.tolist() == [1, 9]
    del junk


def test_rows_are_not_made_while_a_graph_is_captured():
    """Each replay would copy them again, from memory of the host that is other rows' by then."""
    from opworks_b200.tree import PagedCache, Rows

    graph, x = torch.cuda.CUDAGraph(), torch.zeros(4, device="cuda")
    cache = PagedCache(1, 2, 64, 1, 64, "int8")
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        x += 1
        for make in (lambda: Rows([1, 2]), lambda: Rows([2], [[-1, 0]]), lambda: cache.release([0])):
            with pytest.raises(ValueError, match="graph"):
                make()
    graph.replay()
    assert x.tolist() == [1] * 4
