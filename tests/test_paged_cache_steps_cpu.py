"""What PagedCache (opworks_b200/tree.py) keeps from call to call of a step, with a stand-in for the operators: nothing here launches."""

import pytest

torch = pytest.importorskip("torch")


class Ops:
    """Counts the operators' calls and answers none of them."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *args: self.calls.append(name)


def cache(format="int4", batch=2, tokens=96, **kw):
    from opworks_b200.tree import PagedCache

    c = PagedCache(2, batch, tokens, 1, 64, format, device="cpu", **kw)
    c.ops, c._stream = Ops(), lambda: 0
    return c


@pytest.mark.parametrize("made", [False, True])
@pytest.mark.parametrize("format,blocks", [("int4", None), ("int4", 12), ("int8", 12), ("f32", 12)])
def test_a_step_in_inference_mode(made, format, blocks):
    from opworks_b200.tree import Rows

    with torch.inference_mode(made):
        c = cache(format, blocks=blocks)
    with torch.inference_mode():
        for counts in ([5, 2], [1, 1]):
            rows = Rows(counts, device="cpu")
            first = c.place(rows)
            assert all(a is b for a, b in zip(first, c.place(rows)))
            assert c.ops.calls.count("page_take") == 1
            c.ops.calls.clear()
            c.advance(rows)
        assert c.lens.tolist() == [6, 3] and c.bounds == [6, 3]
        c.commit(torch.zeros(2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), rows)
        c.lens.fill_(0)
        if blocks is None:
            first = c.place(rows)
            c.lens += 20
            assert c.place(rows)[0] is not first[0]
            c.lens = c.lens + 1  # nothing counts the changes of this one
            second = c.place(rows)
            c.lens += 1
            assert c.place(rows)[0] is not second[0]


def test_the_number_of_a_capture_wants_a_place():
    import opworks_b200

    with pytest.raises(ValueError, match="null"):
        opworks_b200.ops_lib().ops_capture_id(0, None)


def test_depths_of_drafted_rows():
    from opworks_b200.tree import Rows

    rows = Rows([7, 0, 3, 1], [[-1, 0, 0, 1, 1, 3, 2], [], [-1, 0, -1], [-1]], device="cpu")
    assert rows.lift.dtype == torch.int32
    node = [*range(7), *range(3), 0]
    assert [n + x for n, x in zip(node, rows.lift.tolist())] == [0, 1, 1, 2, 2, 3, 2, 0, 1, 0, 0]
    chain = [-1, 0, 1, 2]
    assert Rows([4], [chain], device="cpu").lift.tolist() == [0, 0, 0, 0] and Rows([4], device="cpu").lift is None


@pytest.mark.parametrize("how", ["in place", "another"])
def test_shared_pages_and_a_length_that_the_program_moves(how):
    from opworks_b200.tree import Rows

    def move(c):
        if how == "in place":
            c.lens += 30
        else:
            c.lens = c.lens + 30

    c, rows = cache(blocks=12), Rows([20, 3], device="cpu")
    c.place(rows)
    move(c)
    zeros = torch.zeros(23, dtype=torch.int32)
    for call in (lambda: c.place(rows), lambda: c.advance(rows), lambda: c.commit(zeros, zeros, rows), lambda: c.write(0, zeros[:, None].expand(23, 64).float(), zeros[:, None].expand(23, 64).float(), rows)):
        with pytest.raises(ValueError, match="lens"):
            call()
    assert c.ops.calls == ["page_take"]
    c.drop()
    assert c.ops.calls == ["page_take", "page_give"] and c.lens.tolist() == [0, 0]
    c.advance(rows)
    assert c.lens.tolist() == [20, 3] and c.bounds == [20, 3]
    move(c)
    for call in (lambda: c.place(rows), lambda: c.advance(rows), lambda: c.release([0])):
        with pytest.raises(ValueError, match="lens"):
            call()
    with pytest.raises(ValueError, match="lens"):
        c.positions(rows)
    own = cache()  # without shared pages it may be moved
    own.place(rows)
    move(own)
    own.place(rows)
    own.advance(rows)
    own.release([1])
    assert own.lens.tolist() == [50, 0]


@pytest.mark.parametrize("blocks", [None, 12])
def test_counts_told_after_a_release(blocks):
    from opworks_b200.tree import Rows

    c, rows = cache(blocks=blocks, batch=3), Rows([4, 3, 2], device="cpu")
    tokens = torch.zeros(9, dtype=torch.int32)
    c.write(0, torch.zeros(9, 64), torch.zeros(9, 64), rows)
    c.commit(tokens, tokens, rows)
    c.release([1])
    for bad in ([1, 2], [5, 0, 1], [1, 0, -1], [1, -1, 1]):
        with pytest.raises(ValueError, match="kept"):
            c.kept(bad)
    c.kept([2, 3, 1])
    assert c.bounds == [2, 0, 1]
    with pytest.raises(ValueError, match="kept"):
        c.kept([2, 3, 1])


@pytest.mark.parametrize("inference", [False, True])
@pytest.mark.parametrize("blocks", [None, 12])
def test_a_table_that_the_program_changes_moves_the_rows(inference, blocks):
    from opworks_b200.tree import Rows

    with torch.inference_mode(inference):
        c, rows = cache(blocks=blocks), Rows([5, 2], device="cpu")
        first = c.place(rows)
        c.table[0, 0] = 7
        second = c.place(rows)
        c.table = c.table.clone()
        third = c.place(rows)
        assert first[1] is not second[1] and second[1] is not third[1] and c.ops.calls == ["page_take"] * 3
