"""What the torch wrapper of the drafted-token step (opworks_b200/tree.py) decides on the host: nothing here launches."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")


def test_record_bytes_through_the_binding():
    import opworks_b200

    ops = opworks_b200.ops_lib()
    assert ops.kv_quant_record_bytes(64) == 32 * 64 + 128 and ops.kv_quant_record_bytes(128) == 32 * 128 + 128
    assert ops.reduction_workspace_size(1 << 20) > 0
    with pytest.raises(ValueError, match="head_dim"):
        ops.kv_quant_record_bytes(80)


def cpu_cache(format="int8", batch=2, tokens=64, **kw):
    from opworks_b200.tree import PagedCache

    return PagedCache(1, batch, tokens, 2, 64, format, device="cpu", **kw)


@pytest.mark.parametrize("format", ["int8", "f32"])
def test_write_refuses_rows_that_it_would_misread(format):
    from opworks_b200.tree import Rows

    cache, rows = cpu_cache(format), Rows([3, 2], device="cpu")
    k = torch.randn(5, 128)
    for bad_k, bad_v in [(k, k.bfloat16()), (k.double(), k.double()), (k[:4], k[:4]), (k, k[:4]), (k, torch.randn(6, 128)),
                         (k[:, :64], k[:, :64]), (k.view(5, 2, 64), k.view(5, 2, 64)), (k, k.to("meta")), (k.half(), k.half())]:
        with pytest.raises(ValueError):
            cache.write(0, bad_k, bad_v, rows)
    for counts in ([5], [3, 1, 1]):
        with pytest.raises(ValueError, match="sequences"):
            cache.write(0, k, k, Rows(counts, device="cpu"))


@pytest.mark.parametrize("format", ["int8", "f32"])
def test_attend_refuses_what_it_would_misread_or_overrun(format):
    from opworks_b200.tree import Rows

    cache, rows = cpu_cache(format), Rows([3, 2], device="cpu")
    q = torch.randn(5, 8, 64)
    for bad_q, bad_out in [(q, q.bfloat16()), (q.half(), q.half()), (q[:4], q[:4]), (q, q[:4]), (q, q[:, :4]), (q[..., :32], q[..., :32]),
                           (q.view(5, 512), q.view(5, 512)), (torch.randn(8, 5, 64).transpose(0, 1), q), (q, torch.randn(5, 64, 8).transpose(1, 2)),
                           (q, q.to("meta"))]:
        with pytest.raises(ValueError):
            cache.attend(0, bad_q, rows, bad_out, 0.125)
    with pytest.raises(ValueError, match="sequences"):
        cache.attend(0, q, Rows([5], device="cpu"), q, 0.125)


def test_commit_refuses_tokens_that_are_none():
    from opworks_b200.tree import Rows

    cache, rows = cpu_cache(), Rows([3, 2], [[-1, 0, 0], [-1, 0]], device="cpu")
    good = torch.zeros(5, dtype=torch.int32)
    for draft, target in [(good.float(), good), (good, good.float()), (good[:4], good), (good, good[:3]), (good.view(5, 1), good),
                          (good, good.to("meta"))]:
        with pytest.raises(ValueError):
            cache.commit(draft, target, rows)
    with pytest.raises(ValueError, match="sequences"):
        cache.commit(good, good, Rows([5], [[-1, 0, 1, 2, 3]], device="cpu"))


def test_the_parents_of_a_chain():
    from opworks_b200.tree import Rows

    assert Rows([3, 0, 2], device="cpu").parents.tolist() == [-1, 0, 1, -1, 0]
    assert Rows([], device="cpu").parents.tolist() == []
    assert Rows([2, 1], [[-1, 0], [-1]], device="cpu").parents.tolist() == [-1, 0, -1]


def test_deepest_path():
    from opworks_b200.tree import deepest

    assert deepest([]) == 0 and deepest([-1]) == 1 and deepest([-1, 0, 1, 2]) == 4
    assert deepest([-1, 0, 0, 1, 1, 3, 3]) == 4
    assert deepest([-1, -1, 1, 2]) == 1  # what hangs on another root is never accepted


def test_the_host_knows_how_full_the_cache_is():
    from opworks_b200.tree import Rows

    cache = cpu_cache(tokens=64)  # 64 places
    tree = Rows([4, 3], [[-1, 0, 0, 2], [-1, 0, 1]], device="cpu")
    cache.advance(Rows([10, 20], device="cpu"))
    assert cache.bounds == [10, 20] and cache.max_len == 20 and cache.lens.tolist() == [10, 20]
    # as after a commit: deepest paths, until the host says what was kept
    cache._before, cache.bounds = cache.bounds, [b + n for b, n in zip(cache.bounds, tree.depths)]
    assert cache.bounds == [13, 23]
    for wrong in ([4, 1], [1], [-1, 0]):
        with pytest.raises(ValueError, match="kept"):
            cache.kept(wrong)
    cache.kept([2, 1])
    assert cache.bounds == [12, 21]
    with pytest.raises(ValueError, match="kept"):
        cache.kept([0, 0])
    cache._room(Rows([52, 43], device="cpu"))
    cache._room(Rows([52, 0], device="cpu"))
    with pytest.raises(ValueError, match="room"):
        cache._room(Rows([1, 44], device="cpu"))


def test_rows_on_the_device_are_what_they_were_on_the_host():
    from opworks_b200.tree import Rows, tree_mask

    trees = [[-1, 0, 0, 2] + [3] * 40, [], [-1]]
    rows = Rows([len(t) for t in trees], trees, device="cpu")
    assert rows.start.tolist() == [0, 44, 44, 45] and rows.words == 2 and rows.mask.shape == (45, 2)
    assert np.array_equal(rows.mask.numpy(), np.concatenate([tree_mask(t, 2) for t in trees]))
    assert rows.parents.tolist() == sum(trees, []) and rows.depths == [4, 0, 1]
    with pytest.raises(ValueError, match="one list"):
        Rows([1, 2], [[-1], [-1]], device="cpu")
    with pytest.raises(ValueError, match="after its parent"):
        Rows([2], [[-1, 1]], device="cpu")


def test_a_cache_that_is_not_on_the_current_device_launches_nothing():
    from opworks_b200.tree import Rows

    cache, rows = cpu_cache(), Rows([3, 2], device="cpu")
    k, q, tokens = torch.randn(5, 128), torch.randn(5, 8, 64), torch.zeros(5, dtype=torch.int32)
    for call in (lambda: cache.write(0, k, k, rows), lambda: cache.read(0, rows), lambda: cache.attend(0, q, rows, q.clone(), 0.125),
                 lambda: cache.commit(tokens, tokens, rows)):
        with pytest.raises(ValueError, match="current CUDA device"):
            call()
    assert cache.bounds == [0, 0]
    with pytest.raises(ValueError, match="float16"):
        cache.read(0, rows, torch.float16)
    with pytest.raises(ValueError, match="sequences"):
        cache.read(0, Rows([1], device="cpu"))
