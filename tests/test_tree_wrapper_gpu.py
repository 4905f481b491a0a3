"""The torch wrapper of the drafted-token step (opworks_b200/tree.py) against plain torch, on the GPU."""

import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("format", ["int8", "e4m3", "f32"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_write_takes_k_and_v_of_different_strides(format, dtype):
    """K a slice of a fused projection and V a tensor of its own, or turned round: as if both lay one row after another."""
    from opworks_b200.tree import PagedCache, Rows

    rows = Rows([5, 0, 33])
    wide = torch.randn(rows.total, 384, device="cuda").to(dtype)
    k, v = wide[:, 128:256], torch.randn(rows.total, 128, device="cuda").to(dtype)
    turned = v.t().contiguous().t()  # inner stride rows.total
    caches = []
    for a, b in ((k.contiguous(), v), (k, v), (k, turned), (v, k)):
        caches.append(PagedCache(1, 3, 100, 2, 64, format))
        caches[-1].write(0, a, b, rows)
    same = lambda x, y: torch.equal(x.pool, y.pool) if format != "f32" else torch.equal(x.k, y.k) and torch.equal(x.v, y.v)  # noqa: E731
    assert same(caches[0], caches[1]) and same(caches[0], caches[2]) and not same(caches[0], caches[3])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attend_over_rows_of_a_wider_tensor(dtype):
    from opworks_b200.tree import PagedCache, Rows

    rows = Rows([4, 7])
    cache = PagedCache(1, 2, 64, 2, 64, "f32")
    k, v = torch.randn(2, rows.total, 128, device="cuda")
    cache.write(0, k, v, rows)
    wide = torch.randn(rows.total, 10, 64, device="cuda").to(dtype)
    out = torch.zeros(rows.total, 10, 64, device="cuda", dtype=dtype)
    cache.attend(0, wide[:, 1:9], rows, out[:, 1:9], 0.125)
    assert not out[:, 0].any() and not out[:, 9].any()
    for b, (lo, hi) in enumerate(((0, 4), (4, 11))):
        for h in range(8):
            kk, vv = (x[lo:hi, h // 4 * 64 : h // 4 * 64 + 64].double() for x in (k, v))
            s = (0.125 * wide[lo:hi, 1 + h].double() @ kk.T).masked_fill(~torch.ones(hi - lo, hi - lo, device="cuda").bool().tril(), -math.inf)
            want = torch.softmax(s, -1) @ vv
            assert (out[lo:hi, 1 + h].double() - want).abs().max() <= (2.0**-7 if dtype == torch.bfloat16 else 2.0**-16) * vv.abs().max()


@pytest.mark.parametrize("kind", [torch.int32, torch.int64, torch.int16])
def test_commit_takes_tokens_of_any_integer_type(kind):
    from opworks_b200.tree import PagedCache, Rows

    cache = PagedCache(1, 2, 64, 2, 64, "int8")
    rows = Rows([4, 3], [[-1, 0, 0, 2], [-1, 0, 1]])
    k, v = torch.randn(2, 7, 128, device="cuda")
    cache.write(0, k, v, rows)
    draft = torch.tensor([5, 6, 7, 8, 5, 6, 7], device="cuda").to(kind)
    target = torch.tensor([7, 0, 8, 9, 1, 2, 3], device="cuda").to(kind)
    path, count, nxt = cache.commit(draft.repeat_interleave(2)[::2], target, rows)
    assert path.tolist() == [0, 2, 3, -1, 0, -1, -1] and count.tolist() == [3, 1] and nxt.tolist() == [9, 1]
    assert cache.lens.tolist() == [3, 1]


@pytest.mark.parametrize("format", ["int8", "f32"])
def test_commit_of_drafted_chains(format):
    from opworks_b200.tree import PagedCache, Rows

    cache = PagedCache(2, 3, 64, 2, 64, format)
    rows = Rows([4, 1, 3])
    k, v = torch.randn(2, 8, 128, device="cuda")
    for layer in range(2):
        cache.write(layer, k, v, rows)
    draft = torch.tensor([5, 6, 7, 8, 1, 2, 3, 4], device="cuda")
    target = torch.tensor([6, 7, 1, 9, 4, 3, 4, 11], device="cuda")  # two of three right; nothing drafted; all right
    path, count, nxt = cache.commit(draft, target, rows)
    assert path.tolist() == [0, 1, 2, -1, 0, 0, 1, 2] and count.tolist() == [3, 1, 3] and nxt.tolist() == [1, 4, 11]
    assert cache.lens.tolist() == [3, 1, 3]


@pytest.mark.parametrize("format", ["int8", "f32"])
@pytest.mark.parametrize("told", [True, False])
def test_a_cache_lasts_for_what_it_keeps(format, told):
    """Trees of 20 nodes, 3 deep, of which 2 are kept, in 128 places: each step takes 2 of them where the host says what was
    kept, else 3, until a tree has no room."""
    from opworks_b200.tree import PagedCache, Rows

    cache = PagedCache(1, 1, 128, 1, 64, format)
    parents = [[-1] + [0] * 10 + [1 + i % 9 for i in range(9)]]
    draft = torch.arange(20, device="cuda")
    target = torch.full((20,), 77, device="cuda")
    target[0] = 10  # node 10 has no children
    k, v = torch.randn(2, 20, 64, device="cuda")
    steps = 0
    rows = Rows([20], parents)
    while True:
        try:
            cache.write(0, k, v, rows)
        except ValueError:
            break
        _, count, _ = cache.commit(draft, target, rows)
        if told:
            cache.kept(count.tolist())
        steps += 1
    assert cache.lens.tolist() == [2 * steps] and steps == (55 if told else 37)  # (128 - 20) // growth + 1


def test_making_rows_does_not_wait_for_the_device():
    from opworks_b200.tree import Rows

    trees = [[-1] + list(range(63))] * 32
    Rows([64] * 32, trees)  # pinned memory is there from here on
    big = torch.empty(1 << 28, device="cuda")
    torch.cuda.synchronize()
    done = torch.cuda.Event()
    for _ in range(200):  # about 60 ms of stores
        big.fill_(1.0)
    done.record()
    rows = Rows([64] * 32, trees)
    first = rows.start
    waited = done.query()
    torch.cuda.synchronize()
    assert not waited
    assert first[-1].item() == 2048 and rows.parents[:64].tolist() == trees[0]
