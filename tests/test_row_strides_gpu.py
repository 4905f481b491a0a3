"""Rows of any stride and any first element (opworks_b200/tree.py): as if they lay one after another."""

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def layouts(x):
    """The rows of x [n, w] as slices of a wider tensor, at odd places, with odd strides, and turned round."""
    n, w = x.shape
    for first, stride in ((0, w + 8), (3, w + 8), (0, w + 1), (5, w + 3), (1, w)):
        flat = torch.zeros(first + n * stride, device=x.device, dtype=x.dtype)
        view = flat[first:].view(n, stride)[:, :w]
        view.copy_(x)
        yield view
    yield x.t().contiguous().t()


@pytest.mark.parametrize("format", ["int4", "int8", "e4m3", "f32"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("counts", [[5, 0, 12], [1, 0, 0]])
def test_write_takes_rows_of_any_stride(format, dtype, counts):
    from opworks_b200.tree import PagedCache, Rows

    rows = Rows(counts)
    k, v = torch.randn(2, rows.total, 128, device="cuda").to(dtype)
    pools = []
    for a, b in [(k, v), *zip(layouts(k), layouts(v)), *((x, v) for x in layouts(k)), *((k, x) for x in layouts(v))]:
        cache = PagedCache(1, 3, 64, 2, 64, format)
        cache.write(0, a, b, rows)
        pools.append((cache.k, cache.v) if format == "f32" else (cache.pool,))
    for pool in pools[1:]:
        assert all(torch.equal(x, y) for x, y in zip(pool, pools[0]))
    cache = PagedCache(1, 3, 64, 2, 64, format)  # one row for all tokens
    cache.write(0, k[:1].expand(rows.total, 128), v[:1].expand(rows.total, 128), rows)
    want = PagedCache(1, 3, 64, 2, 64, format)
    want.write(0, k[:1].repeat(rows.total, 1), v[:1].repeat(rows.total, 1), rows)
    assert torch.equal(cache.k, want.k) if format == "f32" else torch.equal(cache.pool, want.pool)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 7])
def test_norm_and_rotation_take_rows_of_any_stride(dtype, n):
    from opworks_b200.tree import qk_norm_rope

    q, k = torch.randn(n, 256, device="cuda").to(dtype), torch.randn(n, 128, device="cuda").to(dtype)
    pos, inv = torch.arange(n, dtype=torch.int32, device="cuda") * 100, (10000.0 ** (-torch.arange(0, 64, 2) / 64)).cuda()
    weight = torch.rand(64, device="cuda") + 0.5
    heads = lambda x: x.unflatten(1, (-1, 64))  # noqa: E731
    want = qk_norm_rope(heads(q), heads(k), pos, inv, weight, weight)
    for a, b in list(zip(layouts(q), layouts(k)))[:-1]:
        before = a.clone(), b.clone()
        got = qk_norm_rope(heads(a), heads(b), pos, inv, weight, weight)
        assert all(torch.equal(x, y) for x, y in zip(got, want)) and torch.equal(a, before[0]) and torch.equal(b, before[1])
    odd = torch.zeros(1 + n * 256, device="cuda", dtype=dtype)[1:].view(n, 4, 64)
    with pytest.raises(ValueError, match="aligned"):  # what is written has to lie right
        qk_norm_rope(heads(q), heads(k), pos, inv, weight, weight, out=(odd, torch.empty_like(heads(k))))
