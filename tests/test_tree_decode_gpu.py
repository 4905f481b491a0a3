"""The drafted-token path as a program uses it: examples/tree_decode.py on the
GPU, and the wrapper's cache against what was written to it."""

import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("format", ["int8", "e4m3", "f32"])
def test_drafted_trees_give_the_tokens_of_single_steps(format):
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    try:
        import tree_decode
    finally:
        sys.path.pop(0)
    plain, steps, drafted, fewer = tree_decode.main(format, 24, quiet=True)
    assert plain == drafted
    assert fewer < steps  # drafts were accepted
    assert len({tuple(p) for p in plain}) == 3 and len(set(sum(plain, []))) > 10  # and the texts are no constants


@pytest.mark.parametrize("format", ["int8", "e4m3"])
def test_cache_gives_back_what_it_took(format):
    from opworks_b200.tree import PagedCache, Rows

    cache = PagedCache(2, 3, 100, 2, 64, format)
    rows = Rows([5, 0, 33])
    k, v = torch.randn(2, rows.total, 128, device="cuda")
    cache.write(1, k, v, rows)
    got_k, got_v = cache.read(1, rows)
    top = k.view(-1, 2, 64).abs().amax(-1, keepdim=True)
    step = top / 254 if format == "int8" else torch.maximum(k.view(-1, 2, 64).abs() / 16, top / 448 / 1024)
    assert ((got_k - k.view(-1, 2, 64)).abs() <= step * 1.0001).all()
    assert (got_v - v.view(-1, 2, 64)).abs().max() < 0.3
    assert not cache.pool[0].any()
    with pytest.raises(ValueError):
        cache.write(0, k, v, Rows([5, 0, 113]))
