"""What the drafted-token wrapper (opworks_b200/tree.py) and the plain forms of
its GPU tests compute on the host."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import tree_cache_plain as plain  # noqa: E402


def test_tree_mask_is_ancestors_and_self():
    from opworks_b200.tree import tree_mask

    rng = np.random.default_rng(0)
    for n in (1, 5, 33, 70):
        parent, sees = plain.tree(rng, n)
        words = -(-n // 32)
        assert np.array_equal(tree_mask(list(parent), words), plain.pack_mask(sees, words))
    with pytest.raises(ValueError):
        tree_mask([-1, 1], 1)
    with pytest.raises(ValueError):
        tree_mask([-1, -2], 1)


def test_plain_commit_walks_to_the_first_right_child():
    #        0 -> 1, 2, 3 ; 2 -> 4 ; 3 -> 5
    parent = [-1, 0, 0, 0, 2, 3]
    draft, target = [9, 7, 8, 8, 5, 5], [8, 0, 5, 5, 1, 1]
    assert plain.commit(draft, target, parent) == [0, 2, 4]
    assert plain.commit(draft, [3] + target[1:], parent) == [0]
    assert plain.commit([], [], []) == []


@pytest.mark.parametrize("fmt", [1, 2])
def test_plain_quantisation_is_within_half_a_code(fmt):
    x = torch.randn(50, 64, generator=torch.Generator().manual_seed(1))
    x[3] = 0
    c, s = plain.quantise(x, fmt)
    err = (plain.dequantise(c, s) - x.double()).abs()
    half = 0.5 * s[:, None] if fmt == 1 else torch.maximum(x.abs() / 16, s[:, None] / 1024)
    assert (err <= half.double() * (1 + 1e-5)).all()
    bad = x.clone()
    bad[5, 6] = float("inf")
    c, s = plain.quantise(bad, fmt)
    assert torch.isnan(s[5]) and not c[5].float().any()


def test_mask_rows_of_a_random_tree_and_the_attention_agree():
    """One query over three keys by hand."""
    cache = plain.Cache([3], 1, 64, 0, 0)
    q = torch.zeros(1, 1, 64)
    out, _, _ = plain.attention(cache, q, [2], [0, 1], [np.array([[True]])], 1.0)
    assert torch.allclose(out[0, 0], cache.rows(0)[1][:, 0].mean(0))
