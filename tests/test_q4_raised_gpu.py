"""Attention over the 4-bit cache where a row's reference is raised inside a tile (include/ops/tree_attention_q4_tiles.cuh): the
tile's earlier weights, which are stored already, have to go down by the same factor as their sum."""

import math

import numpy as np
import pytest

import q4_plain
import tree_cache_plain as plain

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TYPES = {0: torch.float32, 1: torch.bfloat16}
UNIT = 0.05  # log2 units of score for one unit of the sum of a key's codes, before the row's factor


@pytest.fixture(scope="module")
def ops():
    import opworks_b200

    return opworks_b200.ops_lib()


def cache_with_scores(levels, dim, values, seed):
    """A sequence whose key j has codes that add up to levels[j] and scales of one, so that a query of one number c in all
    dims scores c * levels[j] exactly; V is values[j] in all dims, or random codes of a quarter where that is NaN."""
    n = len(levels)
    cache = q4_plain.Cache4([n], 1, dim, seed)
    kc, vc, ks, vs = q4_plain.views(cache.pool, dim)
    rng = np.random.default_rng(seed)
    for j, level in enumerate(levels):
        block, slot = int(cache.table[0, j // 16]), j % 16
        each, rest = divmod(int(level), dim)
        codes = np.full(dim, each) + (np.arange(dim) < rest)
        assert abs(codes).max() <= 7 and codes.sum() == level
        v = rng.integers(-4, 5, dim) if math.isnan(values[j]) else np.full(dim, round(4 * values[j]))
        for into, scales, c in ((kc, ks, codes), (vc, vs, v)):
            packed = (c[0::2] + 8) | ((c[1::2] + 8) << 4)
            into[block, 0, :, slot] = torch.from_numpy(packed.astype(np.uint8)).view(dim // 32, 16)
            scales[block, 0, :, slot] = 1.0 if scales is ks else 0.25
    return cache


@pytest.mark.parametrize("kind,dim", [(0, 64), (0, 128), (1, 64), (1, 128)])
@pytest.mark.parametrize("n", [20, 40])  # one row tile of two streams of keys; two row tiles
@pytest.mark.parametrize("chunk", [1, 2, 3])
@pytest.mark.parametrize("above", [1.4, 3.0, 5.0, 6.5])
def test_a_reference_raised_within_a_tile(ops, kind, dim, n, chunk, above):
    """Two tiles of equal scores set the references; then 32 keys just below what makes a reference rise, and one key above
    it by `above` log2 units in the chunk behind them, which has no others of weight.

    fp32: scores are whole numbers times the factor of a row, which two roundings of numbers below 32 put off by 2^-18 log2
    units, weights have 22 bits: less than 8e-6 of a weight, of which the output, a mean of numbers up to 1, takes twice as
    much. bf16: weights of 11 bits, rounded once more when they are multiplied down (2^-11 in all; the keys of a kind have
    the same weight, so all of it counts, in a mean of 1 and -1 at most half of it twice), and half a step of the output."""
    rep, ctx = 4, 512
    near = 14.6 if kind else 8.6  # above the reference by less than 15 (fp32 rows: the reference is 6 below the scores)
    levels, values = np.zeros(ctx + n, int), np.full(ctx + n, np.nan)
    levels[256:] = round(-20 / UNIT)
    for tile in (2, 3):
        at = 128 * tile + 32 * (chunk - 1)
        levels[at : at + 32], values[at : at + 32] = round(near / UNIT), 1.0
        levels[at + 32 + 7 * tile], values[at + 32 + 7 * tile] = round((near + above) / UNIT), -1.0
    cache = cache_with_scores(levels, dim, values, 3)
    factor = 1 - torch.arange(n * rep) % 8 / 256
    q = factor[:, None].expand(-1, dim).reshape(n, rep, dim).contiguous()
    scale = UNIT * math.log(2)
    sees = [plain.tree(None, n, "chain")[1]]
    want, _, top = plain.attention(cache, q, [ctx], [0, n], sees, scale)
    assert top.max() <= 1
    out = torch.empty(n, rep, dim, dtype=TYPES[kind], device="cuda")
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    ops.tree_attention_q4(q.to(TYPES[kind]).cuda(), kind, rep * dim, cache.pool.cuda(), torch.from_numpy(cache.table).cuda(), cache.stride, ints([ctx]), ints([0, n]),
                          None, 0, 1, n, n, ctx, rep, 1, dim, scale, out, rep * dim, 0)
    err = (out.cpu().double() - want).abs()
    tol = 2.0**-8 * want.abs() + 2.0**-11 if kind else torch.full_like(want, 2.0**-15)
    assert (err <= tol).all(), f"error {err.max():.3g}, over by {(err - tol).max():.3g}"
