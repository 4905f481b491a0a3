"""GPU tests of tree attention at the ends of its range: large scores, rows of unlike size, masks that leave whole tiles
empty, long prompts.

Tolerance, as in tests/test_tree_cache_gpu.py: 2^-17 mass max|v| + (keys / 16 + 16) 2^-23 max|v|, both maxima over the
keys that the row sees (a key that it does not see has no influence), and for bf16 rows 2^-8 |o| + 2^-10 max|v| more."""

import math

import numpy as np
import pytest

import tree_cache_plain as plain

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TYPES = {0: torch.float32, 1: torch.bfloat16}


@pytest.fixture(scope="module")
def ops():
    import opworks_b200

    return opworks_b200.ops_lib()


def dev(a):
    return (a if isinstance(a, torch.Tensor) else torch.from_numpy(np.ascontiguousarray(a))).cuda()


def starts(rows):
    return np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)


def attend(ops, cache, q, ctx, rows, sees, scale, max_ctx=None):
    """q [total, q_heads, dim] over the cache -> out in 64 bits. sees: a list of [n, n] truth values, or None for chains."""
    total, qh, dim = q.shape
    words = max(1, -(-max(rows) // 32))
    mask = None if sees is None else dev(np.concatenate([plain.pack_mask(s, words) for s in sees]))
    out = torch.full((total, qh, dim), 777.0, dtype=q.dtype, device="cuda")
    kind = 0 if q.dtype == torch.float32 else 1
    # (held until the call has run: an operator takes plain addresses)
    table, lens, start, dq = dev(cache.table), dev(np.array(ctx, np.int32)), dev(starts(rows)), dev(q)
    pools = (dev(cache.k), dev(cache.v)) if cache.fmt == 0 else (dev(cache.pool),)
    rest = (table, cache.stride, lens, start, mask, words, len(rows), total, max(rows), max(ctx) if max_ctx is None else max_ctx,
            qh, cache.kvh, dim, scale, out, qh * dim, 0)
    if cache.fmt == 0:
        ops.tree_attention(dq, kind, qh * dim, *pools, *rest)
    else:
        ops.tree_attention_q8(dq, kind, qh * dim, *pools, cache.fmt, *rest)
    ops.ops_sync(0)
    return out.cpu().double()


def expected(cache, q, ctx, rows, sees, scale):
    """Output in 64 bits, and per row and head the largest scale sum |q k| and the largest |v| that it sees."""
    total, qh, dim = q.shape
    rep, start = qh // cache.kvh, starts(rows)
    out, mass, top = torch.zeros(total, qh, dim, dtype=torch.float64), torch.zeros(total, qh, dtype=torch.float64), torch.zeros(total, qh, dtype=torch.float64)
    for b, n in enumerate(rows):
        if n == 0:
            continue
        k, v = cache.rows(b, 0, ctx[b] + n)
        nodes = np.tril(np.ones((n, n), bool)) if sees is None else sees[b]
        seen = torch.cat([torch.ones(n, ctx[b], dtype=torch.bool), torch.from_numpy(nodes)], 1)
        some = seen.any(0)
        k, v = (torch.where(some[:, None, None], x, torch.zeros((), dtype=torch.float64)) for x in (k, v))
        for h in range(qh):
            x = q[start[b] : start[b + 1], h].double()
            kk, vv = k[:, h // rep], v[:, h // rep]
            s = (scale * (x @ kk.T)).masked_fill(~seen, -math.inf)
            w = torch.softmax(s, 1).nan_to_num(0.0)  # a row of -inf: zeros
            sl = slice(start[b], start[b + 1])
            out[sl, h] = w @ vv
            mass[sl, h] = (abs(scale) * (x.abs() @ kk.abs().T)).masked_fill(~seen, 0.0).amax(1)
            top[sl, h] = vv.abs().amax(1)[None].expand(n, -1).masked_fill(~seen, 0.0).amax(1)
    return out, mass, top


def tolerance(want, mass, top, keys, kind):
    tol = (2.0**-17 * mass * top + (keys / 16 + 16) * 2.0**-23 * top)[..., None].expand_as(want)
    return tol + 2.0**-8 * want.abs() + 2.0**-10 * top[..., None] if kind == 1 else tol


def check(got, want, mass, top, keys, kind):
    tol = tolerance(want, mass, top, keys, kind)
    assert torch.isfinite(got).all()
    err = (got - want).abs()
    assert (err <= tol).all(), f"error {err.max():.3g}, over by {(err - tol).max():.3g}, at {(err - tol).flatten().argmax().item()}"


def queries(total, qh, dim, kind, seed):
    return torch.randn(total, qh, dim, generator=torch.Generator().manual_seed(seed)).to(TYPES[kind])


def set_rows(cache, b, pos, k=None, v=None):
    """Writes rows [n, kvh, dim] of K and V at positions `pos` of sequence b."""
    pos = np.asarray(pos)
    blk, slot = torch.from_numpy(cache.table[b, pos // 16].astype(np.int64)), torch.from_numpy(pos % 16)
    for which, x in ((0, k), (1, v)):
        if x is None:
            continue
        if cache.fmt == 0:
            (cache.k, cache.v)[which][blk, :, slot] = x.float()
        else:
            parts = plain.views(cache.pool, cache.dim, cache.fmt)
            c, s = plain.quantise(x, cache.fmt)
            parts[which].view(torch.uint8)[blk, :, slot] = c.view(torch.uint8)
            parts[2 + which][blk, :, slot] = s


def scale_rows(cache, b, pos, factor):
    """Multiplies the K and V rows at the positions by `factor` (8-bit: their scales)."""
    pos = np.asarray(pos)
    blk, slot = torch.from_numpy(cache.table[b, pos // 16].astype(np.int64)), torch.from_numpy(pos % 16)
    if cache.fmt == 0:
        for x in (cache.k, cache.v):
            x[blk, :, slot] = x[blk, :, slot] * factor
    else:
        for x in plain.views(cache.pool, cache.dim, cache.fmt)[2:]:
            x[blk, :, slot] = x[blk, :, slot] * factor


# ------------------------------------------------------------------ large scores


@pytest.mark.parametrize("size", [1e4, 1e5, 1e6])
@pytest.mark.parametrize("fmt,kind,dim,ctx", [
    (0, 0, 64, 500), (0, 0, 128, 500), (0, 0, 64, 3000), (0, 1, 64, 500), (0, 1, 128, 500), (1, 0, 64, 500), (1, 0, 64, 3000),
    (1, 1, 64, 500), (1, 1, 128, 500), (2, 0, 64, 500), (2, 1, 64, 500), (2, 1, 128, 3000)])
def test_scores_that_leave_no_bits_for_their_difference_end(ops, fmt, kind, size, dim, ctx):
    """Scores of 2^28 to 2^40 with 50 nodes: the call returns, and what it gives is a finite mean of V rows."""
    rows = [50]
    cache = plain.Cache([ctx + 50], 1, dim, fmt, 5)
    q = (queries(50, 4, dim, 0, 6) * size).to(TYPES[kind])
    k, _ = cache.rows(0)
    set_rows(cache, 0, np.arange(ctx + 50), k=k * size)
    got = attend(ops, cache, q, [ctx], rows, None, 1 / math.sqrt(dim))
    assert torch.isfinite(got).all()
    assert got.abs().max() <= cache.rows(0)[1].abs().max() * 1.01


# ------------------------------------------------------------------ bits of the scores


def opposed(rng_seed, n, heads, dim, size):
    """n rows about -size along the direction that `along` queries have, with noise."""
    return torch.randn(n, heads, dim, generator=torch.Generator().manual_seed(rng_seed)) - size


@pytest.mark.parametrize("fmt", [0, 1, 2])
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("ctx,rows", [(300, 3), (300, 60), (2000, 140)])
@pytest.mark.parametrize("size", [60, 200])
def test_scores_keep_their_bits(ops, fmt, kind, dim, ctx, rows, size):
    """Scores of -60 and -200 in log2 units that differ by about one: a K row rounded to 11 bits would show."""
    cache = plain.Cache([ctx + rows], 1, dim, fmt, 7)
    set_rows(cache, 0, np.arange(ctx + rows), k=opposed(1, ctx + rows, 1, dim, size / (math.log2(math.e) * math.sqrt(dim))))
    q = (0.2 * queries(rows, 4, dim, 0, 8) + 1.0).to(TYPES[kind])
    got = attend(ops, cache, q, [ctx], [rows], None, 1 / math.sqrt(dim))
    check(got, *expected(cache, q, [ctx], [rows], None, 1 / math.sqrt(dim)), ctx + rows, kind)


@pytest.mark.parametrize("fmt", [0, 1, 2])
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("size", [60, 200, 800])
def test_scores_keep_their_bits_over_few_keys(ops, fmt, kind, dim, size):
    """The same with 20 keys to a node, among which errors do not average out; 100 nodes are one tile of keys."""
    rows = 100
    cache = plain.Cache([rows], 1, dim, fmt, 9)
    set_rows(cache, 0, np.arange(rows), k=opposed(2, rows, 1, dim, size / (math.log2(math.e) * math.sqrt(dim))))
    q = (0.2 * queries(rows, 4, dim, 0, 8) + 1.0).to(TYPES[kind])
    sees = [node_mask("window", rows)]
    got = attend(ops, cache, q, [0], [rows], sees, 1 / math.sqrt(dim))
    check(got, *expected(cache, q, [0], [rows], sees, 1 / math.sqrt(dim)), rows, kind)


# ------------------------------------------------------------------ masks that leave whole tiles empty


def node_mask(shape, n):
    i, j = np.arange(n)[:, None], np.arange(n)[None]
    if shape == "self":  # every node is a root of its own
        return i == j
    if shape == "window":  # the last 20 nodes
        return (j <= i) & (j > i - 20)
    return (j <= i) & (i // 90 == j // 90)  # packed pieces of 90 tokens


@pytest.mark.parametrize("fmt", [0, 1, 2])
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("shape,ctx,rows", [("self", [0], [200]), ("window", [0, 100], [300, 170]), ("pieces", [0, 3], [600, 150]),
                                            ("self", [30], [1100]), ("pieces", [0], [1300])])
@pytest.mark.parametrize("below", [15, 60])
def test_rows_whose_first_tile_is_masked(ops, fmt, kind, dim, shape, ctx, rows, below):
    """Nodes that see none of the first 128 (or, in a split, any earlier) keys, with scores of about -15 and -60 in log2
    units: one CTA's tiles, and several CTAs' (1100 nodes and more)."""
    sees = [node_mask(shape, n) for n in rows]
    cache = plain.Cache([c + n for c, n in zip(ctx, rows)], 1, dim, fmt, 7)
    size = below / (math.log2(math.e) * math.sqrt(dim))
    for b, (c, n) in enumerate(zip(ctx, rows)):
        set_rows(cache, b, np.arange(c + n), k=opposed(b, c + n, 1, dim, size))
    q = (0.2 * queries(sum(rows), 2, dim, 0, 8) + 1.0).to(TYPES[kind])
    got = attend(ops, cache, q, ctx, rows, sees, 1 / math.sqrt(dim))
    want = expected(cache, q, ctx, rows, sees, 1 / math.sqrt(dim))
    check(got, *want, max(c + n for c, n in zip(ctx, rows)), kind)


# ------------------------------------------------------------------ rows of unlike size


def hidden_large_rows(ops, fmt, kind, dim, ctx, n, factor, alone):
    """Nodes whose K and V rows (8-bit: scales) are `factor` times as large as the others': hidden from every node, or
    (alone) seen by themselves only."""
    rng = np.random.default_rng(3)
    cache = plain.Cache([ctx + n], 2, dim, fmt, 11)
    sees = plain.tree(rng, n)[1]
    bad = sorted({1, n // 2, n - 1})
    for j in bad:
        sees[:, j] = False
        sees[j, j] = alone
    scale_rows(cache, 0, [ctx + j for j in bad], factor)
    q = queries(n, 8, dim, kind, 12)
    got = attend(ops, cache, q, [ctx], [n], [sees], 1 / math.sqrt(dim))
    check(got, *expected(cache, q, [ctx], [n], [sees], 1 / math.sqrt(dim)), ctx + n, kind)


@pytest.mark.parametrize("fmt,kind,dim", [(0, 0, 64), (0, 0, 128), (0, 1, 64), (0, 1, 128), (1, 0, 64), (1, 1, 64), (1, 1, 128),
                                          (2, 0, 64), (2, 1, 64), (2, 1, 128)])
@pytest.mark.parametrize("ctx,n", [(0, 70), (50, 60), (300, 200)])
@pytest.mark.parametrize("factor", [1e6, 1e20, 1e30])
@pytest.mark.parametrize("alone", [False, True])
def test_large_rows_that_a_node_does_not_see(ops, fmt, kind, dim, ctx, n, factor, alone):
    hidden_large_rows(ops, fmt, kind, dim, ctx, n, factor, alone)


@pytest.mark.parametrize("fmt", [0, 1, 2])
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("ctx,n", [(0, 5), (50, 3), (300, 6)])
@pytest.mark.parametrize("factor", [1e6, 1e20, 1e30])
def test_large_rows_that_few_nodes_do_not_see(ops, fmt, kind, dim, ctx, n, factor):
    hidden_large_rows(ops, fmt, kind, dim, ctx, n, factor, False)


@pytest.mark.parametrize("fmt", [1, 2])
@pytest.mark.parametrize("ctx,n", [(0, 70), (300, 100)])
@pytest.mark.parametrize("factor", [1e6, 1e20, 1e30])
def test_large_rows_that_a_node_does_not_see_wide_heads(ops, fmt, ctx, n, factor):
    hidden_large_rows(ops, fmt, 0, 128, ctx, n, factor, False)


@pytest.mark.parametrize("fmt", [0, 1, 2])
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("ctx,n", [(0, 5), (50, 3), (300, 6)])
@pytest.mark.parametrize("factor", [1e6, 1e20, 1e30])
def test_large_rows_that_few_nodes_see(ops, fmt, kind, dim, ctx, n, factor):
    hidden_large_rows(ops, fmt, kind, dim, ctx, n, factor, True)


@pytest.mark.parametrize("fmt", [0, 1, 2])
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("size", [1e3, 1e4, 1e5, 1e6, 1e9])
@pytest.mark.parametrize("ctx,n", [(500, 2), (20, 12), (500, 50), (0, 140)])
def test_large_scores_choose_the_largest(ops, fmt, kind, dim, size, ctx, n):
    """Scores of 2^21 to 2^61: where the largest is ahead by more than the scores' rounding (2^-18 of their mass, and 40),
    the output is its V row."""
    cache = plain.Cache([ctx + n], 1, dim, fmt, 5)
    q = (queries(n, 4, dim, 0, 6) * size).to(TYPES[kind])
    k, _ = cache.rows(0)
    set_rows(cache, 0, np.arange(ctx + n), k=k * size)
    scale = 1 / math.sqrt(dim)
    got = attend(ops, cache, q, [ctx], [n], None, scale)
    assert torch.isfinite(got).all()
    k, v = cache.rows(0)
    seen = torch.cat([torch.ones(n, ctx, dtype=torch.bool), torch.ones(n, n, dtype=torch.bool).tril()], 1)
    s = (scale * torch.einsum("nhd,kd->nhk", q.double(), k[:, 0])).masked_fill(~seen[:, None], -math.inf)
    mass = scale * torch.einsum("nhd,kd->nhk", q.double().abs(), k[:, 0].abs()).amax(-1)
    top = s.sort(-1, descending=True)
    gap = top.values[..., 0] - top.values[..., 1] if ctx + n > 1 else torch.full_like(mass, math.inf)
    sure = gap > 2.0**-18 * mass + 40
    assert sure.double().mean() > 0.9
    want = v[:, 0][top.indices[..., 0]]
    err = (got - want).abs()[sure]
    assert (err <= (2.0**-7 if kind else 2.0**-18) * v.abs().max()).all(), f"{err.max():.3g}"


@pytest.mark.parametrize("fmt", [0, 1, 2])
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [1, 3, 50])
@pytest.mark.parametrize("bits,back", [(10, False), (20, False), (30, False), (20, True)])
def test_small_rows_after_large_ones(ops, fmt, kind, dim, n, bits, back):
    """Pages whose K and V rows are 2^bits times as large as the others' and weigh nothing (their scores are far below):
    the small rows, after them (or before), keep the bits that they have on their own."""
    ctx, large = 2200, 1024
    cache = plain.Cache([ctx + n], 2, dim, fmt, 13)
    at = np.arange(ctx - large, ctx) // 16 * 16 if back else np.arange(large)
    at = np.arange(1168, 1168 + large) if back else at
    k = opposed(3, large, 2, dim, 3.0).clamp(max=-0.5)
    set_rows(cache, 0, at, k=k * 2.0**bits, v=queries(large, 2, dim, 0, 14).float() * 2.0**bits)
    q = (0.2 * queries(n, 4, dim, 0, 8) + 1.0).clamp(min=0.1).to(TYPES[kind])
    scale = 1 / math.sqrt(dim)
    got = attend(ops, cache, q, [ctx], [n], None, scale)
    # what the large rows weigh is 0 in 64 bits too: the others alone give the result and the tolerance
    want, _, _ = expected(cache, q, [ctx], [n], None, scale)
    set_rows(cache, 0, at, k=torch.zeros(large, 2, dim), v=torch.zeros(large, 2, dim))
    _, mass, top = expected(cache, q, [ctx], [n], None, scale)
    check(got, want, mass, top, ctx + n, kind)


@pytest.mark.parametrize("fmt", [0, 1, 2])
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [1, 3, 50])
@pytest.mark.parametrize("bits", [10, 20, 30])
def test_small_rows_after_rows_of_large_values(ops, fmt, kind, dim, n, bits):
    """The same where scores are ordinary: K rows (fp32) with one value of 2^bits that no query looks at, V rows of that
    size, scores of -60 (in log2 units) below the others'."""
    ctx, large = 2200, 1024
    cache = plain.Cache([ctx + n], 2, dim, fmt, 13)
    k = opposed(3, large, 2, dim, 60 / (math.log2(math.e) * math.sqrt(dim)))
    if fmt == 0:
        k[..., 0] = 2.0**bits
    set_rows(cache, 0, np.arange(large), k=k, v=queries(large, 2, dim, 0, 14).float() * 2.0**bits)
    q = (0.2 * queries(n, 4, dim, 0, 8) + 1.0).to(TYPES[kind])
    q[..., 0] = 0
    scale = 1 / math.sqrt(dim)
    got = attend(ops, cache, q, [ctx], [n], None, scale)
    want, _, _ = expected(cache, q, [ctx], [n], None, scale)
    set_rows(cache, 0, np.arange(large), k=torch.zeros(large, 2, dim), v=torch.zeros(large, 2, dim))
    _, mass, top = expected(cache, q, [ctx], [n], None, scale)
    check(got, want, mass, top, ctx + n, kind)


# ------------------------------------------------------------------ many sequences, long prompts


@pytest.mark.parametrize("fmt", [0, 1, 2])
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("dim", [64, 128])
def test_more_sequences_than_run_at_once(ops, fmt, kind, dim):
    """Sequences are taken in the order of their work: it is found in the memory that the first pages are copied to."""
    rng = np.random.default_rng(4)
    ctx, rows = rng.integers(0, 300, 60).tolist(), rng.integers(0, 4, 60).tolist()
    cache = plain.Cache([c + n for c, n in zip(ctx, rows)], 4, dim, fmt, 21)
    q = queries(sum(rows), 8, dim, kind, 22)
    got = attend(ops, cache, q, ctx, rows, None, 1 / math.sqrt(dim))
    check(got, *expected(cache, q, ctx, rows, None, 1 / math.sqrt(dim)), 304, kind)


# ------------------------------------------------------------------ infinities and NaN


@pytest.mark.parametrize("fmt", [0, 1, 2])
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("ctx,n", [(0, 3), (300, 3), (0, 60), (300, 60)])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_queries_that_are_not_finite(ops, fmt, kind, dim, ctx, n, bad):
    """Their own rows are NaN (zeros where they see nothing), all others as they were."""
    cache = plain.Cache([ctx + n], 2, dim, fmt, 23)
    set_rows(cache, 0, np.arange(ctx + n), k=opposed(5, ctx + n, 2, dim, 4.0).clamp(max=-0.5))  # a score of -inf, too
    sees = [np.tril(np.ones((n, n), bool))]
    if ctx == 0:
        sees[0][2] = False
    q = queries(n, 4, dim, kind, 24)
    scale = 1 / math.sqrt(dim)
    want = expected(cache, q, [ctx], [n], sees, scale)
    spoiled = q.clone()
    for i, h in ((0, 1), (1, 2), (2, 0), (n - 1, 3)):
        spoiled[i, h, (7 * i + h) % dim] = bad
    got = attend(ops, cache, spoiled, [ctx], [n], sees, scale)
    hit = ~torch.isfinite(spoiled).all(-1)
    blind = hit & (want[2] == 0)
    assert torch.isnan(got[hit & ~blind]).all() and (got[blind] == 0).all()
    ok = ~hit
    check(got[ok], want[0][ok], want[1][ok], want[2][ok], ctx + n, kind)


@pytest.mark.parametrize("fmt", [0, 1, 2])
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [2, 50])
@pytest.mark.parametrize("at", ["first", "middle", "node"])
def test_keys_that_are_not_finite(ops, fmt, kind, dim, n, at):
    """A NaN and an infinity in a row of the context: every node is NaN; in a node's row: those that see it."""
    ctx = 40
    bad = {"first": 0, "middle": 21, "node": ctx + 1}[at]
    cache = plain.Cache([ctx + n], 2, dim, fmt, 25)
    cache.spoil(0, bad)
    got = attend(ops, cache, queries(n, 8, dim, kind, 26), [ctx], [n], [np.tril(np.ones((n, n), bool))], 1 / math.sqrt(dim))
    first = max(0, bad - ctx)
    assert torch.isnan(got[first:]).all() and torch.isfinite(got[:first]).all()


# ------------------------------------------------------------------ the range of fp32


@pytest.mark.parametrize("fmt", [0, 1, 2])
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("ctx,n", [(0, 5), (300, 3), (0, 60), (900, 60)])
@pytest.mark.parametrize("kexp,vexp", [(100, 0), (-100, 0), (0, 126), (0, -40), (100, 126), (-100, -40)])
def test_rows_at_the_ends_of_fp32(ops, fmt, kind, dim, ctx, n, kexp, vexp):
    """K rows of 2^100 and 2^-100 (with queries that make up for them), V rows up to 3 2^126 and down to 2^-40."""
    cache = plain.Cache([ctx + n], 2, dim, fmt, 27)
    k, v = (queries(ctx + n, 2, dim, 0, s).clamp(-3, 3) for s in (28, 29))
    set_rows(cache, 0, np.arange(ctx + n), k=k * 2.0**kexp, v=v * 2.0**vexp)
    q = queries(n, 8, dim, kind, 30) * 2.0**-kexp
    got = attend(ops, cache, q, [ctx], [n], None, 1 / math.sqrt(dim))
    check(got, *expected(cache, q, [ctx], [n], None, 1 / math.sqrt(dim)), ctx + n, kind)


@pytest.mark.parametrize("fmt", [0, 1, 2])
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kvh,ctx,rows", [(1, [0], [2100]), (2, [1000, 0, 17], [700, 513, 1])])
def test_prompts(ops, fmt, kind, dim, kvh, ctx, rows):
    """Chains of hundreds and thousands of rows, on their own and after a context."""
    cache = plain.Cache([c + n for c, n in zip(ctx, rows)], kvh, dim, fmt, 31)
    q = queries(sum(rows), 2 * kvh, dim, kind, 32)
    got = attend(ops, cache, q, ctx, rows, None, 1 / math.sqrt(dim))
    check(got, *expected(cache, q, ctx, rows, None, 1 / math.sqrt(dim)), max(c + n for c, n in zip(ctx, rows)), kind)


@pytest.mark.parametrize("fmt", [1, 2])
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("dim", [64, 128])
def test_codes_of_rows_that_are_not_finite_are_zero(ops, fmt, kind, dim):
    x = queries(6, 1, dim, kind, 33).view(6, dim)
    x[1, 3], x[2, dim - 1], x[4, 0] = math.inf, math.nan, -math.inf
    cache = plain.Cache([6], 1, dim, fmt, 34)
    pool, rows = dev(cache.pool), dev(x)
    table, first, start = dev(cache.table), dev(np.zeros(1, np.int32)), dev(starts([6]))
    ops.kv_quant_write(rows, rows, kind, dim, pool, fmt, table, cache.stride, first, start, 1, 6, 1, dim, 0)
    codes_k, codes_v, scale_k, scale_v = plain.views(pool.cpu(), dim, fmt)
    blk = int(cache.table[0, 0])
    for codes, scales in ((codes_k, scale_k), (codes_v, scale_v)):
        c, s = codes.view(torch.uint8)[blk, 0, :6], scales[blk, 0, :6]
        for i in range(6):
            bad = i in (1, 2, 4)
            assert bool(torch.isnan(s[i])) == bad and bool(c[i].any()) == (not bad)


# ------------------------------------------------------------------ long sums


@pytest.mark.parametrize("fmt,dim", [(0, 64), (0, 128), (1, 64), (2, 64)])
def test_long_sums_keep_their_bits(ops, fmt, dim):
    """9000 keys of one sign in one CTA (no splits: there are as many sequences as SMs), weights alike: an accumulator that
    is cut off at each of its 560 steps ends up low by half of 560 2^-23. Here it is the same for all the steps: 2^-18, half
    of 64 steps."""
    n, ctx = 33, 9000
    cache = plain.Cache([ctx + n], 1, dim, fmt, 41)
    v = queries(ctx + n, 1, dim, 0, 42).abs().clamp(0.5, 2.0)
    set_rows(cache, 0, np.arange(ctx + n), v=v)
    q = queries(n, 4, dim, 0, 43) * 0.1
    # many sequences with the same pages, so that each gets one CTA
    copies = 150
    many = type("Pages", (), {})()
    many.fmt, many.kvh, many.stride, many.table = fmt, 1, cache.stride, np.repeat(cache.table, copies, 0)
    for name in ("k", "v", "pool"):
        if hasattr(cache, name):
            setattr(many, name, getattr(cache, name))
    got = attend(ops, many, q.repeat(copies, 1, 1), [ctx] * copies, [n] * copies, [np.eye(n, dtype=bool)] * copies, 1 / math.sqrt(dim))
    want, mass, top = expected(cache, q, [ctx], [n], [np.eye(n, dtype=bool)], 1 / math.sqrt(dim))
    got = got.view(copies, n, 4, dim)
    assert (got == got[:1]).all()
    err = ((got[0] - want).abs() / want).max()
    assert err <= 2.0**-18, f"{err:.3g}"


@pytest.mark.parametrize("fmt", [0, 1, 2])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [1, 5])
def test_long_sums_of_few_rows_keep_their_bits(ops, fmt, dim, n):
    """24,000 keys of one sign in one CTA: 190 (8-bit) to 375 steps of a warp; the bound is that of 64 steps cut off."""
    ctx, copies = 24000, 300
    cache = plain.Cache([ctx + n], 1, dim, fmt, 44)
    set_rows(cache, 0, np.arange(ctx + n), v=queries(ctx + n, 1, dim, 0, 45).abs().clamp(0.5, 2.0))
    q = queries(n, 2, dim, 0, 46) * 0.1
    many = type("Pages", (), {})()
    many.fmt, many.kvh, many.stride, many.table = fmt, 1, cache.stride, np.repeat(cache.table, copies, 0)
    for name in ("k", "v", "pool"):
        if hasattr(cache, name):
            setattr(many, name, getattr(cache, name))
    got = attend(ops, many, q.repeat(copies, 1, 1), [ctx] * copies, [n] * copies, None, 1 / math.sqrt(dim)).view(copies, n, 2, dim)
    want, _, _ = expected(cache, q, [ctx], [n], None, 1 / math.sqrt(dim))
    assert (got == got[:1]).all()
    err = ((got[0] - want).abs() / want).max()
    assert err <= 2.0**-18, f"{err:.3g}"


@pytest.mark.parametrize("fmt", [0, 1, 2])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("ctx,n", [(600, 1), (600, 12), (50, 60), (600, 30), (1300, 40)])
def test_fp32_rows_are_off_by_a_millionth_at_most(ops, fmt, dim, ctx, n):
    """Relative 2-norm of the error over all rows: operands and weights to 2^-22, rounded sums: 2^-20 together."""
    cache = plain.Cache([ctx + n], 2, dim, fmt, 51)
    q = queries(n, 8, dim, 0, 52)
    sees = [plain.tree(np.random.default_rng(5), n)[1]]
    got = attend(ops, cache, q, [ctx], [n], sees, 1 / math.sqrt(dim))
    want, _, _ = expected(cache, q, [ctx], [n], sees, 1 / math.sqrt(dim))
    err = (got - want).norm() / want.norm()
    assert err <= 2.0**-20, f"{err:.3g}"


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [1, 3, 50])
@pytest.mark.parametrize("bits", [60, 90, 110, 125])
@pytest.mark.parametrize("fmt", [0, 1])
def test_v_rows_that_differ_by_powers_of_two(ops, fmt, kind, dim, n, bits):
    """Pages of V of 2^bits, then of 1, all weighing alike: the sum stays in fp32's range."""
    ctx, large = 2200, 1024
    cache = plain.Cache([ctx + n], 2, dim, fmt, 61)
    set_rows(cache, 0, np.arange(large), v=queries(large, 2, dim, 0, 62).clamp(-2, 2) * 2.0**bits)
    q = queries(n, 4, dim, kind, 63) * 0.25
    got = attend(ops, cache, q, [ctx], [n], None, 1 / math.sqrt(dim))
    check(got, *expected(cache, q, [ctx], [n], None, 1 / math.sqrt(dim)), ctx + n, kind)
