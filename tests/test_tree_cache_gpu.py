"""GPU tests of the 8-bit paged KV cache and the drafted-token step, through
libopworks_ops.so, against the plain forms of tests/tree_cache_plain.py.

Tolerances. Codes, scales and rows read back are one IEEE operation per value
away from the inputs and must be equal. Attention: a score is a sum of D
products accumulated in fp32 in at most 16 + D / 8 steps, operands exact to
2^-22 (two fp16 terms) or better, so it is off by at most 2^-18 sum|q k| scale;
a softmax weight then by twice that, and so the output by 2^-17 mass max|v|;
the sum over keys adds one fp32 rounding per 16 keys: (keys / 16 + 16) 2^-23
max|v|. bf16 rows add the output's rounding, 2^-8 |o|, and that of the weights
to 11 bits or better, 2^-10 max|v|."""

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


# ------------------------------------------------------------------ write / read


def random_rows(total, kvh, dim, kind, pad, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(total, 2 * kvh * dim + pad, generator=g) * torch.exp(torch.randn(1, 2 * kvh * dim + pad, generator=g))
    return x.to(TYPES[kind])


@pytest.mark.parametrize("fmt", [1, 2])
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kvh,rows,first,pad", [
    (1, [1], [0], 0), (8, [1, 1, 1], [15, 16, 2180], 0), (3, [5, 0, 37, 16], [3, 9, 0, 16], 64), (16, [40], [7], 8),
    (2, [1] * 70, list(range(70)), 0)])
def test_write_then_read(ops, fmt, kind, dim, kvh, rows, first, pad):
    total, start = sum(rows), starts(rows)
    wide = random_rows(total, kvh, dim, kind, pad, dim + kvh + fmt)
    cache = plain.Cache([f + n for f, n in zip(first, rows)], kvh, dim, fmt, 5)
    before = cache.pool.clone()
    pool, w = dev(cache.pool), dev(wide)
    k, v = w[:, : kvh * dim], w[:, kvh * dim : 2 * kvh * dim]
    table, pos, st = dev(cache.table), dev(np.array(first, np.int32)), dev(start)
    ops.kv_quant_write(k, v, kind, w.stride(0), pool, fmt, table, cache.stride, pos, st, len(rows), total, kvh, dim, 0)
    want = before.clone()
    kc, vc, ks, vs = plain.views(want, dim, fmt)
    rows_k, rows_v = (wide[:, i * kvh * dim : (i + 1) * kvh * dim].unflatten(-1, (kvh, dim)) for i in (0, 1))
    for b, n in enumerate(rows):
        for i in range(n):
            blk, slot = int(cache.table[b, (first[b] + i) // 16]), (first[b] + i) % 16
            for codes, scales, x in ((kc, ks, rows_k), (vc, vs, rows_v)):
                c, s = plain.quantise(x[start[b] + i], fmt)
                codes.view(torch.uint8)[blk, :, slot] = c.view(torch.uint8)
                scales[blk, :, slot] = s
    got = pool.cpu()
    assert torch.equal(got, want)  # every byte: the untouched ones too
    # the rows are what they should be to half a code
    for codes, scales, x in ((kc, ks, rows_k), (vc, vs, rows_v)):
        for b, n in enumerate(rows):
            p = first[b] + np.arange(n)
            blk, slot = torch.from_numpy(cache.table[b, p // 16].astype(np.int64)), torch.from_numpy(p % 16)
            s = scales[blk, :, slot].double()[..., None]
            y = plain.dequantise(codes.view(torch.uint8)[blk, :, slot].view(codes.dtype), s[..., 0])
            x64 = x[start[b] : start[b + 1]].double()
            half = 0.5 * s if fmt == 1 else torch.maximum(x64.abs() / 16, s / 1024)
            assert (abs(y - x64) <= half * (1 + 1e-5)).all()
    for out_kind in (0, 1):
        back = torch.zeros(total, 2 * kvh * dim + pad, dtype=TYPES[out_kind], device="cuda")
        bk, bv = back[:, : kvh * dim], back[:, kvh * dim : 2 * kvh * dim]
        ops.kv_quant_read(pool, fmt, table, cache.stride, pos, st, len(rows), total, kvh, dim, bk, bv, out_kind,
                          back.stride(0), 0)
        back = back.cpu()
        assert not back[:, 2 * kvh * dim :].any()
        cache.pool = want
        for b, n in enumerate(rows):
            for x, at in zip(cache.rows(b, first[b], first[b] + n), (0, 1)):
                e = x.float().to(TYPES[out_kind]).flatten(1)  # code * scale: exact in 64 bits, rounded once
                if out_kind == 1:
                    e = x.float().bfloat16().flatten(1)
                assert torch.equal(back[start[b] : start[b + 1], at * kvh * dim : (at + 1) * kvh * dim], e)


@pytest.mark.parametrize("fmt", [1, 2])
def test_write_edge_rows(ops, fmt):
    """Rows of zeros, of denormals, of one spike, with an infinity, with a NaN."""
    dim, kvh = 64, 1
    x = torch.randn(7, dim, generator=torch.Generator().manual_seed(3))
    x[0] = 0
    x[1] *= 1e-42
    x[2, 5], x[3, 7], x[4, 9] = 1e30, float("inf"), float("nan")
    x[5] = -0.0
    x[6] = 3e38 * torch.sign(x[6])
    cache = plain.Cache([7], kvh, dim, fmt, 1)
    pool, rows = dev(cache.pool), dev(x)
    args = (dev(cache.table), cache.stride, dev(np.zeros(1, np.int32)), dev(starts([7])), 1, 7, kvh, dim)
    ops.kv_quant_write(rows, rows, 0, dim, pool, fmt, *args, 0)
    back = torch.empty(2, 7, dim, device="cuda")
    ops.kv_quant_read(pool, fmt, *args, back[0], back[1], 0, dim, 0)
    c, s = plain.quantise(x, fmt)
    want = (c.float() * s[:, None])
    got = back.cpu()
    assert torch.equal(got[0].view(torch.int32), got[1].view(torch.int32))  # NaN rows too
    assert torch.equal(torch.isnan(got[0]), torch.isnan(want)) and torch.isnan(got[0][3:5]).all()
    keep = ~torch.isnan(want)
    assert torch.equal(got[0][keep], want[keep])
    kc = plain.views(pool.cpu(), dim, fmt)[0].view(torch.uint8)
    blk = int(cache.table[0, 0])
    assert not kc[blk, 0, 3:5].any() and not (kc[blk, 0, :7] & 0x7F == 0x7F).any() or fmt == 1


def test_rows_outside_the_table_are_left_out(ops):
    dim, kvh = 64, 2
    cache = plain.Cache([32], kvh, dim, 1, 2, spare_columns=0)
    x = dev(torch.randn(4, kvh * dim))
    pool, before = dev(cache.pool), cache.pool.clone()
    for first in (32, 1000000, 2**31 - 2, -4):
        ops.kv_quant_write(x, x, 0, kvh * dim, pool, 1, dev(cache.table), cache.stride, dev(np.array([first], np.int32)),
                           dev(starts([4])), 1, 4, kvh, dim, 0)
    assert torch.equal(pool.cpu(), before)


# ------------------------------------------------------------------ attention


def attention_case(ops, fmt, kind, dim, kvh, rep, ctx, rows, trees="tree", q_pad=0, seed=0, spoil=(), sees=None,
                   stream=None, scale=None):
    rng = np.random.default_rng(seed)
    qh, total, start = kvh * rep, sum(rows), starts(rows)
    cache = plain.Cache([c + n for c, n in zip(ctx, rows)], kvh, dim, fmt, seed + 1)
    if sees is None:
        sees = [plain.tree(rng, n, trees)[1] for n in rows]
    for b, j in spoil:
        cache.spoil(b, ctx[b] + j)
    q = torch.randn(total, qh * dim + q_pad, generator=torch.Generator().manual_seed(seed + 2)).to(TYPES[kind])
    words = max(1, -(-max(rows) // 32))
    mask = None if trees == "chain" else dev(np.concatenate([plain.pack_mask(s, words) for s in sees]))
    scale = 1 / math.sqrt(dim) if scale is None else scale
    dq = dev(q)
    out = torch.full((total, qh * dim + q_pad), 777.0, dtype=TYPES[kind], device="cuda")
    args = (dev(cache.table), cache.stride, dev(np.array(ctx, np.int32)), dev(start), mask, words, len(rows), total,
            max(rows), max(ctx), qh, kvh, dim, scale, out, qh * dim + q_pad)
    pools = (dev(cache.k), dev(cache.v)) if fmt == 0 else (dev(cache.pool), fmt)
    call = ops.tree_attention if fmt == 0 else ops.tree_attention_q8
    torch.cuda.synchronize()
    call(dq, kind, qh * dim + q_pad, *pools, *args, 0 if stream is None else stream.cuda_stream)
    ops.ops_sync(0 if stream is None else stream.cuda_stream)
    got = out.cpu()
    assert (got[:, qh * dim :] == 777.0).all()
    got = got[:, : qh * dim].double().view(total, qh, dim)
    want, mass, top = plain.attention(cache, q[:, : qh * dim].reshape(total, qh, dim), ctx, start, sees, scale)
    keys = max(c + n for c, n in zip(ctx, rows))
    tol = 2.0**-17 * mass * top + (keys / 16 + 16) * 2.0**-23 * top
    tol = tol[..., None].expand_as(want)
    if kind == 1:
        tol = tol + 2.0**-8 * want.abs() + 2.0**-10 * top[..., None]
    assert torch.isfinite(got).all()
    err = (got - want).abs()
    assert (err <= tol).all(), f"error {err.max():.3g}, over by {(err - tol).max():.3g}"
    return got


@pytest.mark.parametrize("fmt", [0, 1, 2])
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kvh,rep,ctx,rows", [
    (1, 1, [0], [1]),                                  # nothing but itself
    (8, 4, [511], [1]),                                # a plain decode step
    (2, 4, [15, 16, 17, 0], [1, 5, 2, 31]),            # pages that end inside a tree
    (2, 7, [100, 3], [7, 33]),                         # odd group, two mask words
    (1, 16, [31, 64, 200], [26, 0, 8]),                # an empty sequence among others
    (3, 3, [1000], [64]),
    (1, 8, [40, 700], [100, 3])])
def test_tree_attention(ops, fmt, kind, dim, kvh, rep, ctx, rows):
    attention_case(ops, fmt, kind, dim, kvh, rep, ctx, rows, seed=dim + rep)


@pytest.mark.parametrize("fmt", [0, 1, 2])
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("dim,kvh,rep,ctx,rows", [(64, 1, 4, [5000], [1]), (64, 2, 4, [0, 30], [150, 17]),
                                                  (128, 1, 2, [2050, 1], [40, 1]), (64, 8, 4, [3000, 10], [5, 5])])
def test_chains_without_a_mask(ops, fmt, kind, dim, kvh, rep, ctx, rows):
    attention_case(ops, fmt, kind, dim, kvh, rep, ctx, rows, trees="chain", seed=3)


@pytest.mark.parametrize("fmt", [0, 1, 2])
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kvh,rep,ctx,rows", [(1, 4, [5003], [11]), (2, 8, [2600, 4100], [24, 3]), (1, 2, [7000], [2])])
def test_long_contexts(ops, fmt, kind, dim, kvh, rep, ctx, rows):
    """Every ring and barrier phase of the kernels many times over, on few CTAs and on several that are joined."""
    attention_case(ops, fmt, kind, dim, kvh, rep, ctx, rows, seed=5)


@pytest.mark.parametrize("fmt", [0, 1, 2])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [3, 40])
def test_rows_that_see_nothing_are_zero(ops, fmt, dim, n):
    rng = np.random.default_rng(1)
    sees = [rng.random((n, n)) < 0.3, rng.random((2, 2)) < 2]
    sees[0][1] = False
    sees[0][n - 1] = False
    got = attention_case(ops, fmt, 0, dim, 2, 4, [0, 9], [n, 2], sees=sees, seed=7)
    assert (got[1] == 0).all() and (got[n - 1] == 0).all()


@pytest.mark.parametrize("fmt", [0, 1, 2])
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [6, 50])
def test_masked_infinities_and_nans_have_no_influence(ops, fmt, kind, dim, n):
    rng = np.random.default_rng(2)
    sees = [plain.tree(rng, n)[1], plain.tree(rng, n)[1]]
    bad = [(0, 2), (0, n - 1), (1, 4)]
    for b, j in bad:
        sees[b][:, j] = False
    attention_case(ops, fmt, kind, dim, 2, 4, [30, 0], [n, n], sees=sees, spoil=bad, seed=8)


@pytest.mark.parametrize("fmt", [0, 1, 2])
def test_strided_rows_and_another_stream(ops, fmt):
    attention_case(ops, fmt, 0, 64, 2, 4, [77, 5], [9, 3], q_pad=64, seed=9)
    attention_case(ops, fmt, 1, 128, 2, 4, [77, 5], [9, 40], q_pad=8, seed=9)
    attention_case(ops, fmt, 0, 64, 2, 4, [77, 5], [9, 3], seed=10, stream=torch.cuda.Stream())


@pytest.mark.parametrize("fmt", [0, 1, 2])
@pytest.mark.parametrize("scale", [0.0, 4.0, -0.5])
def test_flat_and_peaked_softmax(ops, fmt, scale):
    """scale 0: every key weighs the same; 4: one key takes nearly all; below zero: the order turns round."""
    attention_case(ops, fmt, 0, 64, 1, 4, [600], [8], seed=11, scale=scale)


@pytest.mark.parametrize("fmt", [0, 1, 2])
def test_two_calls_give_the_same_bits(ops, fmt):
    a = attention_case(ops, fmt, 0, 64, 2, 4, [900, 40], [26, 8], seed=12)
    b = attention_case(ops, fmt, 0, 64, 2, 4, [900, 40], [26, 8], seed=12)
    assert torch.equal(a, b)


def test_one_token_agrees_with_the_decode_attention(ops):
    """n = 1 over the fp32 pools is what opw_paged_attention_decode computes."""
    lens, kvh, rep = [37, 900, 1], 8, 4
    cache = plain.Cache(lens, kvh, 64, 0, 4, junk=False)
    q = torch.randn(3, kvh * rep * 64, device="cuda")
    a, b = torch.empty_like(q), torch.empty_like(q)
    k, v, table = dev(cache.k), dev(cache.v), dev(cache.table)
    ops.paged_attention_decode(q, k, v, table, cache.stride, dev(np.array(lens, np.int32)), 3, 900, kvh * rep, kvh, a, 0)
    ops.tree_attention(q, 0, kvh * rep * 64, k, v, table, cache.stride, dev(np.array(lens, np.int32) - 1), dev(starts([1, 1, 1])),
                       None, 0, 3, 3, 1, 899, kvh * rep, kvh, 64, 0.125, b, kvh * rep * 64, 0)
    assert (a - b).abs().max() <= 1e-5 * a.abs().max()


@pytest.mark.parametrize("fmt", [0, 1, 2])
def test_blocks_whose_offsets_pass_32_bits(ops, fmt):
    """Pages at the far end of pools of over 2^31 elements (fp32) or 2^32 bytes (8 bits): written, read, attended, kept."""
    dim, rep, ctx, rows = 64, 4, 20, 40
    small = plain.Cache([ctx + rows], 1, dim, fmt, 6, junk=False)
    pages = -(-(ctx + rows) // 16)
    size = 16 * dim if fmt == 0 else 2176
    blocks = 2**31 // size + 100 if fmt == 0 else 2**32 // size + 100
    far = blocks - 1 - np.arange(small.stride)
    table = dev(far[None].astype(np.int32))
    ids = torch.from_numpy(small.table[0, :pages].astype(np.int64))
    to = torch.from_numpy(far[:pages].copy()).cuda()
    pools = [torch.empty(blocks, 1, 16, dim, device="cuda") for _ in range(2)] if fmt == 0 else [torch.empty(blocks, 1, size, dtype=torch.uint8, device="cuda")]
    for big, one in zip(pools, (small.k, small.v) if fmt == 0 else (small.pool,)):
        big[to] = one[ids].cuda()
    parent, sees = plain.tree(np.random.default_rng(1), rows)
    q = torch.randn(rows, rep * dim, generator=torch.Generator().manual_seed(3))
    start, lens = dev(starts([rows])), dev(np.array([ctx], np.int32))
    scale = 1 / math.sqrt(dim)
    want, mass, top = plain.attention(small, q.view(rows, rep, dim), [ctx], [0, rows], [sees], scale)
    for n in (rows, 5):  # 160 query rows, and 20
        out = torch.empty(rows, rep * dim, device="cuda")
        rest = (table, small.stride, lens, start if n == rows else dev(starts([n])), dev(plain.pack_mask(sees, 2)), 2, 1, n, n, ctx,
                rep, 1, dim, scale, out, rep * dim, 0)
        call = ops.tree_attention if fmt == 0 else ops.tree_attention_q8
        call(dev(q), 0, rep * dim, *pools, *(() if fmt == 0 else (fmt,)), *rest)
        err = (out[:n].cpu().double().view(n, rep, dim) - want[:n]).abs()
        assert (err <= (2.0**-17 * mass * top + 20 * 2.0**-23 * top)[:n, :, None]).all()
    path, count, nxt, new = (torch.empty(rows, dtype=torch.int32, device="cuda") for _ in range(4))
    draft = np.arange(rows, dtype=np.int32)
    target = np.full(rows, -7, np.int32)
    for i in range(rows - 1, 0, -1):
        target[parent[i]] = i  # the first child of each is right
    head = (dev(draft), dev(target), dev(parent), start, lens, 1, rows)
    tail = (1, table, small.stride, 1, dim, path, count, nxt, new, 0)
    kept = plain.commit(draft, target, parent)
    if fmt == 0:
        ops.tree_commit(*head, *pools, 0, *tail)
    else:
        ops.tree_commit_q8(*head, *pools, 0, *tail)
    assert path[: len(kept)].tolist() == kept and count[0].item() == len(kept) and len(kept) > 2
    for big, one in zip(pools, (small.k, small.v) if fmt == 0 else (small.pool,)):
        if fmt:
            one, big = plain.views(one, dim, fmt)[0].view(torch.uint8), plain.views(big, dim, fmt)[0].view(torch.uint8)
        for i, node in enumerate(kept):
            src, dst = ctx + node, ctx + i
            assert torch.equal(big[int(far[dst // 16]), 0, dst % 16].cpu(), one[int(small.table[0, src // 16]), 0, src % 16])
    if fmt:
        rows_in = torch.randn(rows, dim, device="cuda")
        args = (table, small.stride, lens, start, 1, rows, 1, dim)
        ops.kv_quant_write(rows_in, rows_in, 0, dim, pools[0], fmt, *args, 0)
        back = torch.empty(2, rows, dim, device="cuda")
        ops.kv_quant_read(pools[0], fmt, *args, back[0], back[1], 0, dim, 0)
        c, s = plain.quantise(rows_in.cpu(), fmt)
        assert torch.equal(back[0].cpu(), c.float() * s[:, None]) and torch.equal(back[0], back[1])


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("rows", [2, 50])
def test_a_visible_row_that_is_not_finite_shows(ops, fmt, rows):
    """A NaN in the context makes every row NaN; in a node, the rows that see it and no others."""
    dim, rep, ctx = 64, 2, 40
    for bad in (7, ctx + 1):
        cache = plain.Cache([ctx + rows], 1, dim, fmt, 3)
        cache.spoil(0, bad)
        q = torch.randn(rows, rep * dim, device="cuda")
        out = torch.empty_like(q)
        mask = plain.pack_mask(np.tril(np.ones((rows, rows), bool)), 2)
        rest = (dev(cache.table), cache.stride, dev(np.array([ctx], np.int32)), dev(starts([rows])), dev(mask), 2, 1, rows, rows, ctx,
                rep, 1, dim, 0.125, out, rep * dim, 0)
        if fmt == 0:
            ops.tree_attention(q, 0, rep * dim, dev(cache.k), dev(cache.v), *rest)
        else:
            ops.tree_attention_q8(q, 0, rep * dim, dev(cache.pool), fmt, *rest)
        got = torch.isnan(out).cpu()
        first = 0 if bad < ctx else bad - ctx
        assert got[first:].all() and not got[:first].any()


# ------------------------------------------------------------------ commit


@pytest.mark.parametrize("fmt", [0, 1, 2])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kvh,layers,ctx,rows,accept", [
    (1, 1, [0], [1], 1.0), (8, 3, [15, 100, 30], [26, 0, 64], 0.9), (2, 2, [5, 5], [70, 33], 1.0), (4, 1, [12], [20], 0.0),
    (1, 17, [3] * 9, [8] * 9, 0.7)])
def test_commit(ops, fmt, dim, kvh, layers, ctx, rows, accept):
    rng = np.random.default_rng(dim + kvh)
    total, start = sum(rows), starts(rows)
    caches = [plain.Cache([c + n for c, n in zip(ctx, rows)], kvh, dim, fmt, 3) for _ in range(1)]
    c0 = caches[0]
    g = torch.Generator().manual_seed(9)
    if fmt == 0:
        pools = [torch.randn(layers, *c0.k.shape, generator=g) for _ in range(2)]
    else:
        pools = [torch.randint(0, 256, (layers, *c0.pool.shape), generator=g, dtype=torch.uint8)]
    parent, draft, target = (np.zeros(total, np.int32) for _ in range(3))
    want_path, want_count, want_next, want_len = np.full(total, -1, np.int32), [], [], []
    want = [p.clone() for p in pools]
    for b, n in enumerate(rows):
        sl = slice(start[b], start[b + 1])
        par, _ = plain.tree(rng, n)
        if accept == 1.0:  # deep: each node follows one of the last two
            par = np.array([-1] + [int(rng.integers(max(0, i - 2), i)) for i in range(1, n)], np.int32)[:n]
        d, t = rng.integers(0, 4, n).astype(np.int32), rng.integers(0, 1000, n).astype(np.int32)  # siblings share tokens
        for i in range(n):
            below = np.flatnonzero(par == i)
            if below.size and rng.random() < accept:
                t[i] = d[rng.choice(below)]
            elif accept == 0.0:
                t[i] = 5
        parent[sl], draft[sl], target[sl] = par, d, t
        path = plain.commit(d, t, par)
        want_path[start[b] : start[b] + len(path)] = path
        want_count.append(len(path))
        want_next.append(t[path[-1]] if path else -1)
        want_len.append(ctx[b] + len(path))
        for i, node in enumerate(path):
            src, dst = ctx[b] + node, ctx[b] + i
            sb, db = int(c0.table[b, src // 16]), int(c0.table[b, dst // 16])
            for p, w in zip(pools, want):
                if fmt == 0:
                    w[:, db, :, dst % 16] = p[:, sb, :, src % 16]
                else:
                    u, x = plain.views(p, dim, fmt), plain.views(w, dim, fmt)
                    for a, e in zip(u, x):
                        a, e = (y.view(torch.uint8) if y.element_size() == 1 else y.view(torch.int32) for y in (a, e))
                        e[:, db, :, dst % 16] = a[:, sb, :, src % 16]
    gpu = [dev(p) for p in pools]
    out = [torch.full((total,), 99, dtype=torch.int32, device="cuda")] + [torch.full((len(rows),), 99, dtype=torch.int32, device="cuda") for _ in range(3)]
    head = (dev(draft), dev(target), dev(parent), dev(start), dev(np.array(ctx, np.int32)), len(rows), max(rows))
    tail = (layers, dev(c0.table), c0.stride, kvh, dim, *out, 0)
    if fmt == 0:
        ops.tree_commit(*head, *gpu, gpu[0].stride(0), *tail)
    else:
        ops.tree_commit_q8(*head, *gpu, gpu[0].stride(0), *tail)
    for x, e in zip(out, (want_path, want_count, want_next, want_len)):
        assert np.array_equal(x.cpu().numpy(), np.array(e, np.int32))
    for x, e in zip(gpu, want):
        assert torch.equal(x.cpu(), e)
    if accept == 1.0 and max(rows) > 30:
        assert max(want_count) > 8  # paths long enough to move rows through several batches


# ------------------------------------------------------------------ refusals


def test_refusals(ops):
    f, i, u = torch.zeros(4096, device="cuda"), torch.zeros(64, dtype=torch.int32, device="cuda"), torch.zeros(8192, dtype=torch.uint8, device="cuda")
    bad = []

    def refuse(call, args, at, value):
        args = list(args)
        args[at] = value
        with pytest.raises(ValueError):
            call(*args)
        bad.append(at)

    write = [f, f, 0, 128, u, 1, i, 1, i, i, 1, 1, 2, 64, 0]
    for at, value in [(0, None), (1, None), (2, 2), (3, 127), (3, 130), (4, None), (5, 0), (5, 3), (6, None), (7, 0),
                      (8, None), (9, None), (10, -1), (11, -1), (12, 0), (13, 96), (0, f.data_ptr() + 4), (4, u.data_ptr() + 8)]:
        refuse(ops.kv_quant_write, write, at, value)
    read = [u, 1, i, 1, i, i, 1, 1, 2, 64, f, f, 0, 128, 0]
    for at, value in [(0, None), (1, 0), (3, 0), (6, -1), (7, -1), (8, 0), (9, 32), (10, None), (12, 7), (13, 64), (13, 129)]:
        refuse(ops.kv_quant_read, read, at, value)
    attn = [f, 0, 256, f, f, i, 1, i, i, i, 1, 1, 1, 1, 10, 4, 2, 64, 0.125, f, 256, 0]
    for at, value in [(0, None), (1, 5), (2, 255), (2, 258), (3, None), (4, None), (5, None), (6, 0), (7, None), (8, None),
                      (10, 0), (11, -1), (12, -1), (13, 2), (13, -1), (14, -1), (15, 3), (16, 0), (17, 80), (19, None),
                      (20, 128), (19, f.data_ptr() + 8)]:
        refuse(ops.tree_attention, attn, at, value)
    attn8 = attn[:3] + [u, 1] + attn[5:]
    for at, value in [(3, None), (4, 0), (4, 3), (3, u.data_ptr() + 4)]:
        refuse(ops.tree_attention_q8, attn8, at, value)
    com = [i, i, i, i, i, 1, 1, f, f, 1024, 1, i, 1, 1, 64, i, i, i, torch.zeros_like(i), 0]
    for at, value in [(0, None), (1, None), (2, None), (3, None), (4, None), (5, -1), (6, 2049), (6, -1), (7, None), (8, None),
                      (10, 0), (11, None), (12, 0), (13, 0), (14, 63), (15, None), (16, None), (17, None), (18, i)]:
        refuse(ops.tree_commit, com, at, value)
    com8 = com[:7] + [u, 2176] + com[10:]
    for at, value in [(7, None), (7, u.data_ptr() + 4)]:
        refuse(ops.tree_commit_q8, com8, at, value)
    refuse(ops.tree_commit_q8, com8[:9] + [2] + com8[10:], 8, 0)  # two layers need a stride
    assert "tree_commit" in ops.last_error()
    # nothing to do is no error, and touches nothing
    ops.kv_quant_write(None, None, 0, 128, None, 1, None, 1, None, None, 0, 0, 2, 64, 0)
    ops.tree_attention(None, 0, 256, None, None, None, 1, None, None, None, 0, 0, 0, 0, 0, 4, 2, 64, 0.125, None, 256, 0)
    ops.tree_commit(None, None, None, None, None, 0, 0, None, None, 0, 1, None, 1, 1, 64, None, None, None, None, 0)
    ops.ops_sync(0)
    assert len(bad) > 60
