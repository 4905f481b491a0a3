"""GPU tests of pages and slots, of norm and rotation of heads, and of the 4-bit paged cache with attention and commit over
it, through libopworks_ops.so, against the plain forms of tests/q4_plain.py and tests/tree_cache_plain.py.

Tolerances. Pages, slots, codes, scales and rows read back are whole numbers, or one exact product: they must be equal.

Norm and rotation: the sum of squares, its root and the weight cost 12 roundings of 2^-24 relative at most (D / 32 terms a
lane and 5 exchanges, halved by the root; rsqrt 2^-22.9), the angle's cos and sin are 2^-22 off, and the rotation rounds
three times: 2^-20 of |a| + |b| in all. bf16 rounds the result: 2^-8 (half a step is 2^-9; cos and sin signs may cancel).

Attention: K, V are exact in fp16, queries to 2^-22 (two terms) or exactly; a score is a sum of D products in at most 2 D /
16 steps, each cutting off 2^-23 of what it holds: 2^-18 sum|q k| scale. A softmax weight is then off by twice that, and the
output by 2^-17 mass max|v|. The sums over the keys are cut off once per 16 keys, or rounded once per 32: (keys / 16 + 16)
2^-23 max|v|. bf16 rows add the output's rounding, 2^-8 |o|, and that of the weights to 11 bits, 2^-10 max|v|."""

import math

import numpy as np
import pytest

import q4_plain
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


def ints(a):
    return dev(np.array(a, np.int32))


def starts(rows):
    return np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)


# ------------------------------------------------------------------ pages


def run_take(ops, lens, counts, stride, spare=5, pad=0, count=None, table=None, complete=False, seed=0, in_place=False, start=None):
    rng = np.random.default_rng(seed)
    lens = np.array(lens, np.int64)
    start = starts(counts) if start is None else np.array(start, np.int32)
    batch, rows = len(lens), int(start[-1]) + pad
    if table is None:
        table = rng.integers(0, 100000, (batch, stride)).astype(np.int32)
    size = int(np.maximum(0, -(-np.maximum(0, lens + np.diff(start)) // 16)).sum()) + spare
    free = None if complete else rng.permutation(200000)[:size].astype(np.int32)
    count = size if count is None else count
    want = q4_plain.take(lens.tolist(), start.tolist(), rows, table, free, count)
    t, pos, slots = dev(table), torch.full((rows + 3,), 77, dtype=torch.int32, device="cuda"), torch.full((rows + 3,), 77, dtype=torch.int64, device="cuda")
    cnt, status = ints([count]), ints([99])
    left = cnt if in_place else ints([98])
    f = None if complete else dev(free)
    ops.page_take(dev(lens.astype(np.int32)), dev(start), batch, rows, t, stride, f, None if complete else cnt, pos, slots,
                  None if complete else left, status, 0)
    assert status.item() == want[0]
    assert torch.equal(t.cpu(), torch.from_numpy(want[1]))
    assert slots[:rows].tolist() == want[3].tolist() and slots[rows:].eq(77).all() and pos[rows:].eq(77).all()
    if want[0] == 0:
        assert pos[:rows].tolist() == want[2].tolist()
    if not complete:
        assert left.item() == want[4] and torch.equal(f.cpu(), torch.from_numpy(free))
    return want[0]


@pytest.mark.parametrize("lens,counts,stride,pad", [
    ([0], [1], 4, 0), ([0], [0], 1, 0), ([15], [1], 1, 0), ([16], [1], 2, 3), ([5], [0], 2, 2), ([31, 32, 33], [1, 1, 1], 9, 0),
    ([0, 100, 16, 7], [33, 0, 16, 500], 40, 5), ([2180 + i for i in range(32)], [1] * 32, 200, 0), ([3] * 70, list(range(70)), 9, 0)])
@pytest.mark.parametrize("in_place", [False, True])
def test_page_take(ops, lens, counts, stride, pad, in_place):
    assert run_take(ops, lens, counts, stride, pad=pad, in_place=in_place) == 0


@pytest.mark.parametrize("batch,most", [(513, 9), (600, 200), (1500, 3), (48, 2048), (5000, 4), (4096, 2)])
def test_page_take_of_large_batches(ops, batch, most):
    rng = np.random.default_rng(batch)
    lens, counts = rng.integers(0, 500, batch), rng.integers(0, most, batch)
    assert run_take(ops, lens, counts, (500 + most) // 16 + 1, pad=int(rng.integers(0, 3)), in_place=True) == 0


def test_page_take_of_the_last_page_and_of_one_too_many(ops):
    assert run_take(ops, [0, 16], [16, 33], 6, count=4) == 0  # 1 + 3
    assert run_take(ops, [0, 16], [16, 33], 6, count=3) == 1
    assert run_take(ops, [0] * 700, [40] * 700, 3, count=2000, in_place=True) == 100
    assert run_take(ops, [0], [5], 3, count=0) == 1 and run_take(ops, [3], [5], 3, count=0) == 0 and run_take(ops, [0], [5], 3, count=-4) == 1


def test_page_take_refuses_lengths_on_the_device(ops):
    assert run_take(ops, [0, 60], [1, 5], 4) == -1  # the second sequence is longer than its table row
    assert run_take(ops, [0, -1], [1, 5], 4) == -1
    assert run_take(ops, [0, 2**31 - 4], [1, 5], 4) == -1
    assert run_take(ops, [0, 3, 3], [1, 5, 5], 4, start=[0, 5, 3, 9]) == -1
    assert run_take(ops, [64, 60], [0, 4], 4) == 0


def test_slots_of_a_complete_table(ops):
    assert run_take(ops, [0, 37, 5], [40, 1, 0], 9, complete=True, pad=2) == 0
    assert run_take(ops, [0, 140], [40, 5], 9, complete=True) == -1


def test_rows_before_the_first_sequence_have_no_slot(ops):
    pos, slots, status = ints([7] * 6), torch.full((6,), 7, device="cuda"), ints([7])
    ops.page_take(ints([3]), ints([2, 5]), 1, 6, ints([[9, 4]]), 2, None, None, pos, slots, None, status, 0)
    assert status.item() == 0 and slots.tolist() == [-1, -1, 147, 148, 149, -1] and pos.tolist() == [0, 0, 3, 4, 5, 0]


def test_block_ids_whose_slots_pass_32_bits(ops):
    pos, slots, status = ints([0]), torch.zeros(1, dtype=torch.int64, device="cuda"), ints([7])
    ops.page_take(ints([16]), ints([0, 1]), 1, 1, ints([[1, 2]]), 2, ints([2**31 - 1]), ints([1]), pos, slots, ints([0]), status, 0)
    assert slots.item() == (2**31 - 1) * 16


@pytest.mark.parametrize("old,new", [([0], [0]), ([16], [15]), ([17, 16, 40], [0, 16, 33]), ([100] * 40, list(range(5, 205, 5))),
                                     (list(range(700)), [0] * 700), ([17] * 5000, [i % 18 for i in range(5000)])])
@pytest.mark.parametrize("in_place", [False, True])
def test_page_give(ops, old, new, in_place):
    rng = np.random.default_rng(len(old))
    table = rng.integers(0, 1000, (len(old), 60)).astype(np.int32)
    free = rng.integers(0, 1000, 40000).astype(np.int32)
    want, count = q4_plain.give(old, new, table, free, 17)
    f, cnt, status = dev(free), ints([17]), ints([9])
    left = cnt if in_place else ints([9])
    ops.page_give(ints(old), ints(new), len(old), dev(table), 60, f, 40000, cnt, left, status, 0)
    assert status.item() == 0 and left.item() == count and torch.equal(f.cpu(), torch.from_numpy(want))
    # a stack that has room for one id less is left as it was
    f, cnt, left = dev(free), ints([17]), ints([9])
    ops.page_give(ints(old), ints(new), len(old), dev(table), 60, f, count - 1, cnt, left, status, 0)
    if count > 17:
        assert status.item() == -1 and left.item() == 17 and torch.equal(f.cpu(), torch.from_numpy(free))


@pytest.mark.parametrize("old,new", [([5, -1], [0, 0]), ([5, 5], [0, -2]), ([5, 17], [0, 0])])
def test_page_give_refuses_lengths_on_the_device(ops, old, new):
    f, cnt, left, status = ints([1, 2, 3, 4, 5]), ints([1]), ints([9]), ints([9])
    ops.page_give(ints(old), ints(new), 2, ints([[7], [8]]), 1, f, 5, cnt, left, status, 0)
    assert status.item() == -1 and left.item() == 1 and f.tolist() == [1, 2, 3, 4, 5]


def test_no_sequences(ops):
    pos, slots, status, left = ints([7, 7]), torch.full((2,), 7, device="cuda"), ints([7]), ints([7])
    ops.page_take(None, ints([0]), 0, 2, None, 4, ints([1]), ints([1]), pos, slots, left, status, 0)
    assert slots.tolist() == [-1, -1] and status.item() == 0 and left.item() == 1
    ops.page_give(None, None, 0, None, 4, ints([1]), 1, ints([1]), left, status, 0)
    assert status.item() == 0 and left.item() == 1


# ------------------------------------------------------------------ norm and rotation


def norm_case(ops, kind, dim, rot, rows, qh, kvh, weights=(True, True), pad=0, in_place=False, far=5000, seed=0, gain=1.0):
    g = torch.Generator().manual_seed(seed)
    width = (qh + kvh) * dim + pad
    x = (torch.randn(rows, width, generator=g) * gain).to(TYPES[kind])
    w = [torch.rand(dim, generator=g) + 0.5 if on else None for on in weights]
    pos = torch.randint(0, far, (rows,), generator=g, dtype=torch.int32)
    inv = (10000.0 ** (-torch.arange(0, max(rot, 2), 2) / max(rot, 2))).float()
    d = dev(x)
    out = d if in_place else torch.full((rows, width), 777.0, dtype=TYPES[kind], device="cuda")
    part = lambda t, at: t.view(-1)[at:]  # noqa: E731
    dw = [None if v is None else dev(v) for v in w]
    ops.qk_norm_rope(part(d, 0), width, part(d, qh * dim), width, kind, dw[0], dw[1], 1e-5, dev(pos), dev(inv), rot, rows, qh, kvh, dim,
                     part(out, 0), width, part(out, qh * dim), width, 0)
    got = out.cpu()
    if pad:
        assert torch.equal(got[:, width - pad :], x[:, width - pad :] if in_place else torch.full((rows, pad), 777.0, dtype=TYPES[kind]))
    at = 0
    for heads, weight in ((qh, w[0]), (kvh, w[1])):
        one = x[:, at : at + heads * dim].view(rows, heads, dim)
        want = q4_plain.norm_rope(one, weight, 1e-5, pos, inv, rot)
        plainly = q4_plain.norm_rope(one, weight, 1e-5, pos, inv, 0).abs()
        size = plainly.clone()
        if rot:
            both = plainly[..., : rot // 2] + plainly[..., rot // 2 : rot]
            size[..., :rot] = torch.cat([both, both], -1)
        tol = 2.0**-20 * size + (2.0**-8 * want.abs() if kind else 0) + 1e-38
        y = got[:, at : at + heads * dim].double().view(rows, heads, dim)
        assert torch.isfinite(y).all() and ((y - want).abs() <= tol).all(), ((y - want).abs() - tol).max()
        at += heads * dim


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("dim,rot", [(32, 32), (64, 64), (64, 32), (64, 0), (128, 128), (128, 48), (256, 256), (256, 64)])
@pytest.mark.parametrize("rows,qh,kvh,pad", [(1, 1, 1, 0), (5, 32, 8, 0), (33, 7, 1, 16), (2, 96, 3, 8), (3, 0, 2, 0), (3, 2, 0, 8), (2500, 5, 2, 0)])
def test_norm_and_rotation(ops, kind, dim, rot, rows, qh, kvh, pad):
    norm_case(ops, kind, dim, rot, rows, qh, kvh, pad=pad, seed=dim + rows)


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("weights", [(False, True), (True, False), (False, False)])
def test_sides_without_a_norm_and_in_place(ops, kind, weights):
    norm_case(ops, kind, 64, 64, 9, 12, 3, weights, in_place=True)
    norm_case(ops, kind, 128, 64, 9, 12, 3, weights, pad=8, in_place=True)


@pytest.mark.parametrize("kind", [0, 1])
def test_far_positions_and_large_and_small_values(ops, kind):
    norm_case(ops, kind, 128, 128, 50, 4, 2, far=2**31 - 1)
    norm_case(ops, kind, 64, 64, 20, 4, 2, gain=1e12)
    norm_case(ops, kind, 64, 64, 20, 4, 2, gain=1e-12)


def test_norm_rows_of_zeros_and_of_nan(ops):
    x = torch.zeros(2, 2, 64, device="cuda")
    x[1, 0, 3] = float("nan")
    out, w = torch.full_like(x, 5.0), torch.ones(64, device="cuda")
    ops.qk_norm_rope(x, 128, x[:, 1], 128, 0, w, w, 1e-5, ints([0, 9]), torch.ones(32, device="cuda"), 64, 2, 1, 1, 64, out, 128, out[:, 1], 128, 0)
    assert (out[0] == 0).all() and out[1, 0].isnan().all() and (out[1, 1] == 0).all()


# ------------------------------------------------------------------ rows


def rows_case(ops, x_k, x_v, kvh, dim, slots, blocks, seed=0, pad=(0, 0)):
    """Stores rows at their slots over a pool of junk; every byte of it must be right. Then fetches them in both types."""
    total = len(slots)
    kind = 0 if x_k.dtype == torch.float32 else 1
    g = torch.Generator().manual_seed(seed)
    before = torch.randint(0, 256, (blocks, kvh, 18 * dim), generator=g, dtype=torch.uint8)
    pool, sl = dev(before), dev(np.array(slots, np.int64))
    wide = [torch.full((total, kvh * dim + p), 3.0, dtype=x.dtype) for x, p in zip((x_k, x_v), pad)]
    for w, x in zip(wide, (x_k, x_v)):
        w[:, : kvh * dim] = x.reshape(total, -1)
    dk, dv = (dev(w) for w in wide)
    ops.kv4_write(dk, dk.stride(0), dv, dv.stride(0), kind, pool, blocks, sl, total, kvh, dim, 0)
    want = before.clone()
    kc, vc, ks, vs = q4_plain.views(want, dim)
    kept = [i for i, s in enumerate(slots) if 0 <= s < blocks * 16]
    for i in kept:
        for codes, scales, x in ((kc, ks, x_k), (vc, vs, x_v)):
            c, s = q4_plain.quantise(x[i].reshape(kvh, dim))
            codes[slots[i] // 16, :, :, slots[i] % 16] = c
            scales[slots[i] // 16, :, :, slots[i] % 16] = s
    got = pool.cpu()
    gv, wv = q4_plain.views(got, dim), q4_plain.views(want, dim)
    for a, b in zip(gv[:2], wv[:2]):
        assert torch.equal(a, b)
    for a, b in zip(gv[2:], wv[2:]):  # NaN by any of its patterns, where a row was stored
        same = a.view(torch.int16) == b.view(torch.int16)
        assert (same | (a.isnan() & b.isnan())).all()
    values = [q4_plain.dequantise(c, s) for c, s in ((kc.transpose(2, 3), ks.transpose(2, 3)), (vc.transpose(2, 3), vs.transpose(2, 3)))]
    for out_kind in (0, 1):
        back = [torch.full((total, kvh * dim + p), 5.0, dtype=TYPES[out_kind], device="cuda") for p in pad[::-1]]
        ops.kv4_read(pool, blocks, sl, total, kvh, dim, back[0], back[0].stride(0), back[1], back[1].stride(0), out_kind, 0)
        for t, v in zip(back, values):
            t = t.cpu()
            assert (t[:, kvh * dim :] == 5).all()
            for i in range(total):
                row = t[i, : kvh * dim].float()
                if i in kept:
                    e = v[slots[i] // 16, :, slots[i] % 16].flatten().float()
                    assert torch.equal(row.isnan(), e.isnan()) and torch.equal(row.nan_to_num(9), e.nan_to_num(9))  # a bf16 number, too
                else:
                    assert (row == 5).all()
    return values


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kvh,total,pad", [(1, 1, (0, 0)), (8, 40, (0, 64)), (3, 9, (8, 0)), (5, 33, (0, 0)), (16, 3, (16, 16))])
def test_store_and_fetch(ops, kind, dim, kvh, total, pad):
    g = torch.Generator().manual_seed(total + dim)
    x = [(torch.randn(total, kvh, dim, generator=g) * torch.exp(torch.randn(kvh, dim, generator=g))).to(TYPES[kind]) for _ in range(2)]
    blocks = total // 16 + 3
    slots = np.random.default_rng(total).permutation(blocks * 16)[:total].tolist()
    for i in range(0, total, 7):  # rows without a slot
        if total > 1:
            slots[i] = [-1, blocks * 16, 2**40, -(2**40)][i // 7 % 4]
    values = rows_case(ops, *x, kvh, dim, slots, blocks, pad=pad)
    for y, v in zip(x, values):  # off by half a step at most
        for i, s in enumerate(slots):
            if 0 <= s < blocks * 16:
                step = y[i].double().unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True) / 7 * (1 + 2**-5)
                err = (v[s // 16, :, s % 16] - y[i].double()).abs().unflatten(-1, (-1, 32))
                assert (err <= step / 2 * (1 + 2**-20)).all()


@pytest.mark.parametrize("kind", [0, 1])
def test_store_of_ties_and_of_edge_values(ops, kind):
    """Halves of a step and what is next to them; zeros, denormals, one spike, the largest, too large, infinities, NaN."""
    dim, kvh = 64, 1
    rows = []
    for s in (1.0, 1.0625, 0.0078125 * 1.9375, 7936.0, 2.0**-20, 2.0**-24):
        halves = torch.tensor([i + 0.5 for i in range(-7, 7)] + [0.0, -0.0, 7.0]) * s
        x = torch.cat([halves, torch.nextafter(halves[:14], torch.tensor(1e9)), torch.tensor([7.0 * s])])
        y = torch.cat([torch.nextafter(halves[:14], torch.tensor(-1e9)), torch.tensor([-7.0 * s]), halves])
        rows.append(torch.cat([x, y]))
    base = torch.randn(20, dim, generator=torch.Generator().manual_seed(4))
    base[0] = 0
    base[1] *= 1e-42
    base[2, 5], base[3, 7], base[4, 40], base[5, 9] = 3e4, float("inf"), float("nan"), -float("inf")
    base[6] = -0.0
    base[7] = 55552.0 * torch.sign(base[7])
    base[8] = 56000.0 * torch.sign(base[8])
    base[9] = 57600.0 * torch.sign(base[9])
    base[10] = 3e38 * torch.sign(base[10])
    base[11] = 2.0**-24
    base[12] = base[12] * 2.0**-21
    base[13] = base[13] * 3e-8
    base[14, :32] = 0
    for i in range(15, 20):
        base[i] *= 10.0 ** (i - 18)
    x = torch.cat([torch.stack(rows), base]).to(TYPES[kind])[:, None]
    values = rows_case(ops, x, x.flip(0), kvh, dim, list(range(len(x))), 3)
    k = values[0][:, 0].flatten(0, 1)[len(rows) :]
    assert k[3, :32].isnan().all() and k[3, 32:].isfinite().all() and k[4, 32:].isnan().all() and k[5, :32].isnan().all()
    assert k[7].isfinite().all() and k[9].isnan().all() and k[10].isnan().all()


def test_store_of_many_random_rows_of_every_size(ops):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(4000, 4, 64, generator=g) * torch.exp2(torch.randint(-26, 11, (4000, 4, 1), generator=g).float())
    for kind in (0, 1):
        rows_case(ops, x.to(TYPES[kind]), x.flip(0).to(TYPES[kind]), 4, 64, list(range(4000)), 250)


# ------------------------------------------------------------------ attention


def attention_case(ops, kind, dim, kvh, rep, ctx, rows, trees="tree", q_pad=0, seed=0, spoil=(), sees=None, stream=None, scale=None,
                   cache=None, q=None, max_rows=None, max_ctx=None, finite=True):
    rng = np.random.default_rng(seed)
    qh, total, start = kvh * rep, sum(rows), starts(rows)
    if cache is None:
        cache = q4_plain.Cache4([c + n for c, n in zip(ctx, rows)], kvh, dim, seed + 1)
    if sees is None:
        sees = [plain.tree(rng, n, trees)[1] for n in rows]
    for b, j in spoil:
        cache.spoil(b, ctx[b] + j)
    if q is None:
        q = torch.randn(total, qh * dim + q_pad, generator=torch.Generator().manual_seed(seed + 2))
    q = q.to(TYPES[kind])
    words = max(1, -(-max(rows) // 32))
    mask = None if trees == "chain" else dev(np.concatenate([plain.pack_mask(s, words) for s in sees]))
    scale = 1 / math.sqrt(dim) if scale is None else scale
    dq, out = dev(q), torch.full((total + 1, qh * dim + q_pad), 777.0, dtype=TYPES[kind], device="cuda")
    pool = dev(cache.pool)
    args = (dev(cache.table), cache.stride, ints(ctx), dev(start), mask, words, len(rows), total, max(rows) if max_rows is None else max_rows,
            max(ctx) if max_ctx is None else max_ctx, qh, kvh, dim, scale, out, qh * dim + q_pad)
    torch.cuda.synchronize()
    ops.tree_attention_q4(dq, kind, qh * dim + q_pad, pool, *args, 0 if stream is None else stream.cuda_stream)
    ops.ops_sync(0 if stream is None else stream.cuda_stream)
    got = out.cpu()
    assert (got[:, qh * dim :] == 777.0).all() and (got[total] == 777.0).all()
    got = got[:total, : qh * dim].double().view(total, qh, dim)
    want, mass, top = plain.attention(cache, q[:, : qh * dim].reshape(total, qh, dim), ctx, start, sees, scale)
    keys = max(c + n for c, n in zip(ctx, rows))
    tol = 2.0**-17 * mass * top + (keys / 16 + 16) * 2.0**-23 * top
    tol = tol[..., None].expand_as(want)
    if kind == 1:
        tol = tol + 2.0**-8 * want.abs() + 2.0**-10 * top[..., None]
    if finite:
        assert torch.isfinite(got).all()
    err = (got - want).abs()
    ok = torch.isfinite(want).all(-1, keepdim=True).expand_as(want)
    assert got[~ok].isnan().all()  # a row that sees a NaN is NaN in all dims
    assert (err <= tol)[ok].all(), f"error {err[ok].max():.3g}, over by {(err - tol)[ok].max():.3g}"
    return got


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kvh,rep,ctx,rows", [
    (1, 1, [0], [1]),                                  # nothing but itself
    (8, 4, [511], [1]),                                # a plain decode step
    (2, 4, [15, 16, 17, 0], [1, 5, 2, 31]),            # pages that end inside a tree
    (2, 7, [100, 3], [7, 33]),                         # odd group, two mask words
    (1, 16, [31, 64, 200], [26, 0, 8]),                # an empty sequence among others
    (3, 3, [1000], [64]),
    (1, 8, [40, 700], [100, 3]),
    (2, 8, [31, 32, 33], [1, 1, 1]),                   # 8 rows: a tile of both terms
    (2, 9, [31, 32, 33], [1, 1, 1])])                  # 9: a tile of 16
def test_attention(ops, kind, dim, kvh, rep, ctx, rows):
    attention_case(ops, kind, dim, kvh, rep, ctx, rows, seed=dim + rep)


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("dim,kvh,rep,ctx,rows", [(64, 1, 4, [5000], [1]), (64, 2, 4, [0, 30], [150, 17]), (128, 1, 2, [2050, 1], [40, 1]),
                                                  (64, 8, 4, [3000, 10], [5, 5]), (128, 2, 4, [0], [300]), (64, 1, 3, [100, 7], [257, 129])])
def test_chains_without_a_mask(ops, kind, dim, kvh, rep, ctx, rows):
    attention_case(ops, kind, dim, kvh, rep, ctx, rows, trees="chain", seed=3)


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kvh,rep,ctx,rows", [(1, 4, [5003], [11]), (2, 8, [2600, 4100], [24, 3]), (1, 2, [17000], [2]), (1, 1, [1, 9000], [1, 1])])
def test_long_contexts(ops, kind, dim, kvh, rep, ctx, rows):
    """The ring many times over, on few CTAs and on several that are joined."""
    attention_case(ops, kind, dim, kvh, rep, ctx, rows, seed=5)


@pytest.mark.parametrize("kind", [0, 1])
def test_many_sequences(ops, kind):
    """More sequences than fit at once, longest first; more than a block has threads; more than are put in order."""
    rng = np.random.default_rng(3)
    for batch in (70, 300, 1100):
        attention_case(ops, kind, 64, 8, 2, rng.integers(0, 120, batch).tolist(), [1] * batch, trees="chain", seed=batch)


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [2, 3, 40, 80])
def test_rows_that_see_nothing_are_zero(ops, kind, dim, n):
    rng = np.random.default_rng(1)
    sees = [rng.random((n, n)) < 0.3, rng.random((2, 2)) < 2]
    sees[0][0] = sees[0][n - 1] = False
    got = attention_case(ops, kind, dim, 2, 4, [0, 9], [n, 2], sees=sees, seed=7)
    assert (got[0] == 0).all() and (got[n - 1] == 0).all()


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [2, 6, 50, 90])
def test_masked_nans_have_no_influence_and_seen_ones_spoil_the_row(ops, kind, dim, n):
    rng = np.random.default_rng(2)
    sees = [plain.tree(rng, n)[1], plain.tree(rng, n)[1]]
    bad = [(0, 1), (0, n - 1), (1, n // 2)]
    for b, j in bad:
        sees[b][:, j] = False
    attention_case(ops, kind, dim, 2, 4, [30, 0], [n, n], sees=sees, spoil=bad, seed=8)
    sees[0][n - 1, n - 1] = True  # one row sees its own
    got = attention_case(ops, kind, dim, 2, 4, [30, 0], [n, n], sees=sees, spoil=bad, seed=8, finite=False)
    assert got[n - 1].isnan().all() and torch.isfinite(torch.cat([got[: n - 1], got[n:]])).all()


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [1, 9, 70])
@pytest.mark.parametrize("at", [3, 199])
def test_a_nan_in_the_context_spoils_every_row(ops, kind, dim, n, at):
    cache = q4_plain.Cache4([200 + n], 1, dim, 4)
    cache.spoil(0, at)
    got = attention_case(ops, kind, dim, 1, 4, [200], [n], cache=cache, finite=False)
    assert got.isnan().all()


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("n", [1, 9, 70])
@pytest.mark.parametrize("which", [2, 3])
@pytest.mark.parametrize("at", [3, 199])
def test_a_nan_scale_of_one_group_spoils_whole_rows(ops, kind, n, which, at):
    cache = q4_plain.Cache4([200 + n], 1, 128, 4)
    q4_plain.views(cache.pool, 128)[which][int(cache.table[0, at // 16]), 0, 2, at % 16] = float("nan")
    assert attention_case(ops, kind, 128, 1, 4, [200], [n], cache=cache, finite=False).isnan().all()


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("n", [1, 40])
def test_query_rows_with_a_nan_or_an_infinity(ops, kind, n):
    q = torch.randn(n, 4 * 64, generator=torch.Generator().manual_seed(2))
    q[0, 70], q[n - 1, 0] = float("inf"), float("nan")
    got = attention_case(ops, kind, 64, 1, 4, [100], [n], q=q, finite=False)
    assert got[0, 1].isnan().all() and got[n - 1, 0].isnan().all()
    clean = torch.ones(n, 4, dtype=torch.bool)
    clean[0, 1] = clean[n - 1, 0] = False
    assert torch.isfinite(got[clean]).all()


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("dim", [64, 128])
def test_strided_rows_and_another_stream(ops, kind, dim):
    attention_case(ops, kind, dim, 2, 4, [77, 5], [9, 3], q_pad=64, seed=9)
    attention_case(ops, kind, dim, 2, 4, [77, 5], [9, 80], q_pad=8, seed=9)
    attention_case(ops, kind, dim, 2, 4, [77, 5], [9, 3], seed=10, stream=torch.cuda.Stream())


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("n", [2, 8, 70])
@pytest.mark.parametrize("scale", [0.0, 4.0, -0.5, 300.0])
def test_flat_and_peaked_softmax(ops, kind, n, scale):
    attention_case(ops, kind, 64, 1, 4, [600], [n], seed=11, scale=scale)


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("n", [1, 70])
@pytest.mark.parametrize("size", [1e-38, 1e-20, 1e20, 3e38])
def test_queries_of_any_size_give_finite_rows(ops, kind, n, size):
    """Scores in one place at scale 1 / size: the same as those of plain queries. At scale 1: finite, the largest score's row
    where the others are far below."""
    q = torch.randn(n, 4 * 64, generator=torch.Generator().manual_seed(5)).clamp(-1.1, 1.1) * size
    attention_case(ops, kind, 64, 1, 4, [300], [n], q=q, scale=0.125 / size if size > 1e-30 else 1e37)
    cache = q4_plain.Cache4([300 + n], 1, 64, 1)
    out = torch.empty(n, 256, dtype=TYPES[kind], device="cuda")
    ops.tree_attention_q4(dev(q.to(TYPES[kind])), kind, 256, dev(cache.pool), dev(cache.table), cache.stride, ints([300]), ints([0, n]), None, 0, 1,
                          n, n, 300, 4, 1, 64, 3e38, out, 256, 0)
    assert out.isfinite().all()


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("n", [1, 8, 70])
@pytest.mark.parametrize("gain", [1e-6, 1e-3, 1e3, 1e4])
def test_rows_of_any_size_that_the_cache_holds(ops, kind, n, gain):
    """At 1e4 some groups are past what it holds: the heads that see them get NaN."""
    cache = q4_plain.Cache4([400 + n], 2, 64, 9, gain=gain)
    got = attention_case(ops, kind, 64, 2, 4, [400], [n], cache=cache, scale=0.125 / gain, finite=gain < 1e4)
    spoilt = [any(x[:, h].isnan().any() for x in cache.rows(0)) for h in range(2)]
    for h in range(2):
        assert got[:, 4 * h : 4 * h + 4].isnan().all() if spoilt[h] else got[:, 4 * h : 4 * h + 4].isfinite().all()
    assert any(spoilt) == (gain >= 1e4)


def test_one_far_key_does_not_blur_the_others(ops):
    """A masked node and a context key of huge V rows: the first takes nothing, the second only what it weighs."""
    for kind in (0, 1):
        for n in (3, 80):
            cache = q4_plain.Cache4([64 + n], 1, 64, 3)
            _, vc, _, vs = q4_plain.views(cache.pool, 64)
            vs[int(cache.table[0, (64 + n - 1) // 16]), :, :, (64 + n - 1) % 16] = 7936.0
            sees = [plain.tree(np.random.default_rng(0), n)[1]]
            sees[0][:, n - 1] = False
            attention_case(ops, kind, 64, 1, 4, [64], [n], cache=cache, sees=sees)


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("n", [1, 26, 100])
def test_two_calls_give_the_same_bits(ops, kind, n):
    a = attention_case(ops, kind, 64, 2, 4, [900, 40], [n, 8], seed=12)
    assert torch.equal(a, attention_case(ops, kind, 64, 2, 4, [900, 40], [n, 8], seed=12))


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("n", [1, 40])
def test_a_scale_that_is_no_number_gives_nan(ops, kind, n):
    cache = q4_plain.Cache4([90 + n], 1, 64, 3)
    q = torch.randn(n, 256, device="cuda").to(TYPES[kind])
    out = torch.zeros(n, 256, dtype=TYPES[kind], device="cuda")
    ops.tree_attention_q4(q, kind, 256, dev(cache.pool), dev(cache.table), cache.stride, ints([90]), ints([0, n]), None, 0, 1, n, n, 90, 4, 1, 64, float("nan"), out, 256, 0)
    assert out.isnan().all()


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("n", [1, 6, 60])
def test_calls_on_two_streams_at_once(ops, kind, n):
    """Many calls on two streams, of their own inputs over one pool: each gives what it gives alone."""
    cache = q4_plain.Cache4([700 + n, 300 + n], 2, 64, 3)
    pool, table, lens, start = dev(cache.pool), dev(cache.table), ints([700, 300]), ints([0, n, 2 * n])
    q = [torch.randn(2 * n, 512, generator=torch.Generator().manual_seed(i)).to(TYPES[kind]).cuda() for i in range(2)]
    call = lambda x, out, s: ops.tree_attention_q4(x, kind, 512, pool, table, cache.stride, lens, start, None, 0, 2, 2 * n, n, 700, 8, 2, 64, 0.125, out, 512, s)  # noqa: E731
    alone = [torch.empty_like(x) for x in q]
    for x, out in zip(q, alone):
        call(x, out, 0)
    both = [[torch.empty_like(x) for _ in range(20)] for x in q]
    streams = [torch.cuda.Stream() for _ in q]
    torch.cuda.synchronize()
    for i in range(20):
        for x, outs, s in zip(q, both, streams):
            call(x, outs[i], s.cuda_stream)
    torch.cuda.synchronize()
    for a, outs in zip(alone, both):
        assert all(torch.equal(a, out) for out in outs)


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("n", [1, 40])
def test_bounds_that_are_larger_than_the_lengths(ops, kind, n):
    """Plans for more rows and a longer context than there are: padded steps of a captured graph."""
    attention_case(ops, kind, 64, 2, 4, [50, 700], [n, 3], max_ctx=30000, seed=2)
    attention_case(ops, kind, 128, 2, 4, [50, 0], [n, n], max_ctx=0, seed=2)


@pytest.mark.parametrize("kind", [0, 1])
def test_rows_past_the_last_sequence_are_left_as_they_were(ops, kind):
    cache = q4_plain.Cache4([40, 30], 1, 64, 3)
    q = torch.randn(9, 256, device="cuda").to(TYPES[kind])
    out = torch.full((9, 256), 777.0, dtype=TYPES[kind], device="cuda")
    ops.tree_attention_q4(q, kind, 256, dev(cache.pool), dev(cache.table), cache.stride, ints([37, 28]), ints([0, 3, 5]), None, 0, 2, 9, 9, 100, 4, 1, 64,
                          0.125, out, 256, 0)
    assert (out[5:] == 777).all() and (out[:5] != 777).all()


@pytest.mark.parametrize("dim", [64, 128])
def test_blocks_whose_offsets_pass_32_bits(ops, dim):
    """Pages at the far end of a pool of over 2^32 bytes: stored, fetched, attended, kept."""
    rep, ctx, rows, size = 4, 20, 90, 18 * dim
    small = q4_plain.Cache4([ctx + rows], 1, dim, 6)
    pages = -(-(ctx + rows) // 16)
    blocks = 2**32 // size + 100
    far = blocks - 1 - np.arange(small.stride)
    table = dev(far[None].astype(np.int32))
    pool = torch.empty(blocks, 1, size, dtype=torch.uint8, device="cuda")
    pool[torch.from_numpy(far[:pages].copy()).cuda()] = small.pool[torch.from_numpy(small.table[0, :pages].astype(np.int64))].cuda()
    parent, sees = plain.tree(np.random.default_rng(1), rows)
    q = torch.randn(rows, rep * dim, generator=torch.Generator().manual_seed(3))
    start, lens, scale = ints([0, rows]), ints([ctx]), 1 / math.sqrt(dim)
    want, mass, top = plain.attention(small, q.view(rows, rep, dim), [ctx], [0, rows], [sees], scale)
    for n in (rows, 2):
        out = torch.empty(rows, rep * dim, device="cuda")
        ops.tree_attention_q4(dev(q), 0, rep * dim, pool, table, small.stride, lens, ints([0, n]), dev(plain.pack_mask(sees, 3)), 3, 1, n, n, ctx,
                              rep, 1, dim, scale, out, rep * dim, 0)
        err = (out[:n].cpu().double().view(n, rep, dim) - want[:n]).abs()
        assert (err <= (2.0**-17 * mass * top + 24 * 2.0**-23 * top)[:n, :, None]).all()
    pos = ctx + np.arange(rows)
    slots = dev((far[pos // 16] * 16 + pos % 16).astype(np.int64))
    draft, target = np.arange(rows, dtype=np.int32), np.full(rows, -7, np.int32)
    for i in range(rows - 1, 0, -1):
        target[parent[i]] = i
    kept = plain.commit(draft, target, parent)
    path, count, nxt, new = (torch.empty(rows, dtype=torch.int32, device="cuda") for _ in range(4))
    ops.tree_commit_q4(dev(draft), dev(target), dev(parent), start, lens, 1, rows, pool, 0, 1, table, small.stride, 1, dim, path, count, nxt, new, 0)
    assert path[: len(kept)].tolist() == kept and count[0].item() == len(kept) > 2
    back = torch.empty(2, rows, dim, device="cuda")
    ops.kv4_read(pool, blocks, slots, rows, 1, dim, back[0], dim, back[1], dim, 0, 0)
    for i, x in enumerate(small.rows(0, ctx)):
        assert torch.equal(back[i, : len(kept)].cpu().double(), x[kept, 0])
    x = torch.randn(rows, dim, device="cuda")
    ops.kv4_write(x, dim, x, dim, 0, pool, blocks, slots, rows, 1, dim, 0)
    ops.kv4_read(pool, blocks, slots, rows, 1, dim, back[0], dim, back[1], dim, 0, 0)
    assert torch.equal(back[0].cpu().double(), q4_plain.dequantise(*q4_plain.quantise(x.cpu()))) and torch.equal(back[0], back[1])


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n,rep", [(1, 4), (1, 8), (6, 4), (30, 4)])
def test_fp32_rows_are_as_near_to_64_bits_as_fp32_sums_are(ops, dim, n, rep):
    """The 2-norm of the error against that of the same attention in fp32 torch, over 2 heads of 800 keys."""
    ctx, kvh = 800, 2
    cache = q4_plain.Cache4([ctx + n], kvh, dim, 3)
    q = torch.randn(n, kvh * rep * dim, generator=torch.Generator().manual_seed(1))
    got = attention_case(ops, 0, dim, kvh, rep, [ctx], [n], cache=cache, q=q, trees="chain")
    sees = [plain.tree(None, n, "chain")[1]]
    want, _, _ = plain.attention(cache, q.view(n, kvh * rep, dim), [ctx], [0, n], sees, 1 / math.sqrt(dim))
    k, v = (x.float() for x in cache.rows(0))
    rows32 = torch.empty_like(want)
    for i in range(n):
        for h in range(kvh * rep):
            p = (k[: ctx + i + 1, h // rep] @ q[i].view(-1, dim)[h]) / math.sqrt(dim)
            p = (p - p.max()).exp()
            rows32[i, h] = (p @ v[: ctx + i + 1, h // rep]) / p.sum()
    assert (got - want).norm() <= 1.5 * (rows32 - want).norm()


# ------------------------------------------------------------------ commit


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kvh,layers,ctx,rows", [(1, 1, [5], [4]), (8, 16, [700], [26]), (3, 2, [0, 15, 16, 100], [31, 0, 1, 64]), (2, 3, [7] * 70, [9] * 70)])
def test_commit_moves_whole_rows(ops, dim, kvh, layers, ctx, rows):
    rng = np.random.default_rng(dim + sum(rows))
    caches = [q4_plain.Cache4([c + n for c, n in zip(ctx, rows)], kvh, dim, 20 + i) for i in range(layers)]
    for c in caches:
        c.table = caches[0].table
    before = torch.stack([torch.randint(0, 256, c.pool.shape, generator=torch.Generator().manual_seed(i), dtype=torch.uint8) for i, c in enumerate(caches)])
    start, parents, drafts, targets = starts(rows), [], [], []
    for n in rows:
        parent = plain.tree(rng, n)[0]
        draft, target = rng.integers(0, 50, n).astype(np.int32), rng.integers(0, 50, n).astype(np.int32)
        for i in range(n):
            below = np.flatnonzero(parent == i)
            if below.size and rng.random() < 0.9:
                target[i] = draft[rng.choice(below)]
        parents.append(parent), drafts.append(draft), targets.append(target)
    want, kept = before.clone(), [plain.commit(d, t, p) for d, t, p in zip(drafts, targets, parents)]
    for b, path in enumerate(kept):
        for i, node in enumerate(path):
            (sb, ss), (db, ds) = ((int(caches[0].table[b, x // 16]), x % 16) for x in (ctx[b] + node, ctx[b] + i))
            for v, w in zip(q4_plain.views(want, dim), q4_plain.views(want.clone(), dim)):
                v[:, db, :, :, ds] = w[:, sb, :, :, ss]
    total = sum(rows)
    new = lambda n: torch.full((max(1, n),), 55, dtype=torch.int32, device="cuda")  # noqa: E731
    path, count, nxt, lens, pool = new(total), new(len(rows)), new(len(rows)), new(len(rows)), dev(before)
    ops.tree_commit_q4(*(dev(np.concatenate(x)) for x in (drafts, targets, parents)), dev(start), ints(ctx), len(rows), max(rows), pool, pool.stride(0),
                       layers, dev(caches[0].table), caches[0].stride, kvh, dim, path, count, nxt, lens, 0)
    assert torch.equal(pool.cpu(), want)
    assert count.tolist() == [len(p) for p in kept] and lens.tolist() == [c + len(p) for c, p in zip(ctx, kept)]
    assert path[:total].tolist() == sum([p + [-1] * (n - len(p)) for p, n in zip(kept, rows)], [])
