"""Attention over the 4-bit cache where the block table ends before the sequence does, or has no block for a page."""

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


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def finite_block_0(cache):
    """Block 0, which places after the last page stand for, holds numbers that would count."""
    kc, vc, ks, vs = q4_plain.views(cache.pool, cache.dim)
    kc[0], vc[0], ks[0], vs[0] = 0x5B, 0xF1, 1.0, 2.0


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("ctx,n,pages", [(100, 40, 7), (100, 70, 9), (250, 60, 17), (16, 5, 1), (90, 3, 5)])
def test_a_chain_that_is_longer_than_its_table_row(ops, kind, dim, ctx, n, pages):
    """Rows see what the table has pages for, whichever kernel takes them."""
    rep, places = 4, 16 * pages
    cache = q4_plain.Cache4([ctx + n], 1, dim, 5)
    finite_block_0(cache)
    q = torch.randn(n, rep, dim, generator=torch.Generator().manual_seed(1)).to(TYPES[kind])
    k, v = cache.rows(0, 0, places)
    want = torch.zeros(n, rep, dim, dtype=torch.float64)
    scale = 1 / math.sqrt(dim)
    for i in range(n):
        seen = min(places, min(ctx, places) + i + 1)
        want[i] = torch.softmax(scale * q[i].double() @ k[:seen, 0].T, -1) @ v[:seen, 0]
    out = torch.empty(n, rep, dim, dtype=TYPES[kind], device="cuda")
    table = torch.from_numpy(cache.table[:, :pages].copy()).cuda()
    ops.tree_attention_q4(q.cuda(), kind, rep * dim, cache.pool.cuda(), table, pages, ints([ctx]), ints([0, n]), None, 0, 1, n, n, ctx, rep, 1, dim, scale, out,
                          rep * dim, 0)
    err, top = (out.cpu().double() - want).abs(), v.abs().max()
    tol = 2.0**-14 * top + (2.0**-8 * want.abs() + 2.0**-10 * top if kind else 0)
    assert (err <= tol).all(), f"error {err.max():.3g}"


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("n", [3, 40, 90])
def test_a_page_that_no_row_sees_may_have_no_block(ops, kind, n):
    """The last nodes' page has the id -1, and the mask hides all of it: nothing in front of the pool is read, in any kernel."""
    rep, dim, ctx = 4, 64, 48 - n % 16 if n > 16 else 32  # the last page holds nodes only
    cache = q4_plain.Cache4([ctx + n + 16], 1, dim, 5)
    sees = [plain.tree(np.random.default_rng(1), n)[1]]
    hidden = np.arange(n) + ctx >= 16 * ((ctx + n - 1) // 16)
    sees[0][:, hidden] = False
    scale = 1 / math.sqrt(dim)
    q = torch.randn(n, rep, dim, generator=torch.Generator().manual_seed(1)).to(TYPES[kind])
    want, mass, top = plain.attention(cache, q, [ctx], [0, n], sees, scale)
    cache.table[0, (ctx + n - 1) // 16 :] = -1
    words = -(-n // 32)
    out = torch.empty(n, rep, dim, dtype=TYPES[kind], device="cuda")
    ops.tree_attention_q4(q.cuda(), kind, rep * dim, cache.pool.cuda(), torch.from_numpy(cache.table).cuda(), cache.stride, ints([ctx]), ints([0, n]),
                          torch.from_numpy(plain.pack_mask(sees[0], words)).cuda(), words, 1, n, n, ctx, rep, 1, dim, scale, out, rep * dim, 0)
    err = (out.cpu().double() - want).abs()
    tol = (2.0**-17 * mass * top + 24 * 2.0**-23 * top)[..., None] + (2.0**-8 * want.abs() + 2.0**-10 * top[..., None] if kind else 0)
    assert (err <= tol).all(), f"error {err.max():.3g}"
