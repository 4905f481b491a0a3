"""Attention of bf16 rows over long contexts in the 4-bit cache: sums of many products keep their size, and go down with the rest where
a reference is raised late."""

import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def attend(dim, n, rep, ctx, batch, k, v, scales, q, scale, max_ctx=None):
    """Rows of `batch` sequences over one cache of codes k, v [ctx + n, dim] with the scales of K and of V."""
    import opworks_b200

    ops = opworks_b200.ops_lib()
    pages, groups = -(-(ctx + n) // 16), dim // 32
    pool = torch.zeros(pages, 1, 18 * dim, dtype=torch.uint8, device="cuda")
    for at, codes in ((0, k), (groups * 256, v)):
        full = torch.full((pages * 16, dim), 8, dtype=torch.uint8, device="cuda")
        full[: ctx + n] = (codes + 8).to(torch.uint8)
        c = full.view(pages, 16, groups, 32).transpose(1, 2)
        pool[:, 0, at : at + groups * 256] = (c[..., 0::2] | (c[..., 1::2] << 4)).reshape(pages, -1)
    held = pool[..., groups * 512 :].view(torch.float16)
    held[..., : groups * 16], held[..., groups * 16 :] = scales
    table = torch.arange(pages, device="cuda", dtype=torch.int32).expand(batch, pages).contiguous()
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    out = torch.empty_like(q)
    ops.tree_attention_q4(q, 1, rep * dim, pool, table, pages, ints([ctx] * batch), ints([n * b for b in range(batch + 1)]), None, 0, batch, batch * n, n,
                          ctx if max_ctx is None else max_ctx, rep, 1, dim, scale, out, rep * dim, 0)
    ops.ops_sync(0)
    return out


def plain(q, row, n, ctx, k, v, scales, scale):
    """The 64-bit rows [rep, dim] of q's row `row`."""
    seen = ctx + row % n + 1
    return torch.softmax((q[row].double() @ k[:seen].double().T) * (scales[0] * scale), -1) @ (v[:seen].double() * scales[1])


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n,rep,ctx,batch", [(2, 4, 1_000_000, 160),   # 8 rows a head
                                             (4, 4, 300_000, 160),     # 16
                                             (8, 4, 300_000, 160),     # 32
                                             (30, 4, 500_000, 160),    # 120: a row tile of two streams of keys
                                             (50, 4, 300_000, 160)])   # 200: two row tiles
def test_sums_over_long_contexts_are_not_cut_down(dim, n, rep, ctx, batch):
    """V of one sign, sequences enough to fill the device. The mean of the relative error against 64 bits:
    rounding to bf16 has none (4e-5 is three standard errors of 10,000 values of 1.3e-3 each). A sum of 24 bits that is cut off
    loses less than one unit in its last place, which is up to 2^-23 of it, at each product of 16 keys: 6.1e-5 over the 8,192 keys
    of a sum in the kernel for few rows, 1.23e-4 over the 16,384 of one in the tiles. Over all keys of a warp or a stream it was
    2.9e-4 with 8 rows and 1.3e-3 with 120."""
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randint(low, 8, (ctx + n, dim), generator=g, device="cuda") for low in (-7, 0))
    q = torch.randn(batch * n, rep, dim, device="cuda", generator=g).bfloat16()
    scales, scale = (0.25, 1.0), math.sqrt(math.log(ctx / 1000) / dim)  # about 1000 keys count, so that rows are not all the same number
    out = attend(dim, n, rep, ctx, batch, k, v, scales, q, scale)
    off = []
    for row in (b * n + i for b in range(max(4, 80 // n)) for i in range(0, n, max(1, n // 8))):
        want = plain(q, row, n, ctx, k, v, scales, scale)
        off.append(((out[row].double() - want) / want).flatten())
    off = torch.cat(off)
    few = n * rep <= 32
    assert off.numel() >= 8000 and off.abs().max() <= 2.0**-7
    assert abs(off.mean().item()) <= (1e-4 if few else 1.63e-4)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n,rep,ctx,batch", [(2, 4, 100_000, 320), (4, 4, 100_000, 320), (8, 4, 100_000, 320), (30, 4, 70_000, 160), (50, 4, 40_000, 160)])
@pytest.mark.parametrize("late", [300, 5000])
def test_a_reference_raised_late(dim, n, rep, ctx, batch, late):
    """All keys score 0 and have V = 1, but for two far apart near the end, which weigh as much as all others, with V = -1 and 0.5:
    what was put by goes down with the sum of the weights. Weights are exact here but for the rows' factors: 2^-11 of the
    largest of V for weights of 11 bits, 1.23e-4 for sums that are cut off, half a step of the output."""
    levels = torch.zeros(ctx + n, dtype=torch.int64, device="cuda")
    unit = 0.05
    high = round(math.log2(ctx) / unit)
    levels[ctx - late], levels[ctx - late // 2] = high - 20, high
    levels[ctx:] = -400
    each, rest = torch.div(levels, dim, rounding_mode="floor"), levels % dim
    k = each[:, None] + (torch.arange(dim, device="cuda") < rest[:, None]).long()
    assert k.abs().max() <= 7 and torch.equal(k.sum(-1), levels)
    v = torch.full((ctx + n, dim), 4, device="cuda")
    v[ctx - late], v[ctx - late // 2] = -4, 2
    factor = (1 - torch.arange(batch * n * rep, device="cuda") % 8 / 256).bfloat16()
    q = factor[:, None].expand(-1, dim).reshape(batch * n, rep, dim).contiguous()
    scales, scale = (1.0, 0.25), unit * math.log(2)
    out = attend(dim, n, rep, ctx, batch, k, v, scales, q, scale)
    for row in (b * n + i for b in (0, 1, batch - 1) for i in (0, n // 2, n - 1)):
        want = plain(q, row, n, ctx, k, v, scales, scale)
        err = (out[row].double() - want).abs()
        assert (err <= 2.0**-8 * want.abs() + 2.0**-11 + 1.23e-4).all(), f"error {err.max():.3g}"
