"""Attention of bf16 rows over contexts of a million tokens in the 4-bit cache: sums of so many products keep their size."""

import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n,rep,ctx,batch", [(2, 4, 1_000_000, 160),   # 8 rows a head: the kernel for few
                                             (30, 4, 500_000, 160)])   # 120: a row tile of two streams of keys
def test_sums_over_long_contexts_are_not_cut_down(dim, n, rep, ctx, batch):
    """V of one sign, sequences enough to fill the device, one cache for all. The mean of the relative error against 64 bits:
    rounding to bf16 has none (4e-5 is three standard errors of 10,000 values of 1.3e-3 each). A sum of 24 bits that is cut off
    loses less than one unit in its last place, which is up to 2^-23 of it, at each product of 16 keys: 6.1e-5 over the 8,192 keys
    that a warp's sum is held to, 2.4e-4 over half of the 62,500 of a CTA of 8. Over all keys of a warp (1.25e5) or a stream of
    tiles (2.5e5) it was 2.9e-4 and 1.3e-3."""
    import opworks_b200

    ops = opworks_b200.ops_lib()
    pages, groups = -(-(ctx + n) // 16), dim // 32
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randint(low, 16, (pages, groups, 16, 32), generator=g, device="cuda", dtype=torch.uint8) for low in (1, 8))
    pool = torch.empty(pages, 1, 18 * dim, dtype=torch.uint8, device="cuda")
    pack = lambda c: (c[..., 0::2] | (c[..., 1::2] << 4)).reshape(pages, -1)  # noqa: E731
    pool[:, 0, : groups * 256], pool[:, 0, groups * 256 : groups * 512] = pack(k), pack(v)
    scales = pool[..., groups * 512 :].view(torch.float16)
    scales[..., : groups * 16], scales[..., groups * 16 :] = 0.25, 1.0
    table = torch.arange(pages, device="cuda", dtype=torch.int32).expand(batch, pages).contiguous()
    q = torch.randn(batch * n, rep, dim, device="cuda", generator=g).bfloat16()
    scale = math.sqrt(math.log(ctx / 1000) / dim)  # about 1000 keys count, so that rows are not all the same number
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    out = torch.empty_like(q)
    ops.tree_attention_q4(q, 1, rep * dim, pool, table, pages, ints([ctx] * batch), ints([n * b for b in range(batch + 1)]), None, 0, batch, batch * n, n, ctx, rep, 1, dim,
                          scale, out, rep * dim, 0)
    ops.ops_sync(0)
    plain = lambda c, s: ((c.double() - 8) * s).permute(0, 2, 1, 3).reshape(-1, dim)  # noqa: E731
    k, v, off = plain(k, 0.25), plain(v, 1.0), []
    looked = range(40) if n == 2 else range(4)
    for row in (b * n + i for b in looked for i in range(0, n, max(1, n // 8))):
        seen = ctx + row % n + 1
        want = torch.softmax((q[row].double() @ k[:seen].T) * scale, -1) @ v[:seen]
        off.append(((out[row].double() - want) / want).flatten())
    off = torch.cat(off)
    assert off.numel() >= 8000 and abs(off.mean().item()) <= (1e-4 if n == 2 else 2.8e-4) and off.abs().max() <= 2.0**-7
