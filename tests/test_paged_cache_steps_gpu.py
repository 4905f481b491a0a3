"""PagedCache (opworks_b200/tree.py) as programs run it, where the order and the place of the calls matter."""

import numpy as np
import pytest

import q4_plain

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def of(x):
    """What a 4-bit cache gives back of rows [n, 64]."""
    return q4_plain.dequantise(*q4_plain.quantise(x.float().cpu().view(-1, 1, 64)))


def held(cache, b, layer, first, n):
    """K rows [n, kvh, D] of a sequence of a 4-bit cache, in 64 bits."""
    pos = first + np.arange(n)
    table = cache.table.cpu().numpy()
    block, slot = torch.from_numpy(table[b, pos // 16].astype(np.int64)), torch.from_numpy(pos % 16)
    kc, _, ks, _ = q4_plain.views(cache.pool[layer].cpu(), cache.head_dim)
    return q4_plain.dequantise(kc[block, :, :, slot], ks[block, :, :, slot])


@pytest.mark.parametrize("format,blocks", [("int4", None), ("int4", 12), ("int8", 12), ("int8", None), ("f32", 12)])
@pytest.mark.parametrize("whole", [True, False])
def test_steps_in_inference_mode(format, blocks, whole):
    """The cache made in that mode, or before it: the same steps as outside of it, to the bit."""
    from opworks_b200.tree import PagedCache, Rows

    def steps(made, run):
        with torch.inference_mode(made):
            cache = PagedCache(2, 2, 96, 1, 64, format, blocks=blocks)
        outs = []
        with torch.inference_mode(run):
            for counts, parents in (([20, 3], None), ([4, 3], [[-1, 0, 0, 1], [-1, 0, 1]]), ([1, 1], None), ([5, 0], None)):
                rows = Rows(counts, parents)
                g = torch.Generator().manual_seed(rows.total)
                k, v = torch.randn(2, rows.total, 64, generator=g).cuda()
                q = torch.randn(rows.total, 4, 64, generator=g).cuda()
                for layer in range(2):
                    out = torch.empty_like(q)
                    cache.write(layer, k + layer, v, rows)
                    cache.attend(layer, q, rows, out, 0.125)
                    outs.append(out)
                if parents:
                    ids = torch.arange(rows.total, device="cuda")
                    target = torch.tensor([1, 3, 0, 9, 5, 9, 9], device="cuda")
                    outs += cache.commit(ids, target, rows)
                    cache.kept(outs[-2].tolist())
                else:
                    cache.advance(rows)
            if blocks:
                cache.release([1])
            outs.append(cache.lens)
        return [x.tolist() for x in outs]

    assert steps(whole, True) == steps(False, False)


def test_a_length_moved_in_inference_mode_moves_the_rows():
    from opworks_b200.tree import PagedCache, Rows

    with torch.inference_mode():
        cache, rows = PagedCache(1, 1, 64, 1, 64, "int4"), Rows([2])
        x = torch.randn(2, 64, device="cuda")
        for way, at in (("in place", 20), ("another", 40)):
            cache.write(0, x, x, rows)
            if way == "in place":
                cache.lens += 20
            else:
                cache.lens = cache.lens + 20  # made in that mode: nothing counts its changes
            cache.write(0, -x, -x, rows)
            assert torch.equal(held(cache, 0, 0, at, 2), -of(x))
        cache.lens -= 30
        cache.write(0, x * 3, x, rows)
        assert torch.equal(held(cache, 0, 0, 10, 2), of(x * 3))
