"""Commit of drafted trees whose pages have ids from 2^27 on (16 times an id is no int there), in the pools of every format."""

import numpy as np
import pytest

import tree_cache_plain as plain

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

RECORD = {"q4": 18 * 64, "q8": 32 * 64 + 128, "f32": 16 * 64 * 4}  # bytes of a block of one head of 64 dims (f32: of K, of V)


# where a token's parts lie in a block: (first byte, bytes from slot to slot and of a slot)
PARTS = {"q4": [(256 * i, 16) for i in range(4)] + [(1024 + 32 * i, 2) for i in range(4)], "q8": [(0, 64), (1024, 64), (2048, 4), (2112, 4)], "f32": [(0, 256)]}


@pytest.mark.parametrize("form", ["q4", "q8", "f32"])
@pytest.mark.parametrize("first", [0, 2**27 - 3, 2**27, 3 * 2**27, 2**31 - 9])
def test_accepted_rows_move_between_far_blocks(form, first):
    """The pool is 8 blocks; its address is given as that of block 0, `first` blocks further down, so only those 8 are touched."""
    import opworks_b200

    ops = opworks_b200.ops_lib()
    rng = np.random.default_rng(3)
    n, ctx, blocks, size = 60, 37, 8, RECORD[form]
    pools = [torch.randint(0, 256, (blocks, size), generator=torch.Generator().manual_seed(i), dtype=torch.uint8) for i in range(2 if form == "f32" else 1)]
    order = rng.permutation(blocks)
    parent, _ = plain.tree(rng, n)
    draft, target = np.arange(n, dtype=np.int32), np.full(n, -7, np.int32)
    for i in range(n - 1, 0, -1):
        target[parent[i]] = i
    kept = plain.commit(draft, target, parent)
    assert len(kept) > 3 and kept != list(range(len(kept)))
    dev = lambda x: torch.as_tensor(np.asarray(x, np.int32)).cuda()  # noqa: E731
    table, new = dev((order + first)[None]), [torch.empty(n, dtype=torch.int32, device="cuda") for _ in range(4)]
    pool = [p.cuda() for p in pools]
    at = [p.data_ptr() - first * size for p in pool]
    head = (dev(draft), dev(target), dev(parent), dev([0, n]), dev([ctx]), 1, n)
    call = {"q4": ops.tree_commit_q4, "q8": ops.tree_commit_q8, "f32": ops.tree_commit}[form]
    call(*head, *at, 0, 1, table, blocks, 1, 64, *new, 0)
    ops.ops_sync(0)
    assert new[0][: len(kept)].tolist() == kept and new[1][0].item() == len(kept)
    for before, after in zip(pools, pool):
        want = before.clone()
        for i, node in enumerate(kept):
            (sb, ss), (db, ds) = ((int(order[x // 16]), x % 16) for x in (ctx + node, ctx + i))
            for lo, width in PARTS[form]:
                want[db, lo + ds * width : lo + (ds + 1) * width] = before[sb, lo + ss * width : lo + (ss + 1) * width]
        assert torch.equal(after.cpu(), want)
