"""The 8-bit cache's kernels, attention and commit one after another on a stream, launched programmatically (a kernel may
start before the one before it has ended): the same bits as with ordinary launches (tests/native/libtree_step_hook.so)."""

import ctypes
import os

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

HOOK = os.path.join(os.path.dirname(os.path.abspath(__file__)), "native", "libtree_step_hook.so")


def test_programmatic_steps_give_the_same_bits():
    if not os.path.exists(HOOK):
        pytest.fail("tests/native/libtree_step_hook.so is missing: run __graft_entry__.build()")
    run = ctypes.CDLL(HOOK).tree_step_run
    batch, n, kvh, qh, ctx, steps = 6, 5, 4, 8, 5000, 24
    rows, stride = batch * n, -(-(ctx + n) // 16)
    g = torch.Generator().manual_seed(1)
    q = torch.randn(rows, qh * 64, generator=g).cuda()
    k, v = (torch.randn(steps, rows, kvh * 64, generator=g).cuda() for _ in range(2))
    table = torch.randperm(batch * stride, generator=g).int().view(batch, stride).cuda()
    blank = torch.randint(0, 256, (batch * stride, kvh, 2176), generator=g, dtype=torch.uint8)
    blank[..., 2048:] = torch.rand(batch * stride, kvh, 32, generator=g).mul(0.01).view(torch.uint8)
    lens = torch.full((batch,), ctx, dtype=torch.int32).cuda()
    start = torch.arange(0, rows + 1, n, dtype=torch.int32).cuda()
    # paths 0, 2, 4: commits move rows that the attention before has read
    ints = lambda *a: torch.tensor(a * batch, dtype=torch.int32).cuda()  # noqa: E731
    parent, draft, target = ints(-1, 0, 0, 2, 2), ints(9, 1, 2, 3, 4), ints(2, 0, 4, 0, 7)
    got = []
    for programmatic in (0, 1, 1):
        pool = blank.clone().cuda()
        out = torch.zeros(steps, rows, qh * 64, device="cuda")
        back = torch.zeros(steps, 2, rows, kvh * 64, device="cuda")
        path = torch.zeros(steps, rows, dtype=torch.int32, device="cuda")
        count, nxt, new = (torch.zeros(steps, batch, dtype=torch.int32, device="cuda") for _ in range(3))
        torch.cuda.synchronize()
        p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
        rc = run(programmatic, steps, p(q), p(k), p(v), p(pool), p(table), stride, p(lens), p(start), batch, rows, n, ctx, qh, kvh,
                 p(draft), p(target), p(parent), p(path), p(count), p(nxt), p(new), p(out), p(back), ctypes.c_void_p(0))
        torch.cuda.synchronize()
        assert rc == 0
        got.append([x.cpu() for x in (out, back, path, count, nxt, new, pool)])
    assert (got[0][3] == 3).all() and (got[0][5] == ctx + 3).all() and np.isfinite(got[0][0].numpy()).all()
    for other in got[1:]:
        for a, b in zip(got[0], other):
            assert torch.equal(a, b)
