"""Pages, norm and rotation, the 4-bit cache, attention and commit one after another on a stream, launched programmatically (a
kernel may start before the one before it has ended): the same bits as with ordinary launches (tests/native/libq4_step_hook.so)."""

import ctypes
import os

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

HOOK = os.path.join(os.path.dirname(os.path.abspath(__file__)), "native", "libq4_step_hook.so")


@pytest.mark.parametrize("n,rep", [(5, 2), (18, 4)])
def test_programmatic_steps_give_the_same_bits(n, rep):
    if not os.path.exists(HOOK):
        pytest.fail("tests/native/libq4_step_hook.so is missing: run __graft_entry__.build()")
    run = ctypes.CDLL(HOOK).q4_step_run
    batch, kvh, ctx, steps, kept = 6, 4, 3000, 16, 3
    qh, rows = kvh * rep, batch * n
    stride = -(-(ctx + steps * kept + n) // 16)
    blocks = batch * stride
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(steps, rows, (qh + 2 * kvh) * 64, generator=g)
    blank = torch.randint(0, 256, (blocks, kvh, 1152), generator=g, dtype=torch.uint8)
    blank[..., 1024:] = torch.rand(blocks, kvh, 64, generator=g).mul(0.3).half().view(torch.uint8)
    order = torch.randperm(blocks, generator=g).int()
    held = -(-ctx // 16)
    table0 = torch.zeros(batch, stride, dtype=torch.int32)
    table0[:, :held] = order[: batch * held].view(batch, held)
    left = blocks - batch * held
    dev = lambda t: t.clone().cuda()  # noqa: E731
    ints = lambda a: torch.tensor(a * batch, dtype=torch.int32).cuda()  # noqa: E731
    # paths 0, 2, 4: commits move rows that the attention before has read
    parent, draft = ints([-1, 0, 0, 2, 2] + [1] * (n - 5)), ints([9, 1, 2, 3, 4] + [8] * (n - 5))
    target = ints([2, 0, 4, 0, 7] + [0] * (n - 5))
    start = torch.arange(0, rows + 1, n, dtype=torch.int32).cuda()
    ends = (ctx + n + kept * torch.arange(steps, dtype=torch.int32))[:, None].expand(steps, batch).contiguous().cuda()
    weight, inv = torch.ones(64, device="cuda"), (10000.0 ** (-torch.arange(0, 64, 2) / 64)).cuda()
    got = []
    for programmatic in (0, 1, 1):
        x, pool, table, free, count0 = dev(qkv), dev(blank), dev(table0), torch.cat([order[batch * held :], torch.zeros(batch * held, dtype=torch.int32)]).cuda(), None
        count0 = torch.tensor([left], dtype=torch.int32).cuda()
        lens = torch.full((steps + 1, batch), ctx, dtype=torch.int32).cuda()
        zeros = lambda *s, **kw: torch.zeros(*s, device="cuda", **kw)  # noqa: E731
        i32 = dict(dtype=torch.int32)
        path, count, nxt, full, pos = zeros(steps, rows, **i32), zeros(steps, batch, **i32), zeros(steps, batch, **i32), zeros(steps, **i32), zeros(rows, **i32)
        slots, status, out, back = zeros(rows, dtype=torch.int64), zeros(steps, **i32), zeros(steps, rows, qh * 64), zeros(steps, 2, rows, kvh * 64)
        torch.cuda.synchronize()
        p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
        rc = run(programmatic, steps, p(x), p(weight), p(inv), p(pool), blocks, p(table), stride, p(free), p(count0), p(start), p(ends), batch, rows, n,
                 ctx + steps * kept, qh, kvh, p(draft), p(target), p(parent), p(path), p(count), p(nxt), p(lens), p(full), p(pos), p(slots), p(status), p(out), p(back),
                 ctypes.c_void_p(0))
        torch.cuda.synchronize()
        assert rc == 0
        got.append([t.cpu() for t in (x, pool, table, free, count0, lens, path, count, nxt, full, status, slots, out, back)])
    x, pool, table, free, count0, lens, path, count, nxt, full, status, slots, out, back = got[0]
    assert (count == kept).all() and (lens[-1] == ctx + steps * kept).all() and not full.any() and not status.any() and out.isfinite().all() and back.isfinite().all()
    assert count0.item() == left - batch * (-(-(ctx + steps * kept) // 16) - held)
    for other in got[1:]:
        for a, b in zip(got[0], other):
            assert torch.equal(a, b)
