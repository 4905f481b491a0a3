"""What the 4-bit cache, shared pages and norm and rotation decide on the host: refusals, through the binding and the torch
wrapper (opworks_b200/tree.py). Nothing here launches."""

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def ops():
    import opworks_b200

    return opworks_b200.ops_lib()


def refuses(call, good, changes):
    """Each change of the good arguments (by name) is refused before anything is launched."""
    for change in changes:
        args = dict(good, **change)
        with pytest.raises(ValueError):
            call(*args.values())


A = 1 << 20  # an address that is aligned and never touched


def test_record_bytes(ops):
    assert ops.kv4_record_bytes(64) == 1152 and ops.kv4_record_bytes(128) == 2304
    for dim in (0, 32, 80, 256, -64):
        with pytest.raises(ValueError, match="head_dim"):
            ops.kv4_record_bytes(dim)


def test_pages_refuse(ops):
    good = dict(lens=A, start=A, batch=2, rows=5, table=A, stride=4, free=A, count=A, positions=A, slots=A, left=A, status=A, stream=0)
    refuses(ops.page_take, good, [dict(batch=-1), dict(rows=-1), dict(stride=0), dict(stride=2**28), dict(lens=None), dict(start=None), dict(table=None),
                                  dict(positions=None), dict(slots=None), dict(status=None), dict(count=None), dict(left=None)])
    good = dict(old=A, new=A, batch=2, table=A, stride=4, free=A, capacity=9, count=A, left=A, status=A, stream=0)
    refuses(ops.page_give, good, [dict(batch=-1), dict(stride=0), dict(capacity=-1), dict(old=None), dict(new=None), dict(table=None), dict(free=None),
                                  dict(count=None), dict(left=None), dict(status=None), dict(stride=2**28)])


def test_norm_and_rotation_refuse(ops):
    good = dict(q=A, qs=512, k=A, ks=128, type=0, qw=A, kw=A, eps=1e-5, pos=A, inv=A, rot=64, rows=3, qh=8, kvh=2, dim=64, qo=A, qos=512, ko=A, kos=128, stream=0)
    refuses(ops.qk_norm_rope, good, [dict(type=2), dict(rows=-1), dict(qh=-1), dict(kvh=70000), dict(dim=96), dict(dim=512), dict(rot=24), dict(rot=80),
                                     dict(rot=-16), dict(eps=0.0), dict(eps=-1.0), dict(eps=float("nan")), dict(q=None), dict(k=None), dict(qo=None), dict(ko=None),
                                     dict(pos=None), dict(inv=None), dict(qs=511), dict(qs=508), dict(ks=64), dict(qs=513), dict(kos=130), dict(q=A + 4),
                                     dict(ko=A + 8)])
    refuses(ops.qk_norm_rope, dict(good, type=1), [dict(qs=516), dict(q=A + 8)])


def test_rows_refuse(ops):
    good = dict(k=A, ks=128, v=A, vs=128, type=0, pool=A, blocks=3, slots=A, rows=5, kvh=2, dim=64, stream=0)
    refuses(ops.kv4_write, good, [dict(k=None), dict(v=None), dict(pool=None), dict(slots=None), dict(type=2), dict(type=-1), dict(ks=64), dict(vs=124), dict(ks=130),
                                  dict(k=A + 8), dict(v=A + 4), dict(pool=A + 8), dict(blocks=-1), dict(rows=-1), dict(kvh=0), dict(kvh=5000), dict(dim=32)])
    good = dict(pool=A, blocks=3, slots=A, rows=5, kvh=2, dim=64, k=A, ks=128, v=A, vs=128, type=1, stream=0)
    refuses(ops.kv4_read, good, [dict(k=None), dict(pool=None), dict(slots=None), dict(type=3), dict(ks=100), dict(vs=132), dict(pool=A + 4), dict(rows=-2),
                                 dict(kvh=0), dict(dim=256)])


def test_attention_and_commit_refuse(ops):
    good = dict(q=A, type=0, qs=512, pool=A, table=A, stride=4, ctx=A, start=A, mask=A, words=1, batch=2, rows=5, most=3, most_ctx=40, qh=8, kvh=2, dim=64,
                scale=0.125, out=A, os=512, stream=0)
    refuses(ops.tree_attention_q4, good, [dict(type=2), dict(q=None), dict(out=None), dict(pool=None), dict(table=None), dict(ctx=None), dict(start=None),
                                          dict(stride=0), dict(words=0), dict(batch=-1), dict(batch=70000), dict(rows=-1), dict(most=6), dict(most_ctx=-1),
                                          dict(qh=7), dict(kvh=0), dict(dim=32), dict(dim=256), dict(qs=500), dict(os=511), dict(qs=514), dict(q=A + 4),
                                          dict(pool=A + 8), dict(out=A + 8), dict(mask=None, rows=2**30, most=2**30)])
    good = dict(draft=A, target=A, parent=A, start=A, ctx=A, batch=2, most=5, pool=A, layer=1024, layers=2, table=A, stride=4, kvh=2, dim=64, path=A, count=A,
                next=A, new=A + 64, stream=0)
    refuses(ops.tree_commit_q4, good, [dict(draft=None), dict(parent=None), dict(pool=None), dict(most=4000), dict(layers=0), dict(layer=0), dict(layer=1000),
                                       dict(kvh=0), dict(dim=80), dict(new=A), dict(batch=-1), dict(pool=A + 4)])


# ------------------------------------------------------------------ the wrapper


def cache(format="int4", batch=2, tokens=64, **kw):
    from opworks_b200.tree import PagedCache

    return PagedCache(1, batch, tokens, 2, 64, format, device="cpu", **kw)


def test_a_shared_cache_refuses_rows_that_it_has_no_pages_for():
    from opworks_b200.tree import Rows

    c = cache(blocks=5)
    assert c.pool.shape == (1, 5, 2, 1152) and c.free.tolist() == [4, 3, 2, 1, 0] and c.free_count.item() == 5
    with pytest.raises(ValueError, match="pages"):
        c.place(Rows([33, 48], device="cpu"))
    with pytest.raises(ValueError, match="room"):
        c.place(Rows([65, 1], device="cpu"))
    with pytest.raises(ValueError, match="sequences"):
        c.place(Rows([1], device="cpu"))
    c.bounds = [40, 30]
    with pytest.raises(ValueError, match="pages"):
        c.place(Rows([9, 0], device="cpu"))
    for gone in ([2], [-1], [0, 7]):
        with pytest.raises(ValueError, match="release"):
            c.release(gone)


def test_a_step_on_the_cpu_is_refused():
    from opworks_b200.tree import Rows

    rows = Rows([3, 2], device="cpu")
    for c in (cache(), cache(blocks=8), cache("int8", blocks=8)):
        for call in (lambda: c.place(rows) if c.shared else c.write(0, torch.zeros(5, 128), torch.zeros(5, 128), rows), lambda: c.release([0]) if c.shared else c.read(0, rows)):
            with pytest.raises(ValueError, match="device"):
                call()


def test_norm_and_rotation_refuse_tensors_that_they_would_misread():
    from opworks_b200.tree import qk_norm_rope

    q, k, pos, inv, w = torch.randn(5, 8, 64), torch.randn(5, 2, 64), torch.zeros(5, dtype=torch.int32), torch.ones(32), torch.ones(64)
    bad = [(q, k.bfloat16(), pos, inv, w, w), (q.half(), k.half(), pos, inv, w, w), (q[:4], k, pos, inv, w, w), (q[..., :32], k, pos, inv, w, w), (q.view(5, 512), k, pos, inv, w, w),
           (q, k, pos.long(), inv, w, w), (q, k, pos[:4], inv, w, w), (q, k, pos, inv.double(), w, w), (q, k, pos, inv, w[:32], w), (q, k, pos, inv, w, w.half()),
           (q, k, None, inv, w, w), (q.transpose(0, 1)[:5], k, pos, inv, w, w), (torch.randn(5, 64, 8).transpose(1, 2), k, pos, inv, w, w), (q, k, pos, inv, w, w.to("meta")),
           (q, k, torch.zeros(10, dtype=torch.int32)[::2], inv, w, w)]
    for args in bad:
        with pytest.raises(ValueError):
            qk_norm_rope(*args)
    for out in ((q, q), (q.bfloat16(), k), (q[:, :4], k), (q, torch.empty(5, 64, 2).transpose(1, 2))):
        with pytest.raises(ValueError):
            qk_norm_rope(q, k, pos, inv, w, w, out=out)
    with pytest.raises(ValueError, match="device"):
        qk_norm_rope(q, k, pos, inv, w, w)


def test_write_and_attend_refuse_as_the_other_formats_do():
    from opworks_b200.tree import Rows

    c, rows = cache(), Rows([3, 2], device="cpu")
    k = torch.randn(5, 128)
    for bad_k, bad_v in [(k, k.bfloat16()), (k.double(), k.double()), (k[:4], k[:4]), (k, k[:4]), (k[:, :64], k[:, :64]), (k, k.to("meta")), (k.half(), k.half())]:
        with pytest.raises(ValueError):
            c.write(0, bad_k, bad_v, rows)
    q = torch.randn(5, 8, 64)
    for bad_q, bad_out in [(q, q.bfloat16()), (q.half(), q.half()), (q[:4], q[:4]), (q[..., :32], q[..., :32]), (torch.randn(8, 5, 64).transpose(0, 1), q)]:
        with pytest.raises(ValueError):
            c.attend(0, bad_q, rows, bad_out, 0.125)
