"""Cases of the attention half of a serving step over a 4-bit paged KV cache.

Four operators, in the order in which a step of a serving program calls them:

* ``pages``: block tables and slot maps are built on the GPU from the requests' lengths: ``take`` gives every sequence
  the pages that its new tokens need, and says where each token goes; ``give`` puts pages back that are needed no more;
* ``norm``: queries and keys are normalised for each head (root mean square) and rotated by their positions, in one pass;
* ``rows``: K and V rows are stored in 4 bits where the slot map says, and fetched again;
* ``attn``: the new tokens of each sequence (one, a prompt's piece, a drafted tree) attend to its context and to each
  other over the 4-bit cache.

Pages hold 16 tokens, a slot is 16 * block + place in the page. The 4-bit pool has one record of 576 G bytes per block
and kv head, G = D / 32 groups of 32 dims: K codes [G][16 tokens][16 bytes], V codes the same, K scales fp16 [G][16], V
scales fp16 [G][16]. Byte i of a group's 16 holds dims 2 i (low half) and 2 i + 1. A value is (code - 8) * scale, the
scale max|x| / 7 of the group rounded to an fp16 number of 5 significant bits, so that every value is an fp16 number too.

``run`` computes the plain form with elementary torch operations, or calls the framework where ``own`` is true.
"""

import math

import numpy as np
import torch

own = False

PAGE = 16
GROUP = 32
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
TYPE_CODES = {"f32": 0, "bf16": 1}
EPS = 1e-5


# ------------------------------------------------------------------ cases


def listed():
    return [
        # 32 sequences take what one more token each needs: the smallest call
        dict(name="take_step", op="pages", way="take", batch=32, ctx=2180, rows=1, stride=257),
        # pages and slots of a batch of prompts, some behind prefixes that are cached already
        dict(name="take_prompts", op="pages", way="take", batch=48, ctx=1000, rows=2048, stride=300),
        # a large batch gives back what it has, or what its drafts did not need
        dict(name="give_batch", op="pages", way="give", batch=512, ctx=4000, rows=64, stride=260),
        # one new token of each of 32 sequences, fp32 rows of the projections
        dict(name="norm_step", op="norm", dtype="f32", rows=32, qh=32, kvh=8, dim=128, rot=128, far=8192),
        # prompts in bf16, wide heads, queries and keys as slices of one projection
        dict(name="norm_prompts", op="norm", dtype="bf16", rows=16384, qh=32, kvh=8, dim=128, rot=128, far=131072),
        # one new token of each of 32 sequences is stored, and read back as a check would
        dict(name="store_step", op="rows", way="store", dtype="f32", batch=32, ctx=2180, rows=1, kvh=8, dim=64, pad=0),
        # ragged prompts stored and fetched, K and V as slices of one projection
        dict(name="store_prompts", op="rows", way="store", dtype="bf16", batch=16, ctx=333, rows=2048, kvh=8, dim=128, pad=4096),
        # shared prefixes fetched for attention that wants plain rows
        dict(name="fetch_prefixes", op="rows", way="fetch", dtype="bf16", batch=16, ctx=0, rows=4096, kvh=8, dim=64, pad=0),
        # a decode step of 32 sequences
        dict(name="attn_decode", op="attn", dtype="f32", batch=32, ctx=2180, rows=1, qh=32, kvh=8, dim=64, tree="chain"),
        # a decode step of a few very long sequences, wide heads
        dict(name="attn_long", op="attn", dtype="bf16", batch=12, ctx=32000, rows=1, qh=32, kvh=8, dim=128, tree="chain"),
        # ordinary drafted trees, ragged contexts
        dict(name="attn_trees", op="attn", dtype="f32", batch=8, ctx=4099, rows=26, qh=32, kvh=8, dim=64, tree="tree"),
        # the largest: pieces of prompts behind what is cached of them
        dict(name="attn_prompts", op="attn", dtype="bf16", batch=3, ctx=2100, rows=2048, qh=32, kvh=8, dim=128, tree="chain"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["pages", "norm", "rows", "rows", "attn", "attn", "attn"])
    dim = rng.choice([64, 128])
    kvh = rng.choice([1, 2, 4, 8, 8, 16])
    if op == "pages":
        batch = _log(rng, 1, 600)
        rows = _log(rng, 1, max(2, min(4096, 90000 // batch)))
        ctx = rng.randrange(0, 6000)
        return dict(op=op, way=rng.choice(["take", "take", "give"]), batch=batch, ctx=ctx, rows=rows,
                    stride=(ctx + rows) // PAGE + rng.randrange(2, 60))
    if op == "norm":
        qh = kvh * rng.choice([1, 2, 3, 4, 4, 7, 8])
        return dict(op=op, dtype=rng.choice(["f32", "bf16"]), rows=_log(rng, 1, max(2, min(20000, 16384 * 40 * 64 // ((qh + kvh) * dim)))),
                    qh=qh, kvh=kvh, dim=dim, rot=rng.choice([dim, dim, dim, dim // 2, 32]), far=_log(rng, 100, 1000000))
    batch = _log(rng, 1, 64)
    if op == "rows":
        most = max(1, 26000 * 8 * 64 // (batch * kvh * dim))
        return dict(op=op, way=rng.choice(["store", "store", "fetch"]), dtype=rng.choice(["f32", "bf16"]), batch=batch,
                    ctx=rng.randrange(0, 3000), rows=_log(rng, 1, min(8192, most)), kvh=kvh, dim=dim,
                    pad=rng.choice([0, 64, 512]))
    rep = rng.choice([1, 2, 3, 4, 4, 7, 8])
    kvh = rng.choice([1, 2, 4, 8, 8])
    dtype = rng.choice(["f32", "bf16", "bf16"])
    tree = rng.choice(["chain", "chain", "tree"])
    rows = rng.choice([1, 1, _log(rng, 2, 100), _log(rng, 100, 1500) if tree == "chain" else _log(rng, 2, 70)])
    # no more work, rows of scores and rows of the cache than the largest listed cases have
    rows = min(rows, max(1, int(math.sqrt(3e10 / (batch * rep * kvh * dim)))))
    most = max(64, min(32000, int(3 * 2048 * 3000 * 32 * 128 * 0.4 / (batch * rows * rep * kvh * dim)),
                       int(12 * 32000 * 8 * 0.6 / (batch * kvh))))
    return dict(op=op, dtype=dtype, batch=batch, ctx=_log(rng, 1, most), rows=rows, qh=kvh * rep, kvh=kvh, dim=dim, tree=tree)


# ------------------------------------------------------------------ sizes of a case


def _counts(case):
    """(context length, new rows) of each sequence: the case's own are the largest, the others spread below them."""
    b = np.arange(case["batch"])
    ctx = np.round(case["ctx"] * (1.0 - 0.5 * ((b * 0.6180339887498949) % 1.0))).astype(np.int64)
    rows = np.maximum(1, np.round(case["rows"] * (1.0 - 0.4 * ((b * 0.7548776662466927) % 1.0)))).astype(np.int64)
    return ctx, rows


def _pages(tokens):
    return -(-tokens // PAGE)


def work(case):
    if case["op"] == "norm":
        e = 4 if case["dtype"] == "f32" else 2
        values = case["rows"] * (case["qh"] + case["kvh"]) * case["dim"]
        return {"bytes": 2 * values * e + 4 * case["rows"] + 8 * case["dim"], "flops": 7 * values}
    ctx, rows = _counts(case)
    total = int(rows.sum())
    if case["op"] == "pages":
        moved = int((_pages(ctx + rows) - _pages(ctx)).sum())
        if case["way"] == "take":  # ids read and written; lengths; a position and a slot for each row
            return {"bytes": 8 * moved + 12 * case["batch"] + 12 * total, "flops": 4 * total}
        return {"bytes": 8 * moved + 8 * case["batch"], "flops": moved}
    kvh, dim = case["kvh"], case["dim"]
    code_row = 2 * kvh * (dim // 2 + 2 * (dim // GROUP))
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "rows":
        wide = 2 * dim * kvh * e
        ways = 2 if case["way"] == "store" else 1  # stored and fetched, or fetched
        return {"bytes": ways * total * (code_row + wide + 8), "flops": ways * total * 4 * dim * kvh}
    seen = int((rows * ctx + rows * (rows + 1) // 2).sum())
    return {"bytes": int((ctx + rows).sum()) * code_row + 2 * total * case["qh"] * dim * e, "flops": 4 * dim * case["qh"] * seen}


# ------------------------------------------------------------------ the 4-bit format


def _quantise(x):
    """Codes 0 .. 15 (int32) and scales (fp32) [..., G] of rows x [..., D]."""
    g = x.float().unflatten(-1, (-1, GROUP))
    top = g.abs().amax(-1) * torch.tensor(1.0 / 7.0, dtype=torch.float32, device=x.device)
    bits = top.view(torch.int32)
    scale = ((bits + 0x3FFFF + ((bits >> 19) & 1)) & ~0x7FFFF).view(torch.float32)
    scale = torch.where(top < 2.0**-20, (top * 2.0**24).round() * 2.0**-24, scale)  # fp16 has no finer step
    y = torch.where(scale[..., None] > 0, g / scale[..., None], torch.zeros_like(g))
    return (y.round().clamp_(-7, 7) + 8).to(torch.int32).flatten(-2), scale


def _views(pool, dim):
    """K codes, V codes [..., G, 16, 16 bytes] and K, V scales fp16 [..., G, 16] of a pool [..., record]."""
    g = dim // GROUP
    n = g * PAGE * 16
    k, v = (pool[..., i * n : (i + 1) * n].unflatten(-1, (g, PAGE, 16)) for i in (0, 1))
    s = pool[..., 2 * n :].view(torch.float16)
    return k, v, s[..., : g * PAGE].unflatten(-1, (g, PAGE)), s[..., g * PAGE :].unflatten(-1, (g, PAGE))


def _store(codes, scales, where, x):
    """Rows x [n, kvh, D] into the places `where` = (block, slot in the page) of K's or of V's views."""
    c, s = _quantise(x)
    c = c.unflatten(-1, (-1, 16, 2))
    packed = (c[..., 0] | (c[..., 1] << 4)).to(torch.uint8)  # [n, kvh, G, 16]
    block, slot = where
    codes[block, :, :, slot] = packed
    scales[block, :, :, slot] = s.to(torch.float16)


def _fetch(codes, scales, where):
    """The rows at `where`, [n, kvh, D] in fp32."""
    block, slot = where
    c = codes[block, :, :, slot].to(torch.int32)
    c = torch.stack([c & 15, c >> 4], -1).flatten(-2) - 8
    return (c.float() * scales[block, :, :, slot].float()[..., None]).flatten(-2)


def _rows(shape, gen):
    """K or V rows: normal values, channels of unlike size."""
    x = torch.randn(shape, generator=gen, device="cuda")
    return x.mul_(torch.randn(shape[-1:], generator=gen, device="cuda").mul_(0.5).exp_())


def _random_pool(blocks, kvh, dim, gen):
    """Pool [blocks, kvh, record] of random rows, filled in pieces."""
    pool = torch.empty(blocks, kvh, 18 * dim, dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 25) // (PAGE * dim * kvh))
    slot = torch.arange(PAGE, device="cuda")
    for i in range(0, blocks, step):
        part = pool[i : i + step]
        n = part.shape[0]
        kc, vc, ks, vs = _views(part, dim)
        at = (torch.arange(n, device="cuda").repeat_interleave(PAGE), slot.repeat(n))
        for codes, scales in ((kc, ks), (vc, vs)):
            _store(codes, scales, at, _rows((n * PAGE, kvh, dim), gen))
    return pool


# ------------------------------------------------------------------ inputs


def _tree(rng, n, shape):
    """Ancestor rows (with the node itself) of one tree; a node comes after its parent."""
    sees = np.zeros((n, n), bool)
    for i in range(n):
        if i:
            sees[i] = sees[i - 1 if shape == "chain" else rng.integers(max(0, i // 3 - 2), i)]
        sees[i, i] = True
    return sees


def _pack(sees, words):
    out = np.zeros((sees.shape[0], words * 32), np.uint32)
    out[:, : sees.shape[1]] = sees
    return (out.reshape(-1, words, 32) << np.arange(32, dtype=np.uint32)).sum(-1, dtype=np.uint32).view(np.int32)


def _ints(*arrays):
    return [torch.from_numpy(np.ascontiguousarray(a).astype(np.int32)).cuda() for a in arrays]


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    if case["op"] == "norm":
        return _prepare_norm(case, gen, rng)
    ctx, rows = _counts(case)
    batch, total = case["batch"], int(rows.sum())
    pages = _pages(ctx + rows)
    stride = max(int(pages.max()) + 2, case.get("stride", 0))  # a table wider than the longest sequence needs
    blocks = int(pages.sum()) + 7
    order = rng.permutation(blocks)
    start = np.concatenate([[0], np.cumsum(rows)])
    held = _pages(ctx) if case["op"] == "pages" and case["way"] == "take" else pages  # pages that the table has already
    table, at = np.zeros((batch, stride), np.int32), 0
    for b in range(batch):
        table[b, : held[b]] = order[at : at + held[b]]
        at += int(held[b])
    s = dict(case=dict(case), op=case["op"], batch=batch, total=total, stride=stride, blocks=blocks, most=int(rows.max()),
             most_ctx=int(ctx.max()))
    s["table"], s["ctx"], s["start"], owner = _ints(table, ctx, start, np.repeat(np.arange(batch), rows))
    s["owner"] = owner.long()
    s["node"] = torch.arange(total, device="cuda") - s["start"].long()[s["owner"]]
    if case["op"] == "pages":
        stack = np.zeros(blocks, np.int32)
        stack[: blocks - at] = order[at:]
        s["free"], s["count"] = _ints(stack, [blocks - at])
        s["left"], s["status"] = torch.empty_like(s["count"]), torch.empty_like(s["count"])
        if case["way"] == "take":
            s["positions"] = torch.empty(total, dtype=torch.int32, device="cuda")
            s["slots"] = torch.empty(total, dtype=torch.int64, device="cuda")
        else:  # a third of the sequences end, the others keep all or some of their last rows
            keep = np.where(rng.random(batch) < 0.33, 0, ctx + np.minimum(rows, rng.integers(0, case["rows"] + 1, batch)))
            s["old"], s["new"] = _ints(ctx + rows, keep)
        return s
    kvh, dim, s["dtype"] = case["kvh"], case["dim"], TYPES[case["dtype"]]
    s["kvh"], s["dim"] = kvh, dim
    pos = s["ctx"].long()[s["owner"]] + s["node"]
    s["slots"] = s["table"].long()[s["owner"], pos // PAGE] * PAGE + pos % PAGE
    if case["op"] == "rows":
        width = kvh * dim
        s["width"] = width
        if case["way"] == "store":
            s["pool"] = torch.zeros(blocks, kvh, 18 * dim, dtype=torch.uint8, device="cuda")
            wide = torch.cat([torch.zeros(total, case["pad"], device="cuda"), _rows((total, kvh, dim), gen).view(total, width),
                              _rows((total, kvh, dim), gen).view(total, width)], 1).to(s["dtype"])
            s["k"], s["v"] = wide[:, case["pad"] : case["pad"] + width], wide[:, case["pad"] + width :]
        else:
            s["pool"] = _random_pool(blocks, kvh, dim, gen)
        s["k_out"], s["v_out"] = (torch.empty(total, width, dtype=s["dtype"], device="cuda") for _ in range(2))
        return s
    most, qh = s["most"], case["qh"]
    s["pool"] = _random_pool(blocks, kvh, dim, gen)
    s["qh"] = qh
    s["q"] = _rows((total, qh, dim), gen).to(s["dtype"])
    s["out"] = torch.empty_like(s["q"])
    s["scale"] = 1.0 / math.sqrt(dim)
    s["words"] = _pages(most) // 2 + 1
    s["mask"], s["sees"] = None, None
    if case["tree"] == "tree":
        masks, sees = [], torch.zeros(batch, most, most, dtype=torch.bool)
        for b in range(batch):
            one = _tree(rng, int(rows[b]), "tree")
            masks.append(_pack(one, s["words"]))
            sees[b, : rows[b], : rows[b]] = torch.from_numpy(one)
        s["mask"], s["sees"] = torch.from_numpy(np.concatenate(masks)).cuda(), sees.cuda()
    return s


def _prepare_norm(case, gen, rng):
    rows, qh, kvh, dim, rot = (case[n] for n in ("rows", "qh", "kvh", "dim", "rot"))
    x = torch.randn(rows, qh + 2 * kvh, dim, generator=gen, device="cuda").mul_(torch.rand(rows, 1, 1, generator=gen, device="cuda").add_(0.3))
    x = x.to(TYPES[case["dtype"]])
    s = dict(case=dict(case), op="norm", rows=rows, qh=qh, kvh=kvh, dim=dim, rot=rot, dtype=x.dtype, qkv=x)
    s["q"], s["k"] = x[:, :qh], x[:, qh : qh + kvh]
    s["q_out"], s["k_out"] = (torch.empty(rows, h, dim, dtype=x.dtype, device="cuda") for h in (qh, kvh))
    s["q_weight"], s["k_weight"] = (torch.rand(dim, generator=gen, device="cuda").add_(0.5) for _ in range(2))
    s["inv_freq"] = torch.from_numpy((500000.0 ** (-np.arange(0, rot, 2) / rot)).astype(np.float32)).cuda()
    first = rng.integers(0, case["far"], max(1, rows // 512))  # pieces of 512 positions in a row, anywhere up to `far`
    pos = (first[np.minimum(np.arange(rows) // 512, len(first) - 1)] + np.arange(rows) % 512) % case["far"]
    (s["positions"],) = _ints(pos)
    return s


# ------------------------------------------------------------------ one pass


def run(s):
    if own:
        return {"pages": _own_pages, "norm": _own_norm, "rows": _own_rows, "attn": _own_attn}[s["op"]](s)
    return {"pages": _plain_pages, "norm": _plain_norm, "rows": _plain_rows, "attn": _plain_attn}[s["op"]](s)


def _ops():
    import opworks_b200

    return opworks_b200.ops_lib(), torch.cuda.current_stream().cuda_stream


def _own_pages(s):
    ops, stream = _ops()
    if s["case"]["way"] == "take":
        ops.page_take(s["ctx"], s["start"], s["batch"], s["total"], s["table"], s["stride"], s["free"], s["count"], s["positions"],
                      s["slots"], s["left"], s["status"], stream)
        return {"table": s["table"], "positions": s["positions"], "slots": s["slots"], "left": s["left"], "status": s["status"]}
    ops.page_give(s["old"], s["new"], s["batch"], s["table"], s["stride"], s["free"], s["blocks"], s["count"], s["left"],
                  s["status"], stream)
    return {"free": s["free"], "left": s["left"], "status": s["status"]}


def _own_norm(s):
    ops, stream = _ops()
    row = (s["qh"] + 2 * s["kvh"]) * s["dim"]
    ops.qk_norm_rope(s["q"], row, s["k"], row, TYPE_CODES[s["case"]["dtype"]], s["q_weight"], s["k_weight"], EPS, s["positions"],
                     s["inv_freq"], s["rot"], s["rows"], s["qh"], s["kvh"], s["dim"], s["q_out"], s["qh"] * s["dim"], s["k_out"],
                     s["kvh"] * s["dim"], stream)
    return {"q": s["q_out"], "k": s["k_out"]}


def _own_rows(s):
    ops, stream = _ops()
    kind = TYPE_CODES[s["case"]["dtype"]]
    if s["case"]["way"] == "store":
        ops.kv4_write(s["k"], s["k"].stride(0), s["v"], s["v"].stride(0), kind, s["pool"], s["blocks"], s["slots"], s["total"],
                      s["kvh"], s["dim"], stream)
    ops.kv4_read(s["pool"], s["blocks"], s["slots"], s["total"], s["kvh"], s["dim"], s["k_out"], s["width"], s["v_out"], s["width"],
                 kind, stream)
    return {"k": s["k_out"], "v": s["v_out"]}


def _own_attn(s):
    ops, stream = _ops()
    row = s["qh"] * s["dim"]
    ops.tree_attention_q4(s["q"], TYPE_CODES[s["case"]["dtype"]], row, s["pool"], s["table"], s["stride"], s["ctx"], s["start"],
                          s["mask"], s["words"], s["batch"], s["total"], s["most"], s["most_ctx"], s["qh"], s["kvh"], s["dim"],
                          s["scale"], s["out"], row, stream)
    return s["out"]


def _before(n):
    return torch.cumsum(n, 0) - n


def _plain_pages(s):
    table, stride = s["table"], s["stride"]
    index = torch.arange(stride, device="cuda")
    if s["case"]["way"] == "take":
        ctx = s["ctx"].long()
        have = (ctx + PAGE - 1) // PAGE
        need = (ctx + s["start"].diff().long() + PAGE - 1) // PAGE - have
        total = need.sum()
        which = _before(need)[:, None] + index - have[:, None]  # the how-manieth page taken
        new = (index >= have[:, None]) & (index < (have + need)[:, None])
        at = (s["count"].long() - 1 - which).clamp(0, s["blocks"] - 1)
        table.copy_(torch.where(new, s["free"][at], table))
        pos = ctx[s["owner"]] + s["node"]
        slots = table.long()[s["owner"], pos // PAGE] * PAGE + pos % PAGE
        return {"table": table, "positions": pos.int(), "slots": slots, "left": (s["count"] - total).int(),
                "status": torch.zeros_like(s["status"])}
    old, new = ((s[n].long() + PAGE - 1) // PAGE for n in ("old", "new"))
    gone = (old - new).clamp_min(0)
    ends = (index >= new[:, None]) & (index < old[:, None])
    to = torch.where(ends, s["count"].long() + _before(gone)[:, None] + index - new[:, None], s["blocks"])
    free = torch.cat([s["free"], s["free"][:1]]).scatter_(0, to.flatten(), table.flatten())[:-1]
    return {"free": free, "left": (s["count"] + gone.sum()).int(), "status": torch.zeros_like(s["status"])}


def _plain_norm(s):
    half = s["rot"] // 2
    angle = s["positions"].double()[:, None, None] * s["inv_freq"].double()
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    out = {}
    for name in ("q", "k"):
        x = s[name].float()
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * s[name + "_weight"]
        a, b = x[..., :half], x[..., half : 2 * half]
        out[name] = torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * half :]], -1).to(s["dtype"])
    return out


def _places(s):
    return torch.div(s["slots"], PAGE, rounding_mode="floor"), s["slots"] % PAGE


def _plain_rows(s):
    at = _places(s)
    kc, vc, ks, vs = _views(s["pool"], s["dim"])
    if s["case"]["way"] == "store":
        _store(kc, ks, at, s["k"].unflatten(-1, (s["kvh"], s["dim"])))
        _store(vc, vs, at, s["v"].unflatten(-1, (s["kvh"], s["dim"])))
    return {"k": _fetch(kc, ks, at).flatten(1).to(s["dtype"]), "v": _fetch(vc, vs, at).flatten(1).to(s["dtype"])}


def _plain_keys(s, pages):
    """K and V of all sequences, [batch, kvh, pages * 16, D] in fp32."""
    kc, vc, ks, vs = _views(s["pool"][s["table"][:, :pages].long()], s["dim"])
    out = []
    for codes, scales in ((kc, ks), (vc, vs)):
        c = codes.to(torch.int8)  # [batch, pages, kvh, G, 16, 16 bytes]
        c = torch.stack([c & 15, (c >> 4) & 15], -1).flatten(-2).float().sub_(8.0).mul_(scales.float()[..., None])
        out.append(c.permute(0, 2, 1, 4, 3, 5).flatten(4).flatten(2, 3))
    return out


def _plain_attn(s):
    batch, most, kvh, dim = s["batch"], s["most"], s["kvh"], s["dim"]
    rep = s["qh"] // kvh
    ctx, rows = _counts(s["case"])  # a user's program knows its lengths
    k, v = _plain_keys(s, int(_pages(ctx + rows).max()))
    keys = k.shape[2]
    node = torch.arange(keys, device="cuda") - s["ctx"].long()[:, None]  # that a key belongs to; below zero: the context
    if s["sees"] is None:
        hidden = node[:, None, :] > torch.arange(most, device="cuda")[:, None]
    else:
        hidden = (node >= 0)[:, None, :] & ~s["sees"].gather(2, node.clamp(0, most - 1)[:, None, :].expand(-1, most, -1))
        hidden |= (node >= most)[:, None, :]
    q = torch.zeros(batch, most, s["qh"], dim, device="cuda")
    q[s["owner"], s["node"]] = s["q"].float()
    q = q.view(batch, most, kvh, rep, dim).permute(0, 2, 3, 1, 4).reshape(batch, kvh, rep * most, dim)
    p = torch.matmul(q, k.transpose(2, 3)).mul_(s["scale"]).view(batch, kvh, rep, most, keys)
    p.masked_fill_(hidden[:, None, None], -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True).clamp_min(-3e38)).exp_()
    total = p.sum(-1, keepdim=True).clamp_min(1e-38)
    o = torch.matmul(p.view(batch, kvh, rep * most, keys), v).view(batch, kvh, rep, most, dim) / total
    return o.permute(0, 3, 1, 2, 4).reshape(batch, most, s["qh"], dim)[s["owner"], s["node"]].to(s["dtype"])


# ------------------------------------------------------------------ 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    return {"pages": _exact_pages, "norm": _exact_norm, "rows": _exact_rows, "attn": _exact_attn}[s["op"]](s)


def _exact_pages(s):
    """By a loop over the sequences, as an allocator on the host would do it."""
    table, free, count = s["table"].cpu().numpy().copy(), s["free"].cpu().numpy().copy(), int(s["count"])
    if s["case"]["way"] == "take":
        ctx, start = s["ctx"].tolist(), s["start"].tolist()
        positions, slots = [], []
        for b in range(s["batch"]):
            end = ctx[b] + start[b + 1] - start[b]
            for page in range(_pages(ctx[b]), _pages(end)):
                count -= 1
                table[b, page] = free[count]
            pos = np.arange(ctx[b], end)
            positions.append(pos)
            slots.append(table[b, pos // PAGE].astype(np.int64) * PAGE + pos % PAGE)
        return {"table": torch.from_numpy(table), "positions": torch.from_numpy(np.concatenate(positions).astype(np.int32)),
                "slots": torch.from_numpy(np.concatenate(slots)), "left": torch.tensor([count], dtype=torch.int32),
                "status": torch.zeros(1, dtype=torch.int32)}
    old, new = s["old"].tolist(), s["new"].tolist()
    for b in range(s["batch"]):
        for page in range(_pages(new[b]), _pages(old[b])):
            free[count] = table[b, page]
            count += 1
    return {"free": torch.from_numpy(free), "left": torch.tensor([count], dtype=torch.int32), "status": torch.zeros(1, dtype=torch.int32)}


def _exact_norm(s):
    rot, out = s["rot"], {}
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["positions"].double()[:, None] * s["inv_freq"].double()[None])
    for name in ("q", "k"):
        x = s[name].double()
        y = x / torch.linalg.vector_norm(x, dim=-1, keepdim=True).square().div(s["dim"]).add(EPS).sqrt() * s[name + "_weight"].double()
        z = torch.complex(y[..., : rot // 2], y[..., rot // 2 : rot]) * turn[:, None]
        y[..., : rot // 2], y[..., rot // 2 : rot] = z.real, z.imag
        out[name] = y
    return out


def _exact_rows(s):
    if s["case"]["way"] == "fetch":
        return {n: _exact_tokens(s, i, s["slots"]).flatten(1) for i, n in enumerate(("k", "v"))}
    out = {}
    for name in ("k", "v"):
        x = s[name].double().view(s["total"], -1, GROUP) if s[name].is_contiguous() else s[name].double().reshape(s["total"], -1, GROUP)
        want = torch.linalg.vector_norm(x, ord=math.inf, dim=-1) / 7.0
        unit = torch.exp2((torch.floor(torch.log2(want.clamp_min(2.0**-100))) - 4).clamp_min(-24))  # of a scale's last bit
        scale = (torch.round(want / unit) * unit)[..., None]
        out[name] = (torch.round(x / scale.clamp_min(2.0**-200)).clamp(-7, 7) * scale).view(s["total"], s["width"])
    return out


def _exact_tokens(s, which, slots):
    """K (0) or V (1) rows at `slots`, [n, kvh, D] in 64 bits, from the record's bytes."""
    g = s["dim"] // GROUP
    block, place = torch.div(slots, PAGE, rounding_mode="floor"), slots % PAGE
    rec = s["pool"][block].long()  # [n, kvh, record]
    byte = (which * g * 256 + torch.arange(g, device="cuda")[None, :, None] * 256 + place[:, None, None] * 16
            + torch.arange(16, device="cuda")[None, None, :]).flatten(1)
    c = rec.gather(2, byte[:, None, :].expand(-1, rec.shape[1], -1))
    c = torch.stack([c % 16, c // 16], -1).flatten(2).double() - 8
    at = 2 * g * 256 + which * g * 32 + torch.arange(g, device="cuda")[None, :] * 32 + place[:, None] * 2
    lo, hi = (rec.gather(2, (at + i)[:, None, :].expand(-1, rec.shape[1], -1)) for i in (0, 1))
    bits = lo + 256 * hi
    exponent, fraction = (bits >> 10) & 31, (bits & 1023).double()
    scale = torch.where(exponent == 0, fraction * 2.0**-24, (1024.0 + fraction) * torch.exp2((exponent - 25).double()))
    return c * scale.repeat_interleave(GROUP, 2)


def _exact_attn(s):
    rep, start, ctx = s["qh"] // s["kvh"], s["start"].tolist(), s["ctx"].tolist()
    out = torch.empty(s["total"], s["qh"], s["dim"], dtype=torch.float64, device="cuda")
    for b in range(s["batch"]):
        lo, n = start[b], start[b + 1] - start[b]
        pos = torch.arange(ctx[b] + n, device="cuda")
        slots = s["table"][b].long()[pos // PAGE] * PAGE + pos % PAGE
        k, v = (torch.cat([_exact_tokens(s, i, part) for part in slots.split(4096)]) for i in (0, 1))
        hidden = torch.zeros(n, ctx[b] + n, dtype=torch.bool, device="cuda")
        hidden[:, ctx[b] :] = ~s["sees"][b, :n, :n] if s["sees"] is not None else torch.ones(n, n, dtype=torch.bool, device="cuda").triu_(1)
        for h in range(s["kvh"]):
            for i in range(0, n, 512):
                q = s["q"][lo + i : lo + min(i + 512, n), h * rep : (h + 1) * rep].double()
                w = (torch.einsum("nrd,kd->nrk", q, k[:, h]) * s["scale"]).masked_fill(hidden[i : i + 512, None], -math.inf)
                out[lo + i : lo + i + q.shape[0], h * rep : (h + 1) * rep] = torch.einsum("nrk,kd->nrd", torch.softmax(w, -1), v[:, h])
    return out
