"""Serving operators of the paged KV cache: their workloads and plain forms.

Operators that work together around an 8-bit paged cache:

  rope     rotary positions of query and key rows (and their gradient)
  append   rotary positions, then K and V quantised into int8 pages
  attend   causal attention of several new tokens per sequence over int8 pages
  fork     fork sequences, reserve pages for their next tokens, free them
  compact  move the live pages of a fragmented pool to its front

`run` computes one pass: with `own` false in elementary torch operations, with
`own` true through the kvx package.  `exact` computes the same from the
definitions in 64 bits.
"""
import math
import random

import torch

own = False

HEAD_DIM, PAGE = 128, 16


# ------------------------------------------------------------------- cases ---

def listed():
    return [
        # one decode step of 64 sequences, 28-layer 3B geometry, q and k as views of the packed projection
        dict(name="rope 64 tokens", op="rope", tokens=64, hq=24, hkv=8, dim=128, rotary=128, layout="half", scaling="llama3",
             dtype="f16", inverse=False, packed=True, far=131072),
        # gradient of the rotation over a long training or scoring batch, part of the head rotated
        dict(name="rope gradient 8191 tokens", op="rope", tokens=8191, hq=64, hkv=8, dim=128, rotary=64, layout="interleaved",
             scaling="yarn", dtype="f32", inverse=True, packed=False, far=65536),
        # one decode step: 32 sequences append one token each
        dict(name="append 32 x 1", op="append", batch=32, new=1, ragged=False, ctx=8192, hq=24, hkv=8, rotary=128, layout="half",
             scaling="llama3", dtype="f16", shape=11),
        # prompt chunks of several requests with odd lengths, 70B geometry
        dict(name="append 6 ragged chunks", op="append", batch=6, new=2731, ragged=True, ctx=4096, hq=64, hkv=8, rotary=128,
             layout="half", scaling="none", dtype="f16", shape=12),
        # checking 5 drafted tokens of 8 sequences over long contexts
        dict(name="attend 8 x 5 verify", op="attend", batch=8, new=5, ragged=False, ctx=8192, hq=24, hkv=8, dtype="f16", shape=21),
        # one short prompt of odd length, nothing cached before it
        dict(name="attend 1 x 1001 prompt", op="attend", batch=1, new=1001, ragged=False, ctx=0, hq=24, hkv=8, dtype="f16", shape=22),
        # ragged chunks with contexts of their own, 70B heads, 32-bit queries and outputs
        dict(name="attend 4 ragged f32", op="attend", batch=4, new=300, ragged=True, ctx=4096, hq=64, hkv=8, dtype="f32", shape=23),
        # the last chunk of a 32k prompt
        dict(name="attend 1 x 4096 on 28672", op="attend", batch=1, new=4096, ragged=False, ctx=28672, hq=24, hkv=8, dtype="f16",
             shape=24),
        # 4 more samples of a running request
        dict(name="fork 4 i8", op="fork", rows=16, forks=4, num_pages=1024, layers=28, hkv=8, pool="i8", ctx=700, shape=31),
        # beams of a large batch
        dict(name="fork 96 f16", op="fork", rows=256, forks=96, num_pages=4096, layers=8, hkv=8, pool="f16", ctx=400, shape=32),
        # a small pool after a few requests have left
        dict(name="compact 257 pages", op="compact", rows=8, num_pages=257, live=101, layers=28, hkv=8, pool="i8", shape=41),
        # a pool that is one third live, before its rear part is given back
        dict(name="compact 6000 pages", op="compact", rows=64, num_pages=6000, live=2000, layers=4, hkv=8, pool="f16", shape=42),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("rope", "append", "attend", "fork", "compact"))
    shape = rng.randrange(1 << 20)
    hq, hkv = rng.choice(((24, 8), (64, 8), (8, 8), (16, 2), (21, 3)))
    layout, scaling = rng.choice(("half", "interleaved")), rng.choice(("none", "linear", "ntk", "llama3", "yarn"))
    dtype = rng.choice(("f16", "f16", "f32"))
    if op == "rope":
        dim = rng.choice((64, 80, 96, 128, 128, 192, 256))
        rotary = rng.choice((dim, dim, dim // 2, dim // 4))
        return dict(op=op, tokens=_log(rng, 1, 8192), hq=hq, hkv=hkv, dim=dim, rotary=rotary // 2 * 2, layout=layout, scaling=scaling,
                    dtype=dtype, inverse=rng.random() < 0.3, packed=rng.random() < 0.5, far=_log(rng, 1000, 1000000))
    if op == "append":
        batch = _log(rng, 1, 64)
        return dict(op=op, batch=batch, new=_log(rng, 1, max(1, 12288 // batch)), ragged=rng.random() < 0.6, ctx=_log(rng, 1, 32768),
                    hq=hq, hkv=hkv, rotary=rng.choice((128, 128, 64, 32)), layout=layout, scaling=scaling, dtype=dtype, shape=shape)
    if op == "attend":
        batch = _log(rng, 1, 16)
        ctx = rng.choice((0, _log(rng, 1, 16384)))
        new = _log(rng, 1, 2048)
        while batch * hq * new * (ctx + new) > 24 * 2048 * 16384:
            new = max(1, new // 2)
            batch = max(1, batch * 3 // 4)
        return dict(op=op, batch=batch, new=new, ragged=rng.random() < 0.6, ctx=ctx, hq=hq, hkv=hkv, dtype=dtype, shape=shape)
    pool = rng.choice(("f16", "i8"))
    if op == "fork":
        rows = _log(rng, 4, 256)
        ctx = _log(rng, 1, 600)
        forks = rng.randint(1, max(1, rows // 2 - 1))
        return dict(op=op, rows=rows, forks=forks, num_pages=rows * (ctx // PAGE + 3) + rng.randrange(64), layers=rng.choice((1, 4, 8)),
                    hkv=rng.choice((1, 4)), pool=pool, ctx=ctx, shape=shape)
    num_pages = _log(rng, 16, 6000)
    return dict(op=op, rows=rng.randint(1, 64), num_pages=num_pages, live=rng.randint(1, num_pages), layers=rng.choice((1, 2, 4)),
                hkv=rng.choice((1, 8)), pool=pool, shape=shape)


def _lens(case):
    """(cached tokens, new tokens) of each sequence, from the case alone."""
    r = random.Random(case["shape"])
    ctx, new = [], []
    for _ in range(case["batch"]):
        ctx.append(r.randint(case["ctx"] // 4, case["ctx"]) if case["batch"] > 1 else case["ctx"])
        new.append(r.randint(0, case["new"]) if case["ragged"] else case["new"])
    new[-1] = case["new"]  # the longest is always there
    return ctx, new


def _torch_dtype(case):
    return torch.float16 if case["dtype"] == "f16" else torch.float32


# ------------------------------------------------------- rotary frequencies ---

def _rope_config(case):
    return dict(rotary_dim=case["rotary"], base=500000.0, scaling=case["scaling"], factor=1.0 if case["scaling"] == "none" else 8.0,
                low=1.0, high=4.0 if case["scaling"] == "llama3" else 32.0, original_context=8192.0)


def _frequencies(cfg):
    """Angle per position of each rotated pair (64 bits), and the factor on cos and sin."""
    d, base, factor, low, high, ctx = (cfg[k] for k in ("rotary_dim", "base", "factor", "low", "high", "original_context"))
    i = torch.arange(d // 2, dtype=torch.float64)
    kind = cfg["scaling"]
    if kind == "ntk" and d > 2:
        base = base * factor ** (d / (d - 2))
    inv = base ** (-2.0 * i / d)
    if kind == "linear":
        return inv / factor, 1.0
    if kind == "llama3":
        mix = ((ctx * inv / (2 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
        return (1 - mix) * inv / factor + mix * inv, 1.0
    if kind == "yarn":
        first = max(math.floor(d * math.log(ctx / (high * 2 * math.pi)) / (2 * math.log(base))), 0)
        last = min(math.ceil(d * math.log(ctx / (low * 2 * math.pi)) / (2 * math.log(base))), d - 1)
        ramp = ((i - first) / max(last - first, 0.001)).clamp(0.0, 1.0)
        return inv * (1 - ramp) + inv / factor * ramp, 0.1 * math.log(factor) + 1.0
    return inv, 1.0


def _rotate(x, cos, sin, rotary, layout):
    """x [tokens][heads][dim] with cos, sin [tokens][1][rotary / 2]."""
    r = x[..., :rotary]
    if layout == "half":
        a, b = r[..., : rotary // 2], r[..., rotary // 2:]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    else:
        a, b = r[..., 0::2], r[..., 1::2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    return torch.cat((y, x[..., rotary:]), -1)


def _rotate32(s, x, pos, inverse=False):
    """32-bit rotation; the angles of far positions need 64."""
    ang = pos.double()[:, None, None] * s["inv"]
    cos, sin = (ang.cos() * s["amp"]).float(), (ang.sin() * s["amp"]).float()
    return _rotate(x.float(), cos, -sin if inverse else sin, s["rotary"], s["layout"])


def _rope_state(case, s):
    cfg = _rope_config(case)
    inv, amp = _frequencies(cfg)
    s.update(inv=inv.cuda(), amp=amp, rotary=case["rotary"], layout=case["layout"])
    if own:  # the table that a program makes once for a model
        import kvx
        s["table"] = kvx.rope_table(cfg["rotary_dim"], base=cfg["base"], layout=case["layout"], scaling=cfg["scaling"],
                                    factor=cfg["factor"], low=cfg["low"], high=cfg["high"], original_context=cfg["original_context"])
    return s


# ------------------------------------------------------------------ inputs ---

def _kvx_path():
    import os
    import sys
    p = os.path.join(os.getcwd(), "adaptive-hierarchical-llm-inference-engine_b200")
    if p not in sys.path:
        sys.path.insert(0, p)


def prepare(case, seed):
    if own:
        _kvx_path()
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return _PREPARE[case["op"]](case, seed, g)


def _normal(g, shape, dtype=torch.float16):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _quantise(x):
    """The cache's int8 form of blocks [...][16][128]: codes and {min, max, scale, zero point} of each block."""
    x = x.float()
    lo, hi = x.amin((-2, -1)), x.amax((-2, -1))
    scale = (hi - lo) / 255
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    codes = ((x - lo[..., None, None]) / scale[..., None, None] + 0.5).floor().clamp(0, 255) - 128
    return codes.to(torch.int8), torch.stack((lo, hi, scale, lo), -1)


def _values(codes, stats, dtype=torch.float32):
    """What int8 blocks [...][16][128] stand for."""
    return (stats[..., 3, None, None] + (codes.float() + 128) * stats[..., 2, None, None]).to(dtype)


def _prepare_rope(case, seed, g):
    t, hq, hkv, dim, dtype = case["tokens"], case["hq"], case["hkv"], case["dim"], _torch_dtype(case)
    qkv = _normal(g, (t, hq + 2 * hkv, dim), dtype)
    q, k = qkv[:, :hq], qkv[:, hq:hq + hkv]
    if not case["packed"]:
        q, k = q.contiguous(), k.contiguous()
    pos = torch.randint(0, case["far"], (t,), generator=g, device="cuda", dtype=torch.int32)
    s = dict(op="rope", q=q, k=k, pos=pos, inverse=case["inverse"], qo=torch.empty(q.shape, dtype=dtype, device="cuda"),
             ko=torch.empty(k.shape, dtype=dtype, device="cuda"))
    return _rope_state(case, s)


def _ragged(case):
    ctx, new = _lens(case)
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    seq = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new)).cuda()
    positions, q_start = torch.tensor(ctx, dtype=torch.int32).cuda(), torch.tensor(start, dtype=torch.int32).cuda()
    pos = positions[seq] + torch.arange(start[-1], device="cuda", dtype=torch.int32) - q_start[seq]
    return ctx, new, start, seq, positions, q_start, pos


def _prepare_append(case, seed, g):
    """Only the pages that the new tokens fall into are here: the append touches no others."""
    ctx, new, start, seq, positions, q_start, pos = _ragged(case)
    total, hq, hkv, dtype = start[-1], case["hq"], case["hkv"], _torch_dtype(case)
    max_pages = max((c + n + PAGE - 1) // PAGE for c, n in zip(ctx, new)) + 1
    spans = [(c // PAGE, (c + n + PAGE - 1) // PAGE if n else c // PAGE) for c, n in zip(ctx, new)]
    num_pages = sum(b - a for a, b in spans) + 3
    ids = list(range(num_pages))
    random.Random(seed).shuffle(ids)
    table = torch.full((case["batch"], max_pages), -1, dtype=torch.int32)
    used = 0
    for row, (a, b) in enumerate(spans):
        table[row, a:b] = torch.tensor(ids[used:used + b - a], dtype=torch.int32)
        used += b - a
    codes, stats = _quantise(_normal(g, (num_pages, 2, hkv, PAGE, HEAD_DIM)))
    qkv = _normal(g, (total, hq + 2 * hkv, HEAD_DIM), dtype)
    s = dict(op="append", pool=codes, stats=stats, table_=table.cuda(), q_start=q_start, positions=positions, seq=seq, pos=pos,
             q=qkv[:, :hq], k=qkv[:, hq:hq + hkv], v=qkv[:, hq + hkv:], qo=torch.empty((total, hq, HEAD_DIM), dtype=dtype, device="cuda"),
             values=torch.empty(codes.shape, dtype=torch.float16, device="cuda"))
    return _rope_state(case, s)


def _prepare_attend(case, seed, g):
    ctx, new, start, seq, positions, q_start, pos = _ragged(case)
    hq, hkv, dtype = case["hq"], case["hkv"], _torch_dtype(case)
    pages = [(c + n + PAGE - 1) // PAGE for c, n in zip(ctx, new)]
    max_pages, num_pages = max(max(pages), 1), sum(pages) + 1
    perm = torch.randperm(num_pages, generator=g, device="cuda").int().cpu()
    table = torch.full((case["batch"], max_pages), -1, dtype=torch.int32)
    used = 0
    for row, n in enumerate(pages):
        table[row, :n] = perm[used:used + n]
        used += n
    codes = torch.empty((num_pages, 2, hkv, PAGE, HEAD_DIM), dtype=torch.int8, device="cuda")
    stats = torch.empty((num_pages, 2, hkv, 4), dtype=torch.float32, device="cuda")
    for a in range(0, num_pages, 4096):
        codes[a:a + 4096], stats[a:a + 4096] = _quantise(_normal(g, (min(4096, num_pages - a), 2, hkv, PAGE, HEAD_DIM)))
    q = _normal(g, (start[-1], hq, HEAD_DIM), dtype)
    s = dict(op="attend", pool=codes, stats=stats, table_=table.cuda(), q_start=q_start, positions=positions, seq=seq, pos=pos, q=q,
             out=torch.empty_like(q), hkv=hkv, most=max(new))
    if own:  # scratch that a program keeps from step to step
        import kvx
        s["workspace"] = kvx.attend_chunk_workspace(case["batch"], start[-1], hq, hkv, max_pages)
    return s


def _pool(case, g, num_pages):
    shape = (case["layers"], num_pages, 2, case["hkv"], PAGE, HEAD_DIM)
    if case["pool"] == "i8":
        pool = torch.randint(-128, 128, shape, generator=g, device="cuda", dtype=torch.int8)
        return pool, torch.rand(shape[:4] + (4,), generator=g, device="cuda")
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float16), None


def _books(case, refs, table, lens):
    """The three arrays of the bookkeeping in one buffer, so that a pass can begin from the same state again."""
    flat = torch.cat((refs.flatten(), table.flatten(), lens.flatten())).int().cuda()
    a, b = refs.numel(), refs.numel() + table.numel()
    s = dict(flat=flat, saved=flat.clone(), refs=flat[:a], table_=flat[a:b].view(table.shape), lens=flat[b:])
    return s


def _handle(case, s):
    if own:  # the handle and scratch that a program keeps
        import kvx.pages
        pools = [s["pool"][i] for i in range(case["layers"])]
        stats = [s["stats"][i] for i in range(case["layers"])] if s["stats"] is not None else None
        s["pages"] = kvx.pages.Pages(s["refs"], s["table_"], s["lens"], pools, stats)
    return s


def _fork_lens(case):
    r = random.Random(case["shape"])
    live = case["rows"] - case["forks"]
    return [r.randint(max(1, case["ctx"] // 4), case["ctx"]) for _ in range(live)]


def _prepare_fork(case, seed, g):
    r = random.Random(seed)
    lens = _fork_lens(case)
    rows, live, forks = case["rows"], len(lens), case["forks"]
    max_pages = case["ctx"] // PAGE + 2
    ids = list(range(case["num_pages"]))
    r.shuffle(ids)
    table = torch.full((rows, max_pages), -1, dtype=torch.int32)
    refs = torch.zeros(case["num_pages"], dtype=torch.int32)
    order = list(range(rows))
    r.shuffle(order)
    all_lens, used = torch.zeros(rows, dtype=torch.int32), 0
    for row, n in zip(order[:live], lens):
        k = (n + PAGE - 1) // PAGE
        mine = torch.tensor(ids[used:used + k])
        table[row, :k], refs[mine], all_lens[row] = mine.int(), 1, n
        used += k
    parents = [order[r.randrange(live)] for _ in range(forks)]
    children = order[live:live + forks]
    pool, stats = _pool(case, g, case["num_pages"])
    grow = torch.ones(rows, dtype=torch.int32)
    s = dict(op="fork", pool=pool, stats=stats, parents=torch.tensor(parents, dtype=torch.int32).cuda(),
             children=torch.tensor(children, dtype=torch.int32).cuda(), grow=grow.cuda(),
             gone=torch.tensor(children[::2], dtype=torch.int32).cuda(), **_books(case, refs, table, all_lens))
    return _handle(case, s)


def _prepare_compact(case, seed, g):
    r = random.Random(seed)
    n, live, rows = case["num_pages"], case["live"], case["rows"]
    ids = r.sample(range(n), live)
    refs = torch.zeros(n, dtype=torch.int32)
    refs[torch.tensor(ids)] = 1
    each = (live + rows - 1) // rows
    table = torch.full((rows, each), -1, dtype=torch.int32)
    table.view(-1)[:live] = torch.tensor(ids, dtype=torch.int32)
    if rows > 1:  # a prefix that two sequences share
        table[-1, 0] = table[0, 0]
        refs = torch.bincount(table[table >= 0].long(), minlength=n).int()
    lens = (table >= 0).sum(1).int() * PAGE
    pool, stats = _pool(case, g, n)
    s = dict(op="compact", pool=pool, stats=stats, live=torch.zeros(1, dtype=torch.int32, device="cuda"),
             **_books(case, refs, table, lens))
    return _handle(case, s)


# --------------------------------------------------------------------- run ---

def run(state):
    return (_RUN_OWN if own else _RUN)[state["op"]](state)


def _rope_plain(s):
    dtype = s["q"].dtype
    return tuple(_rotate32(s, x, s["pos"], s["inverse"]).to(dtype) for x in (s["q"], s["k"]))


def _rope_own(s):
    import kvx
    return kvx.rope(s["q"], s["k"], s["pos"], s["table"], q_out=s["qo"], k_out=s["ko"], inverse=s["inverse"])


def _append_plain(s):
    """Old rows of a page keep their codes where the block's range stays, else they are quantised anew."""
    pool, stats, pos, seq = s["pool"], s["stats"], s["pos"].long(), s["seq"]
    hkv = pool.shape[2]
    q = _rotate32(s, s["q"], pos).to(s["q"].dtype)
    rows = torch.stack((_rotate32(s, s["k"], pos), s["v"].float()), 1)  # [tokens][K, V][hkv][128]
    page = s["table_"][seq, pos // PAGE].long()
    slot = pos % PAGE
    where = torch.arange(pool.shape[0], device=pool.device)
    inf = torch.full((pool.shape[0], 2, hkv), float("inf"), device=pool.device)
    index = page[:, None, None].expand(-1, 2, hkv)
    lo = inf.scatter_reduce(0, index, rows.amin(-1), "amin")
    hi = (-inf).scatter_reduce(0, index, rows.amax(-1), "amax")
    touched = torch.zeros_like(where).index_add_(0, page, torch.ones_like(page)) > 0
    first = torch.full_like(where, PAGE).scatter_reduce(0, page, slot, "amin")  # rows before it were there
    old = (first > 0)[:, None, None]
    lo, hi = torch.where(old, torch.minimum(lo, stats[..., 0]), lo), torch.where(old, torch.maximum(hi, stats[..., 1]), hi)
    scale = (hi - lo) / 255
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    wide = lambda x: x[..., None, None]  # noqa: E731
    again = (((_values(pool, stats) - wide(lo)) / wide(scale) + 0.5).floor().clamp(0, 255) - 128).to(torch.int8)
    kept = (lo == stats[..., 0]) & (hi == stats[..., 1])
    requant = wide(touched[:, None, None] & ~kept) & (torch.arange(PAGE, device=pool.device)[:, None] < wide(first[:, None, None]))
    pool.copy_(torch.where(requant, again, pool))
    codes = ((rows - lo[page][..., None]) / scale[page][..., None] + 0.5).floor().clamp(0, 255) - 128
    pool[page, :, :, slot] = codes.to(torch.int8)
    stats.copy_(torch.where(touched[:, None, None, None], torch.stack((lo, hi, scale, lo), -1), stats))
    return q, _values(pool, stats, torch.float16), stats


def _append_own(s):
    import kvx
    kvx.rope_append(s["pool"], s["table_"], s["q_start"], s["positions"], s["k"], s["v"], q=s["q"], q_out=s["qo"], table=s["table"],
                    stats=s["stats"])
    kvx.decompress_int8(s["pool"], s["stats"], out=s["values"])
    return s["qo"], s["values"], s["stats"]


def _attend_plain(s):
    """Padded to the longest: keys [batch][hkv][keys][128], queries [batch][hkv][group * new][128]."""
    table, seq, pos, q, hkv, most = s["table_"], s["seq"], s["pos"], s["q"], s["hkv"], s["most"]
    batch, max_pages = table.shape
    hq = q.shape[1]
    at = table.clamp(min=0).long()
    kv = _values(s["pool"][at], s["stats"][at]).permute(2, 0, 3, 1, 4, 5).reshape(2, batch, hkv, max_pages * PAGE, HEAD_DIM)
    offset = torch.arange(q.shape[0], device=q.device) - s["q_start"].long()[seq]
    padded = torch.zeros((batch, most, hq, HEAD_DIM), device=q.device)
    padded[seq, offset] = q.float()
    rows = padded.view(batch, most, hkv, hq // hkv, HEAD_DIM).permute(0, 2, 3, 1, 4).reshape(batch, hkv, hq // hkv * most, HEAD_DIM)
    score = rows @ kv[0].transpose(-1, -2)
    score = score.mul_(1 / math.sqrt(HEAD_DIM)).view(batch, hq, most, -1)
    last = s["positions"][:, None] + torch.arange(most, device=q.device)  # the key that each query still sees
    score.masked_fill_(torch.arange(max_pages * PAGE, device=q.device) > last[:, None, :, None], float("-inf"))
    score = score.sub_(score.amax(-1, keepdim=True)).exp_()
    total = score.sum(-1, keepdim=True)
    out = score.view(batch, hkv, hq // hkv * most, -1) @ kv[1]
    out = (out.view(batch, hq, most, HEAD_DIM) / total).transpose(1, 2)
    return out[seq, offset].to(q.dtype)


def _attend_own(s):
    import kvx
    return kvx.attend_chunk(s["pool"], s["table_"], s["q_start"], s["positions"], s["q"], stats=s["stats"], out=s["out"],
                            workspace=s["workspace"])


def _lowest_free(refs, need):
    """For every True of `need`, in order, the next lowest page that nobody holds (0 elsewhere)."""
    free = torch.argsort((refs > 0).int(), stable=True)
    rank = need.int().flatten().cumsum(0) - 1
    return torch.where(need, free[rank.clamp(min=0)].view(need.shape), torch.zeros_like(rank).view(need.shape))


def _fork_plain(s):
    refs, table, lens, parents, children = s["refs"], s["table_"], s["lens"], s["parents"].long(), s["children"].long()
    s["flat"].copy_(s["saved"])
    column = torch.arange(table.shape[1], device=table.device)
    plen = lens[parents].long()
    full, tail = plen // PAGE, plen % PAGE > 0
    rows = table[parents]
    share = column < full[:, None]
    new = _lowest_free(refs, tail)
    source = rows.gather(1, full.clamp(max=table.shape[1] - 1)[:, None])[:, 0].long()
    refs.index_add_(0, rows.clamp(min=0).long().flatten(), share.int().flatten())
    refs.index_add_(0, new, tail.int())
    rows = torch.where(share, rows, -1)
    table[children] = torch.where(tail[:, None] & (column == full[:, None]), new[:, None].int(), rows)
    lens[children] = plen.int()
    source, new = source[tail], new[tail]
    s["pool"][:, new] = s["pool"][:, source]
    if s["stats"] is not None:
        s["stats"][:, new] = s["stats"][:, source]
    # pages for each sequence's next token
    have, want = (lens.long() + PAGE - 1) // PAGE, (lens.long() + s["grow"] + PAGE - 1) // PAGE
    need = (column >= have[:, None]) & (column < want[:, None])
    got = _lowest_free(refs, need)
    refs.index_add_(0, got.flatten(), need.int().flatten())
    table.copy_(torch.where(need, got.int(), table))
    forked = s["flat"].clone()
    # some of the samples end
    gone = s["gone"].long()
    rows = table[gone]
    refs.index_add_(0, rows.clamp(min=0).long().flatten(), -(rows >= 0).int().flatten())
    table[gone] = -1
    lens[gone] = 0
    return forked, refs, table, lens, s["pool"], s["stats"]


def _fork_own(s):
    s["flat"].copy_(s["saved"])
    pages = s["pages"]
    pages.fork(s["parents"], s["children"])
    pages.reserve(s["grow"])
    forked = s["flat"].clone()
    pages.free(s["gone"])
    return forked, s["refs"], s["table_"], s["lens"], s["pool"], s["stats"]


def _compact_plain(s):
    s["flat"].copy_(s["saved"])
    refs, table = s["refs"], s["table_"]
    held = refs > 0
    count = held.sum()
    page = torch.arange(refs.numel(), device=refs.device)
    source = (held & (page >= count)).nonzero()[:, 0]
    to = (~held & (page < count)).nonzero()[:, 0]
    s["pool"][:, to] = s["pool"][:, source]
    if s["stats"] is not None:
        s["stats"][:, to] = s["stats"][:, source]
    refs[to] = refs[source]
    refs[source] = 0
    at = page.int()
    at[source] = to.int()
    table.copy_(torch.where(table >= 0, at[table.clamp(min=0).long()], table))
    return count.int().view(1), refs, table, s["pool"], s["stats"]


def _compact_own(s):
    s["flat"].copy_(s["saved"])
    s["pages"].compact(num_live=s["live"])
    return s["live"], s["refs"], s["table_"], s["pool"], s["stats"]


_PREPARE = dict(rope=_prepare_rope, append=_prepare_append, attend=_prepare_attend, fork=_prepare_fork, compact=_prepare_compact)
_RUN = dict(rope=_rope_plain, append=_append_plain, attend=_attend_plain, fork=_fork_plain, compact=_compact_plain)
_RUN_OWN = dict(rope=_rope_own, append=_append_own, attend=_attend_own, fork=_fork_own, compact=_compact_own)


# -------------------------------------------------------------------- work ---

def work(case):
    op = case["op"]
    size = 2 if case.get("dtype") == "f16" else 4
    if op == "rope":
        rows = case["tokens"] * (case["hq"] + case["hkv"])
        return dict(bytes=2 * rows * case["dim"] * size + 4 * case["tokens"], flops=3 * rows * case["rotary"])
    if op in ("append", "attend"):
        ctx, new = _lens(case)
        total, hq, hkv = sum(new), case["hq"], case["hkv"]
    if op == "append":
        pages = sum((c + n + PAGE - 1) // PAGE - c // PAGE for c, n in zip(ctx, new) if n)
        # q, k, v read, q written, the pages written and read back as 16-bit values, the statistics
        block = pages * 2 * hkv * PAGE * HEAD_DIM
        return dict(bytes=total * HEAD_DIM * size * (2 * hq + 2 * hkv) + 4 * block + pages * 2 * hkv * 32,
                    flops=total * HEAD_DIM * (3 * hq + 7 * hkv))
    if op == "attend":
        keys = sum(c + n for c, n in zip(ctx, new) if n)
        pairs = sum(n * c + n * (n + 1) // 2 for c, n in zip(ctx, new))
        return dict(bytes=keys * hkv * 2 * (HEAD_DIM + 1) + 2 * total * hq * HEAD_DIM * size, flops=4 * HEAD_DIM * hq * pairs)
    page = 2 * case["hkv"] * PAGE * HEAD_DIM * (2 if case["pool"] == "f16" else 1) + (32 * case["hkv"] if case["pool"] == "i8" else 0)
    if op == "fork":
        # nearly every parent ends inside a page, which is copied; the tables are read and written
        return dict(bytes=2 * case["forks"] * page * case["layers"] + 8 * (case["num_pages"] + case["rows"] * (case["ctx"] // PAGE + 3)),
                    flops=0)
    moved = case["live"] * (1 - case["live"] / case["num_pages"])
    return dict(bytes=2 * moved * page * case["layers"] + 8 * (case["num_pages"] + case["live"]), flops=0)


# ------------------------------------------------------------------- exact ---

def exact(case, seed):
    if case["op"] in ("fork", "compact"):
        return None  # nothing is computed: whole numbers and copies
    s = prepare(case, seed)
    return dict(rope=_rope_exact, append=_append_exact, attend=_attend_exact)[case["op"]](case, s)


def _turn(case, x, pos, sign=1.0):
    """Rotation as a product with e^(i angle), in 64 bits."""
    inv, amp = _frequencies(_rope_config(case))
    d = case["rotary"]
    turn = torch.polar(torch.full((1, 1), amp, dtype=torch.float64, device=x.device).expand(len(pos), d // 2),
                       sign * pos.double()[:, None] * inv.to(x.device))[:, None]
    x = x.double()
    pairs = x[..., :d].unflatten(-1, (2, d // 2)).transpose(-1, -2) if case["layout"] == "half" else x[..., :d].unflatten(-1, (d // 2, 2))
    y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    y = y.transpose(-1, -2).flatten(-2) if case["layout"] == "half" else y.flatten(-2)
    return torch.cat((y, x[..., d:]), -1)


def _rope_exact(case, s):
    return tuple(_turn(case, x, s["pos"], -1.0 if case["inverse"] else 1.0) for x in (s["q"], s["k"]))


def _append_exact(case, s):
    k, v = _turn(case, s["k"], s["pos"]), s["v"].double()
    ctx, new = _lens(case)
    table, begin = s["table_"].cpu(), s["q_start"].cpu().tolist()
    stats = s["stats"].double()
    values = stats[..., 3, None, None] + (s["pool"].double() + 128) * stats[..., 2, None, None]
    for row in range(case["batch"]):
        at = ctx[row]
        while at < ctx[row] + new[row]:
            page, slot = int(table[row, at // PAGE]), at % PAGE
            n = min(PAGE - slot, ctx[row] + new[row] - at)
            a = begin[row] + at - ctx[row]
            fresh = torch.stack((k[a:a + n], v[a:a + n])).transpose(1, 2)  # [K, V][hkv][n][128]
            lo, hi = fresh.amin((-1, -2)), fresh.amax((-1, -2))
            if slot:
                lo, hi = torch.minimum(lo, stats[page, ..., 0]), torch.maximum(hi, stats[page, ..., 1])
            scale = (hi - lo) / 255
            scale[scale == 0] = 1
            lo_, scale_ = lo[..., None, None], scale[..., None, None]
            near = lambda x: lo_ + ((x - lo_) / scale_ + 0.5).floor().clamp(0, 255) * scale_  # noqa: E731, B023
            if slot:
                same = ((lo == stats[page, ..., 0]) & (hi == stats[page, ..., 1]))[..., None, None]
                values[page, :, :, :slot] = torch.where(same, values[page, :, :, :slot], near(values[page, :, :, :slot]))
            values[page, :, :, slot:slot + n] = near(fresh)
            behind = slice(slot + n, PAGE)  # codes left as they were stand for other values in another range
            codes = s["pool"][page, :, :, behind].double() + 128
            values[page, :, :, behind] = lo_ + codes * scale_
            stats[page] = torch.stack((lo, hi, scale, lo), -1)
            at += n
    return _turn(case, s["q"], s["pos"]), values, stats


def _attend_exact(case, s):
    ctx, new = _lens(case)
    hq, hkv = case["hq"], case["hkv"]
    if 4 * HEAD_DIM * hq * sum(n * (c + n) for c, n in zip(ctx, new)) > 6e12:
        return None
    group, begin = hq // hkv, s["q_start"].cpu().tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for row in range(case["batch"]):
        n, keys = new[row], ctx[row] + new[row]
        if not n:
            continue
        pages = s["table_"][row, : (keys + PAGE - 1) // PAGE].long()
        for h in range(hkv):
            st, codes = s["stats"][pages, :, h].double(), s["pool"][pages, :, h].double()
            kv = st[..., 3, None, None] + (codes + 128) * st[..., 2, None, None]
            k, v = kv[:, 0].reshape(-1, HEAD_DIM)[:keys], kv[:, 1].reshape(-1, HEAD_DIM)[:keys]
            for a in range(0, n, 1024):
                b = min(n, a + 1024)
                q = s["q"][begin[row] + a:begin[row] + b, h * group:(h + 1) * group].double()
                score = torch.einsum("tgd,kd->gtk", q, k) / math.sqrt(HEAD_DIM)
                seen = torch.arange(keys, device="cuda")[None] <= ctx[row] + torch.arange(a, b, device="cuda")[:, None]
                p = torch.softmax(score.masked_fill(~seen, -math.inf), -1)
                out[begin[row] + a:begin[row] + b, h * group:(h + 1) * group] = torch.einsum("gtk,kd->tgd", p, v)
    return out
