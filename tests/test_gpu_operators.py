"""GPU parity of the 8-bit serving operators against plain implementations in
64 bits: rotary positions, the rotated append into int8 / fp16 / fp32 pages,
attention of several new tokens over int8 pages, and the page bookkeeping.

Tolerances count roundings.  E16 = 2^-11 and E32 = 2^-24 are half a step of
fp16 and fp32, relative to the value.
"""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

E16, E32 = 2.0 ** -11, 2.0 ** -24
TINY16 = 2.0 ** -25  # half a step of fp16's subnormals
F16, F32, F64 = torch.float16, torch.float32, torch.float64


@pytest.fixture(scope="module")
def kvx():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import kvx as k
    import kvx.pages  # noqa: F401
    assert k.lib.kvx_device_check() == 0, "not an sm_100 device"
    return k


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def normal(g, *shape, dtype=F16):
    return torch.randn(shape, generator=g, device="cuda", dtype=F32).to(dtype)


def ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def flag():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------- rotary ---

def turn64(x, pos, table, inverse=False):
    """The rotation in 64 bits; the angle from the table's own integers."""
    r, half = table.rotary_dim, table.rotary_dim // 2
    turns = [int(t) % (1 << 64) for t in table.turns.tolist()]
    frac = torch.tensor([[(t * int(p)) % (1 << 64) / 2.0 ** 64 for t in turns] for p in pos.tolist()], dtype=F64).reshape(-1, half)
    ang = (2 * math.pi * frac).to(x.device)[:, None]
    c, s = ang.cos() * table.amplitude, ang.sin() * table.amplitude * (-1 if inverse else 1)
    y, x = x.double().clone(), x.double()
    if table.layout == "half":
        a, b = x[..., :half], x[..., half:r]
        y[..., :half], y[..., half:r] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., :r:2], x[..., 1:r:2]
        y[..., :r:2], y[..., 1:r:2] = a * c - b * s, b * c + a * s
    return y


def turn_bound(x, table):
    """Bound on the fp32 error of a rotated element: the argument and sincospi
    (5 E32 of cosine and sine, absolute), amplitude, product, sum: 8 E32 of
    |a| + |b|."""
    r, half = table.rotary_dim, table.rotary_dim // 2
    x = x.double().abs()
    e = torch.zeros_like(x)
    if table.layout == "half":
        e[..., :r] = (x[..., :half] + x[..., half:r]).repeat(1, 1, 2)
    else:
        e[..., :r] = (x[..., :r:2] + x[..., 1:r:2]).repeat_interleave(2, -1)
    return 8 * E32 * abs(table.amplitude) * e


def assert_turned(got, x, pos, table, inverse=False):
    want = turn64(x, pos, table, inverse)
    tol = turn_bound(x, table)
    tol = tol + (E16 * (want.abs() + tol) + TINY16 if got.dtype == F16 else E32 * want.abs())
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} elements off, worst {(got.double() - want).abs().max():.3e}"


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("tokens,hq,hk,dim,rotary", [
    (1, 24, 8, 128, 128), (7, 64, 8, 128, 64), (33, 3, 1, 80, 80), (5, 2, 2, 96, 48), (4, 1, 1, 6, 2), (3, 5, 2, 17, 10),
    (2, 1, 1, 1024, 1024), (2, 3, 1, 1024, 2), (130, 21, 3, 256, 192), (1, 1, 1, 2, 2), (9, 4, 4, 64, 24)])
def test_rope(kvx, dtype, layout, tokens, hq, hk, dim, rotary):
    g = gen(tokens * 1000 + dim)
    q, k = normal(g, tokens, hq, dim, dtype=dtype), normal(g, tokens, hk, dim, dtype=dtype)
    pos = torch.randint(0, 200000, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    t = kvx.rope_table(rotary, base=500000.0, layout=layout, scaling="yarn", factor=4.0, high=32.0)
    for inverse in (False, True):
        qo, ko = kvx.rope(q, k, pos, t, inverse=inverse)
        assert_turned(qo, q, pos, t, inverse)
        assert_turned(ko, k, pos, t, inverse)
        assert torch.equal(qo[..., rotary:], q[..., rotary:]) and torch.equal(ko[..., rotary:], k[..., rotary:])


def test_rope_positions_far_negative_and_zero(kvx):
    pos = ints([0, 1, -1, 2 ** 31 - 1, -2 ** 31, 10 ** 9, 123456789, -77])
    for scaling in ("none", "linear", "ntk", "llama3", "yarn"):
        t = kvx.rope_table(128, scaling=scaling, factor=8.0, low=1.0, high=32.0)
        x = normal(gen(3), 8, 4, 128, dtype=F32)
        y, _ = kvx.rope(x, None, pos, t)
        assert_turned(y, x, pos, t)
        if t.amplitude == 1.0:
            assert torch.equal(y[0], x[0])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_rope_strides_in_place_and_unaligned(kvx, layout, dtype):
    """Views of a packed projection, heads before tokens, a view that starts
    off a 16-byte boundary, an expanded input: the same bits as contiguous."""
    g = gen(5)
    t = kvx.rope_table(96, layout=layout)
    pos = torch.randint(0, 9000, (19,), generator=g, device="cuda", dtype=torch.int32)
    packed = normal(g, 19, 12, 128, dtype=dtype)
    q, k = packed[:, :8], packed[:, 8:10]
    qo, ko = kvx.rope(q.contiguous(), k.contiguous(), pos, t)
    assert all(torch.equal(a, b) for a, b in zip(kvx.rope(q, k, pos, t), (qo, ko)))
    rest = packed[:, 10:].clone()
    kvx.rope(q, k, pos, t, q_out=q, k_out=k)  # in place, inside the projection
    assert torch.equal(packed, torch.cat((qo, ko, rest), 1))
    heads_first = normal(g, 8, 19, 128, dtype=dtype)
    out = torch.zeros(8, 19, 128, dtype=dtype, device="cuda")
    kvx.rope(heads_first.transpose(0, 1), None, pos, t, q_out=out.transpose(0, 1))
    assert torch.equal(out.transpose(0, 1), kvx.rope(heads_first.transpose(0, 1).contiguous(), None, pos, t)[0])
    flat = normal(g, 1 + 19 * 3 * 128, dtype=dtype)
    odd = flat[1:].view(19, 3, 128)
    assert torch.equal(kvx.rope(odd, None, pos, t)[0], kvx.rope(odd.clone(), None, pos, t)[0])
    one = normal(g, 1, 1, 128, dtype=dtype)
    wide = one.expand(19, 3, 128)
    assert torch.equal(kvx.rope(wide, None, pos, t)[0], kvx.rope(wide.contiguous(), None, pos, t)[0])
    with pytest.raises(ValueError):
        kvx.rope(odd, None, pos, t, q_out=torch.empty(1, 1, 128, dtype=dtype, device="cuda").expand(19, 3, 128))


def test_rope_inverse_is_the_gradient(kvx):
    """<w, rope(x)> changes by <inverse(w), dx>: against differences, and the
    formula's transpose (the rotation is linear, so a difference has no error
    of its own beyond rounding)."""
    g = gen(8)
    for layout in ("half", "interleaved"):
        t = kvx.rope_table(64, layout=layout, scaling="yarn", factor=8.0, high=32.0)
        x, w, dx = (normal(g, 6, 5, 96, dtype=F32) for _ in range(3))
        pos = torch.randint(0, 100000, (6,), generator=g, device="cuda", dtype=torch.int32)
        grad, _ = kvx.rope(w, None, pos, t, inverse=True)
        assert_turned(grad, w, pos, t, True)
        y0, y1 = kvx.rope(x, None, pos, t)[0], kvx.rope(x + dx, None, pos, t)[0]
        change = (w.double() * (y1.double() - y0.double())).sum()
        tol = (w.double().abs() * (turn_bound(x, t) + turn_bound(x + dx, t) + E32 * (y0.double().abs() + y1.double().abs())
                                   + 2 * E32 * (x + dx).double().abs())).sum()
        tol = tol + (turn_bound(w, t) * dx.double().abs()).sum() + (E32 * grad.double().abs() * dx.double().abs()).sum()
        assert abs(change - (grad.double() * dx.double()).sum()) <= tol


def test_rope_rows_of_no_tokens_and_no_heads(kvx):
    t = kvx.rope_table(128)
    q, k = kvx.rope(torch.empty(0, 4, 128, dtype=F16, device="cuda"), None, ints([]), t)
    assert q.shape == (0, 4, 128) and k is None
    q, k = kvx.rope(torch.empty(2, 0, 128, dtype=F16, device="cuda"), torch.ones(2, 1, 128, dtype=F16, device="cuda"), ints([0, 0]), t)
    assert torch.equal(k, torch.ones_like(k))


# ------------------------------------------------------------------- append ---

def round_half_away(t):
    f = np.floor(t)
    return f + (t - f >= 0.5)


def quantise32(x):
    """The reference's codec on one block [n][128] of fp32, operation by operation."""
    x = x.astype(np.float32)
    lo, hi = x.min(), x.max()
    scale = np.float32((hi - lo) / np.float32(255))
    scale = np.float32(1) if scale == 0 else scale
    codes = np.clip(round_half_away((x - lo) / scale), 0, 255) - 128
    return codes.astype(np.int8), np.array([lo, hi, scale, lo], np.float32)


def requantise32(codes, old, lo, hi):
    scale = np.float32((hi - lo) / np.float32(255))
    scale = np.float32(1) if scale == 0 else scale
    x = old[3] + (codes.astype(np.float32) + np.float32(128)) * old[2]
    return (np.clip(round_half_away((x - lo) / scale), 0, 255) - 128).astype(np.int8)


def append_i8_plain(pool, stats, bt, ctx, new, k, v):
    """Unrotated append in numpy: exact codes and statistics."""
    row = 0
    for s, (c, n) in enumerate(zip(ctx, new)):
        at = c
        while at < c + n:
            page, slot = bt[s][at // 16], at % 16
            m = min(16 - slot, c + n - at)
            for h in range(pool.shape[2]):
                for i, x in enumerate((k, v)):
                    block = x[row:row + m, h].astype(np.float32)
                    old = stats[page, i, h].copy()
                    lo, hi = block.min(), block.max()
                    if slot:
                        lo, hi = min(lo, old[0]), max(hi, old[1])
                        if not (lo == old[0] and hi == old[1]):
                            pool[page, i, h, :slot] = requantise32(pool[page, i, h, :slot], old, lo, hi)
                    scale = np.float32((hi - lo) / np.float32(255))
                    scale = np.float32(1) if scale == 0 else scale
                    pool[page, i, h, slot:slot + m] = np.clip(round_half_away((block - lo) / scale), 0, 255) - 128
                    stats[page, i, h] = (lo, hi, scale, lo)
            row += m
            at += m


def layout_of(ctx, new, seed, extra=2):
    need = [(c + n + 15) // 16 for c, n in zip(ctx, new)]
    num_pages, max_pages = sum(need) + extra, max(max(need), 1) + 1
    ids = np.random.RandomState(seed).permutation(num_pages)
    bt = np.full((len(ctx), max_pages), -1, np.int32)
    used = 0
    for s, n in enumerate(need):
        bt[s, :n] = ids[used:used + n]
        used += n
    start = np.concatenate(([0], np.cumsum(new))).astype(np.int32)
    return bt, num_pages, start


def random_i8_pool(g, num_pages, hkv):
    pool = torch.randint(-128, 128, (num_pages, 2, hkv, 16, 128), generator=g, device="cuda", dtype=torch.int8)
    lo = -1 - torch.rand((num_pages, 2, hkv), generator=g, device="cuda")
    hi = 1 + torch.rand((num_pages, 2, hkv), generator=g, device="cuda")
    return pool, torch.stack((lo, hi, (hi - lo) / 255, lo), -1).contiguous()


RAGGED = [([0], [1]), ([0], [16]), ([15], [1]), ([15], [2]), ([3, 0, 16, 100, 31], [1, 1, 1, 1, 1]),
          ([0, 5, 16, 250, 7], [33, 0, 16, 100, 9]), ([1], [500]), ([40, 0, 9], [0, 0, 3])]


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("ctx,new", RAGGED)
@pytest.mark.parametrize("hkv", [1, 8])
def test_append_i8_without_rotation_is_exact(kvx, dtype, ctx, new, hkv):
    bt, num_pages, start = layout_of(ctx, new, 3)
    g = gen(sum(ctx) + sum(new) + hkv)
    pool, stats = random_i8_pool(g, num_pages, hkv)
    k, v = normal(g, int(start[-1]), hkv, 128, dtype=dtype), normal(g, int(start[-1]), hkv, 128, dtype=dtype) * 3
    want, wstats = pool.cpu().numpy(), stats.cpu().numpy()
    append_i8_plain(want, wstats, bt, ctx, new, k.float().cpu().numpy(), v.float().cpu().numpy())
    err = flag()
    kvx.rope_append(pool, ints(bt), ints(start), ints(ctx), k, v, stats=stats, error_flag=err)
    assert err.item() == 0
    assert np.array_equal(pool.cpu().numpy(), want)
    assert np.array_equal(stats.cpu().numpy().view(np.uint32), wstats.view(np.uint32))


def test_append_i8_of_whole_pages_is_the_codec(kvx):
    """Pages filled from their first slot: the bits of kvx_compress_int8 of
    those blocks.  More than 16 x 148 tokens, the prompt-sized launch."""
    n = 16 * 160
    g = gen(9)
    k, v = normal(g, n, 2, 128), normal(g, n, 2, 128)
    pool = torch.zeros(n // 16, 2, 2, 16, 128, dtype=torch.int8, device="cuda")
    stats = torch.zeros(n // 16, 2, 2, 4, device="cuda")
    table = torch.randperm(n // 16, generator=g, device="cuda").int()
    kvx.rope_append(pool, table[None], ints([0, n]), ints([0]), k, v, stats=stats)
    plain = torch.stack((k, v)).view(2, n // 16, 16, 2, 128).permute(1, 0, 3, 2, 4).contiguous()
    codes, want = kvx.compress_int8(plain)
    assert torch.equal(pool[table.long()].flatten(), codes)
    assert torch.equal(stats[table.long()].flatten(), want.flatten())


@pytest.mark.parametrize("layout,rotary", [("half", 128), ("interleaved", 128), ("half", 64), ("interleaved", 50), ("half", 50),
                                           ("half", 2), ("interleaved", 2)])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("ctx,new", [([0, 37, 4], [50, 1, 30]), ([13], [2500])])
def test_append_i8_rotated(kvx, layout, rotary, dtype, ctx, new):
    """Keys quantised from their rotated fp32 values: every new value within
    half a step of the rotated key, the range within its error."""
    bt, num_pages, start = layout_of(ctx, new, 4)
    g, hq, hkv = gen(rotary + len(ctx)), 6, 2
    pool, stats = random_i8_pool(g, num_pages, hkv)
    before, sbefore = pool.clone(), stats.clone()
    packed = normal(g, int(start[-1]), hq + 2 * hkv, 128, dtype=dtype)
    q, k, v = packed[:, :hq], packed[:, hq:hq + hkv], packed[:, hq + hkv:]
    t = kvx.rope_table(rotary, layout=layout, scaling="llama3", factor=8.0)
    err = flag()
    qo = kvx.rope_append(pool, ints(bt), ints(start), ints(ctx), k, v, q=q, table=t, stats=stats, error_flag=err)
    assert err.item() == 0
    pos = torch.cat([torch.arange(c, c + n) for c, n in zip(ctx, new)]).int().cuda()
    assert torch.equal(qo, kvx.rope(q, None, pos, t)[0])  # the same rows, the same bits
    seq = torch.repeat_interleave(torch.arange(len(ctx)), torch.tensor(new)).cuda()
    page, slot = ints(bt).long()[seq, pos.long() // 16], pos.long() % 16
    turned, slack = turn64(k, pos, t), turn_bound(k, t)
    for i, (x, e) in enumerate(((turned, slack), (v.double(), torch.zeros_like(slack)))):
        st = stats[page, i].double()  # [tokens][hkv][4]
        got = st[..., 3:] + (pool[page, i, :, slot].double() + 128) * st[..., 2:3]
        # half a step; quotient and scale in fp32 are off by 2 E32 of up to 255 steps each
        tol = st[..., 2:3] * (0.5 + 4 * 255 * E32) + e + 2 * E32 * st[..., :2].abs().amax(-1, keepdim=True)
        assert ((got - x).abs() <= tol).all()
        assert (x + e >= st[..., :1]).all() and (x - e <= st[..., 1:2]).all()
    # the range is reached: min and max are those of the rows (and of what was there)
    for p in range(num_pages):
        rows = (page == p).nonzero()[:, 0]
        if not len(rows):
            assert torch.equal(pool[p], before[p]) and torch.equal(stats[p], sbefore[p])
            continue
        first, last = int(slot[rows].min()), int(slot[rows].max())
        for i, x in enumerate((turned, v.double())):
            lo, hi = x[rows].amin((0, 2)), x[rows].amax((0, 2))
            if first:
                lo, hi = torch.minimum(lo, sbefore[p, i, :, 0].double()), torch.maximum(hi, sbefore[p, i, :, 1].double())
            e = slack[rows].amax((0, 2)) + E32 * torch.maximum(lo.abs(), hi.abs())
            assert ((stats[p, i, :, 0] - lo).abs() <= e).all() and ((stats[p, i, :, 1] - hi).abs() <= e).all()
        assert torch.equal(pool[p, :, :, last + 1:], before[p, :, :, last + 1:])


def test_append_i8_token_by_token_drifts_by_half_a_step_each(kvx):
    """16 appends into one page: each widening rounds the earlier rows once
    more, by half a step of the range it widens to."""
    g = gen(12)
    k = normal(g, 16, 4, 128) * torch.linspace(0.1, 2, 16, device="cuda", dtype=F16)[:, None, None]
    v = normal(g, 16, 4, 128)
    pool = torch.zeros(1, 2, 4, 16, 128, dtype=torch.int8, device="cuda")
    stats = torch.full((1, 2, 4, 4), float("nan"), device="cuda")  # an unused page's statistics are not read
    drift = torch.zeros(16, 2, 4, dtype=F64, device="cuda")
    last = torch.full((2, 4), -1.0, dtype=F64, device="cuda")
    for i in range(16):
        kvx.rope_append(pool, ints([[0]]), ints([0, 1]), ints([i]), k[i:i + 1], v[i:i + 1], stats=stats)
        scale = stats[0, ..., 2].double()
        grew = scale != last
        drift[:i] += torch.where(grew, 0.5 * scale * (1 + 2 ** -10), 0.0)
        drift[i] = 0.5 * scale * (1 + 2 ** -10)
        last = scale
    got = kvx.decompress_int8(pool, stats).view(2, 4, 16, 128).double()
    want = torch.stack((k, v)).permute(0, 2, 1, 3).double()
    assert ((got - want).abs() <= drift.permute(1, 2, 0)[..., None]).all()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("layout,rotary", [("half", 128), ("interleaved", 96), ("half", 10)])
def test_append_to_float_pools_is_rope_then_append(kvx, dtype, layout, rotary):
    ctx, new = [0, 5, 16, 47, 8], [33, 1, 0, 20, 8]
    bt, num_pages, start = layout_of(ctx, new, 6)
    g = gen(rotary)
    q, k, v = (normal(g, int(start[-1]), h, 128, dtype=dtype) for h in (6, 2, 2))
    pool = normal(g, num_pages, 2, 2, 16, 128, dtype=dtype)
    want = pool.clone()
    t = kvx.rope_table(rotary, layout=layout)
    pos = torch.cat([torch.arange(c, c + n) for c, n in zip(ctx, new)]).int().cuda()
    tq, tk = kvx.rope(q, k, pos, t)
    for s, (c, n) in enumerate(zip(ctx, new)):
        a, b = int(start[s]), int(start[s + 1])
        if n:
            kvx.append_chunk(want, ints(bt[s:s + 1]), ints([c]), tk[None, a:b].contiguous(), v[None, a:b].contiguous())
    qo = kvx.rope_append(pool, ints(bt), ints(start), ints(ctx), k, v, q=q, table=t)
    assert torch.equal(qo, tq) and torch.equal(pool, want)
    # without a table: a plain ragged append, q copied
    plain, again = want.clone(), want.clone()
    for s, (c, n) in enumerate(zip(ctx, new)):
        a, b = int(start[s]), int(start[s + 1])
        if n:
            kvx.append_chunk(plain, ints(bt[s:s + 1]), ints([c]), k[None, a:b].contiguous(), v[None, a:b].contiguous())
    assert torch.equal(kvx.rope_append(again, ints(bt), ints(start), ints(ctx), k, v, q=q), q) and torch.equal(again, plain)


@pytest.mark.parametrize("kind", ["f16", "i8"])
def test_append_skips_and_reports_bad_rows(kvx, kind):
    """A negative position, a page outside pool or table, rows of no sequence:
    skipped, nothing else touched; q rows behind the last sequence stay."""
    g = gen(14)
    hkv, total = 2, 60
    if kind == "i8":
        pool, stats = random_i8_pool(g, 4, hkv)
    else:
        pool, stats = normal(g, 4, 2, hkv, 16, 128), None
    before = pool.clone()
    k, v, q = (normal(g, total, h, 128) for h in (hkv, hkv, 4))
    q_out = torch.full_like(q, 7.0)
    bt = ints([[0, -1], [9, 1], [2, 3], [3, 3]])
    # seq 0: positions 10..29, page 1 missing; 1: page 9 outside the pool, then page 1; 2: negative; 3: runs out of the table at 32
    start, pos = ints([0, 20, 40, 45, 50]), ints([10, 10, -3, 30])
    err = flag()
    kvx.rope_append(pool, bt, start, pos, k, v, q=q, q_out=q_out, table=kvx.rope_table(128), stats=stats, error_flag=err)
    assert err.item() == 2
    assert torch.equal(pool[2], before[2])  # the negative position's page
    assert torch.equal(q_out[50:], torch.full_like(q[50:], 7.0)) and not (q_out[:50] == 7.0).all(-1).any()
    assert torch.equal(pool[0, :, :, :10], before[0, :, :, :10]) or kind == "i8"
    assert not torch.equal(pool[0, :, :, 10:], before[0, :, :, 10:])
    assert not torch.equal(pool[1, :, :, :14], before[1, :, :, :14]) and torch.equal(pool[1, :, :, 14:], before[1, :, :, 14:])
    assert not torch.equal(pool[3, :, :, 14:], before[3, :, :, 14:])
    # no row may be left without a flag pointer either
    kvx.rope_append(pool, bt, start, pos, k, v, table=kvx.rope_table(128), stats=stats)


def test_append_i8_of_nan_inf_and_constant_blocks(kvx):
    """NaN stays out of the range; a constant block has scale 1; an infinite
    one an infinite scale, as the codec has it; none touches its neighbours."""
    k = torch.full((16, 4, 128), 2.5, dtype=F32, device="cuda")
    k[3, 1, 5] = float("nan")
    k[:, 2] = float("nan")
    k[2, 3, 7] = float("inf")
    pool = torch.zeros(1, 2, 4, 16, 128, dtype=torch.int8, device="cuda")
    stats = torch.zeros(1, 2, 4, 4, device="cuda")
    kvx.rope_append(pool, ints([[0]]), ints([0, 16]), ints([0]), k, torch.zeros_like(k), stats=stats)
    s = stats[0, 0].cpu()
    assert s[0].tolist() == [2.5, 2.5, 1.0, 2.5] and s[1].tolist() == [2.5, 2.5, 1.0, 2.5]
    assert s[2].isnan().sum() == 4 and s[3, 1] == float("inf") and s[3, 2] == float("inf")
    assert (pool[0, 0] == -128).all() and stats[0, 1].flatten().tolist() == [0.0, 0.0, 1.0, 0.0] * 4


# ------------------------------------------------------------------- attend ---

def attend64(pool, stats, bt, start, ctx, q, scale=None, causal=True):
    """(output, sum of p |s c|, score size, score span) in 64 bits, row by row
    of each sequence; pages that name none are left out."""
    scale = scale or 1 / math.sqrt(128)
    hkv, hq, group = pool.shape[2], q.shape[1], q.shape[1] // pool.shape[2]
    out = torch.zeros(q.shape, dtype=F64, device="cuda")
    size, noise = torch.zeros_like(out), torch.zeros(q.shape[:2] + (1,), dtype=F64, device="cuda")
    for s in range(len(ctx)):
        a, b = int(start[s]), int(start[s + 1])
        if a == b or ctx[s] < 0:
            continue
        keys = min(ctx[s] + b - a, bt.shape[1] * 16)
        ids = torch.tensor(np.asarray(bt[s][: (keys + 15) // 16]), dtype=torch.int64)
        known = ((ids >= 0) & (ids < pool.shape[0])).repeat_interleave(16)[:keys].cuda()
        ids = torch.where((ids >= 0) & (ids < pool.shape[0]), ids, 0).cuda()
        last = torch.arange(ctx[s], ctx[s] + b - a, device="cuda") if causal else torch.full((b - a,), keys, device="cuda")
        seen = (torch.arange(keys, device="cuda")[None] <= last[:, None]) & known[None]
        for h in range(hkv):
            st, c = stats[ids, :, h].double(), pool[ids, :, h].double()
            mid, part = st[..., 3, None, None] + 128 * st[..., 2, None, None], c * st[..., 2, None, None]
            kk, vv = ((mid + part)[:, i].reshape(-1, 128)[:keys] for i in (0, 1))
            vpart = (part[:, 1].abs() + mid[:, 1].abs()).reshape(-1, 128)[:keys]
            kpart = (part[:, 0].abs() + mid[:, 0].abs()).reshape(-1, 128)[:keys]
            qq = q[a:b, h * group:(h + 1) * group].double()
            score = torch.einsum("tgd,kd->tgk", qq, kk) * scale
            rough = torch.einsum("tgd,kd->tgk", qq.abs(), kpart) * scale
            mask = seen[:, None, :]
            some = mask.any(-1, keepdim=True)
            p = torch.softmax(score.masked_fill(~mask, -math.inf), -1)
            p = torch.where(some & mask, p, 0.0)
            out[a:b, h * group:(h + 1) * group] = torch.einsum("tgk,kd->tgd", p, vv)
            size[a:b, h * group:(h + 1) * group] = torch.einsum("tgk,kd->tgd", p, vpart)
            noise[a:b, h * group:(h + 1) * group] = torch.where(mask, rough, 0.0).amax(-1, keepdim=True)
    return out, size, noise


def assert_attended(got, ref):
    """A score is a sum of 128 products (and 2 more) in fp32, off by at most
    130 steps of 2^-23 (the tensor core may truncate) of its absolute sum; so
    is its exponent, which moves p by that fraction, and once more through the
    sum.  fp16 calls round p (E16 of it), all calls their output; fp32 calls
    split q and p to 2^-22.  The second product sums in fp32: for n keys the
    error grows like the walk of its roundings; 64 steps of 2^-23 of the
    absolute sum bound it by far."""
    out, size, noise = ref
    half = got.dtype == F16
    eps = 130 * 2.0 ** -23 * noise + 2.0 ** -20
    tol = (2 * eps + 64 * 2.0 ** -23 + (E16 if half else 2.0 ** -21)) * size
    tol = tol + ((E16 * (out.abs() + tol) + TINY16) if half else E32 * out.abs())
    bad = ~((got.double() - out).abs() <= tol)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} elements off, worst {(got.double() - out).abs().max():.3e}, "
                           f"first at {bad.nonzero()[0].tolist()}")


def attend_case(seed, ctx, new, hq, hkv, dtype, scale_of=None):
    bt, num_pages, start = layout_of(ctx, new, seed)
    g = gen(seed)
    x = normal(g, num_pages, 2, hkv, 16, 128, dtype=F32)
    if scale_of is not None:
        x = x * scale_of(g, num_pages, hkv)
    lo, hi = x.amin((-2, -1)), x.amax((-2, -1))
    scale = (hi - lo) / 255
    pool = (((x - lo[..., None, None]) / scale[..., None, None]).round().clamp(0, 255) - 128).to(torch.int8)
    stats = torch.stack((lo, hi, scale, lo), -1).contiguous()
    return pool, stats, bt, start, normal(g, int(start[-1]), hq, 128, dtype=dtype)


ATTEND = [
    ([0], [1]), ([0], [2]), ([5], [1]), ([15], [1]), ([16], [1]), ([127], [1]), ([128], [1]), ([300], [3]), ([0], [16]), ([0], [43]),
    ([0], [129]), ([0], [200]), ([1000], [5]), ([77, 0, 513, 4], [1, 5, 2, 1]), ([0, 300, 40], [130, 0, 70]), ([0, 0], [0, 9]),
    ([511], [257]), ([3000, 17], [2, 90]),
]


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("hq,hkv", [(24, 8), (16, 2), (3, 3), (21, 3), (40, 2)])
@pytest.mark.parametrize("ctx,new", ATTEND)
def test_attend(kvx, dtype, hq, hkv, ctx, new):
    pool, stats, bt, start, q = attend_case(sum(ctx) + hq, ctx, new, hq, hkv, dtype)
    err = flag()
    out = kvx.attend_chunk(pool, ints(bt), ints(start), ints(ctx), q, stats=stats, error_flag=err)
    assert err.item() == 0
    assert_attended(out, attend64(pool, stats, bt, start, ctx, q))


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("ctx,new", [([0], [1]), ([0], [130]), ([77, 0, 513], [1, 150, 2]), ([900], [300])])
def test_attend_without_causal_mask(kvx, dtype, ctx, new):
    pool, stats, bt, start, q = attend_case(len(ctx) + new[0], ctx, new, 16, 2, dtype)
    out = kvx.attend_chunk(pool, ints(bt), ints(start), ints(ctx), q, stats=stats, causal=False, sm_scale=0.05)
    assert_attended(out, attend64(pool, stats, bt, start, ctx, q, scale=0.05, causal=False))


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("seed,ctx,new,hq,hkv", [(1, [9000], [600], 24, 8), (2, [33000, 20], [4, 700], 8, 1), (3, [0], [3000], 8, 8),
                                                 (4, [40 * i for i in range(70)], [1 + i % 3 for i in range(70)], 12, 4)])
def test_attend_long_and_many(kvx, dtype, seed, ctx, new, hq, hkv):
    pool, stats, bt, start, q = attend_case(seed, ctx, new, hq, hkv, dtype)
    out = kvx.attend_chunk(pool, ints(bt), ints(start), ints(ctx), q, stats=stats)
    assert_attended(out, attend64(pool, stats, bt, start, ctx, q))


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("ctx,new,hq,hkv", [([3000], [801], 24, 8), ([2500, 40, 3001], [500, 2, 700], 16, 8), ([700] * 40, [20] * 40, 8, 2),
                                            ([1100 + 7 * i for i in range(35)], [17 + i for i in range(35)], 16, 4),
                                            ([9001, 0], [1, 260], 16, 8), ([5000], [130], 8, 1)])
def test_attend_more_row_tiles_than_sms(kvx, dtype, ctx, new, hq, hkv):
    """Whole row tiles and, behind them, split ones; more than 32 sequences."""
    pool, stats, bt, start, q = attend_case(sum(new), ctx, new, hq, hkv, dtype)
    for causal in (True, False):
        out = kvx.attend_chunk(pool, ints(bt), ints(start), ints(ctx), q, stats=stats, causal=causal)
        assert_attended(out, attend64(pool, stats, bt, start, ctx, q, causal=causal))


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("ctx,new", [([600], [2]), ([500, 77], [5, 40]), ([64], [300])])
def test_attend_over_constant_pages(kvx, dtype, ctx, new):
    """Pages of one value (their scale is zero), among pages of a tiny and of
    a large range: values of 2^12 +- 2^-8 or 2^8 in V."""
    pool, stats, bt, start, q = attend_case(61, ctx, new, 8, 2, dtype)
    for i, page in enumerate(sorted({int(p) for row in bt for p in row if p >= 0})):
        if i % 3 == 0:
            stats[page, :, :, 2] = 0.0
        elif i % 3 == 1:
            stats[page, 1, :, 2:] *= 2.0 ** -9
            stats[page, 1, :, 3] += 4096.0
        else:
            stats[page, 1, :, 2:] *= 2.0 ** 6
    out = kvx.attend_chunk(pool, ints(bt), ints(start), ints(ctx), q, stats=stats)
    assert_attended(out, attend64(pool, stats, bt, start, ctx, q))


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("ratio", [6, 9, 12, 15])
def test_attend_rows_that_see_small_pages_only(kvx, dtype, ratio):
    """The first rows see a page whose V scale is 2^-ratio of the next page's."""
    ctx, new = [0, 0], [40, 300]
    pool, stats, bt, start, q = attend_case(63 + ratio, ctx, new, 8, 2, dtype)
    for row in bt:
        stats[int(row[0]), 1, :, 2:] *= 2.0 ** -ratio
    out = kvx.attend_chunk(pool, ints(bt), ints(start), ints(ctx), q, stats=stats)
    assert_attended(out, attend64(pool, stats, bt, start, ctx, q))


@pytest.mark.parametrize("dtype", [F16, F32])
def test_attend_with_starts_that_do_not_ascend(kvx, dtype):
    """Ranges that overlap claim more rows than there are: no result is
    promised, but the workspace's end holds and every row is a number."""
    rows, hq, hkv = 400, 16, 8
    start = [0, 400, 2, 390, 1, 400, 5, 400]
    ctx = [1500] * (len(start) - 1)
    pool, stats, bt, _, _ = attend_case(64, ctx, [400] * len(ctx), hq, hkv, dtype)
    q = normal(gen(65), rows, hq, 128, dtype=dtype)
    ws = kvx.attend_chunk_workspace(len(ctx), rows, hq, hkv, bt.shape[1])
    guarded = torch.full((ws.numel() + 4096,), 171, dtype=torch.uint8, device="cuda")
    out = kvx.attend_chunk(pool, ints(bt), ints(start), ints(ctx), q, stats=stats, workspace=guarded[: ws.numel()])
    assert (guarded[ws.numel():] == 171).all() and torch.isfinite(out).all()


def test_attend_two_at_once(kvx):
    """Calls of two streams, a workspace each: the bits of the same calls
    alone.  Mixed lengths, both types, the dense attention beside them (it
    takes tensor memory too)."""
    cases = []
    for seed, dtype in ((66, F16), (67, F32)):
        ctx, new = [2000, 40, 700], [5, 300, 40]
        pool, stats, bt, start, q = attend_case(seed, ctx, new, 16, 4, dtype)
        args = (pool, ints(bt), ints(start), ints(ctx), q)
        cases.append((args, dict(stats=stats, workspace=kvx.attend_chunk_workspace(3, len(q), 16, 4, bt.shape[1]))))
    want = [kvx.attend_chunk(*args, **kw) for args, kw in cases]
    x = normal(gen(68), 512, 128, dtype=F32)
    dense = kvx.attention_dense(x, x, x)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (args, kw) in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                got[i].append(kvx.attend_chunk(*args, **kw))
        with torch.cuda.stream(streams[2]):
            again = kvx.attention_dense(x, x, x)
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])
    assert torch.equal(again, dense)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_attend_in_place(kvx, dtype):
    """out may be q."""
    ctx, new = [3000, 100, 513], [801, 4, 60]
    pool, stats, bt, start, q = attend_case(62, ctx, new, 24, 8, dtype)
    want = kvx.attend_chunk(pool, ints(bt), ints(start), ints(ctx), q, stats=stats)
    got = q.clone()
    kvx.attend_chunk(pool, ints(bt), ints(start), ints(ctx), got, stats=stats, out=got)
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("ctx,new", [([600], [7]), ([64], [300])])
def test_attend_over_pages_of_very_different_ranges(kvx, dtype, ctx, new):
    """Blocks whose scales differ by up to 2^20, keys far off zero."""
    def spread(g, pages, hkv):
        e = torch.randint(-10, 11, (pages, 2, hkv, 1, 1), generator=g, device="cuda").float()
        return torch.stack((torch.exp2(e[:, 0] / 5), torch.exp2(e[:, 1])), 1)
    pool, stats, bt, start, q = attend_case(31, ctx, new, 8, 2, dtype, spread)
    stats[:, 0, :, 3] += 4.0  # zero points of the keys
    out = kvx.attend_chunk(pool, ints(bt), ints(start), ints(ctx), q, stats=stats)
    assert_attended(out, attend64(pool, stats, bt, start, ctx, q))


@pytest.mark.parametrize("dtype", [F16, F32])
def test_attend_with_dominant_and_distant_scores(kvx, dtype):
    """Large queries: scores of hundreds, one key takes nearly all; rising
    scores, so that the running maximum moves in every tile."""
    ctx, new = [1500], [40]
    pool, stats, bt, start, q = attend_case(41, ctx, new, 8, 2, dtype)
    rise = torch.linspace(-2, 2, bt.shape[1] * 16, device="cuda")
    for lp, page in enumerate(bt[0]):
        if page >= 0:
            stats[page, 0, :, 3] = rise[lp * 16]
    out = kvx.attend_chunk(pool, ints(bt), ints(start), ints(ctx), q * 6, stats=stats)
    assert_attended(out, attend64(pool, stats, bt, start, ctx, q * 6))


@pytest.mark.parametrize("dtype", [F16, F32])
def test_attend_missing_pages_and_empty_rows(kvx, dtype):
    """Pages that name none are left out, a query that sees no key gives a
    zero row; a context longer than the table, a negative position; rows of no
    sequence keep what they hold."""
    ctx, new = [40, 0, 8, 200], [30, 5, 4, 20]
    pool, stats, bt, start, q = attend_case(51, ctx, new, 8, 2, dtype)
    bt[0, 1] = 10 ** 6
    bt[1, 0] = -1  # sequence 1 sees nothing
    bt[3, 3:6] = -7
    q = torch.cat((q, normal(gen(1), 11, 8, 128, dtype=dtype)))
    out = torch.full_like(q, 3.0)
    err = flag()
    kvx.attend_chunk(pool, ints(bt), ints(start), ints(ctx), q, stats=stats, out=out, error_flag=err)
    assert err.item() == 2
    n = int(start[-1])
    assert_attended(out[:n], attend64(pool, stats, bt, start, ctx, q[:n]))
    assert (out[int(start[1]):int(start[2])] == 0).all() and (out[n:] == 3.0).all()
    # beyond the table: the keys that it holds
    short = np.ascontiguousarray(bt[3:4, :8])
    err.zero_()
    got = kvx.attend_chunk(pool, ints(short), ints([0, 20]), ints([200]), q[:20], stats=stats, error_flag=err)
    assert err.item() & 4
    assert_attended(got, attend64(pool, stats, short, [0, 20], [200], q[:20]))
    # a negative position leaves its sequence out
    err.zero_()
    got = kvx.attend_chunk(pool, ints(bt[:1]), ints([0, 20]), ints([-1]), q[:20], stats=stats, error_flag=err)
    assert err.item() & 2 and (got == 0).all()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_attend_keeps_masked_infinities_out(kvx, dtype, bad):
    """Statistics of a later page that hold an infinity or NaN do not reach
    the queries before it, in the same tile or in another row tile."""
    ctx, new = [20], [60]
    pool, stats, bt, start, q = attend_case(61, ctx, new, 8, 2, dtype)
    clean = attend64(pool, stats, bt, start, ctx, q)  # 0 * inf would be NaN in its products
    stats[bt[0, 3]] = bad  # tokens 48..63: queries from row 28 on see it
    stats[bt[0, 4], 1] = bad
    got = kvx.attend_chunk(pool, ints(bt), ints(start), ints(ctx), q, stats=stats)
    assert_attended(got[:28], tuple(x[:28] for x in clean))
    assert not torch.isfinite(got[30:]).any()


def test_attend_agrees_with_single_token_decode(kvx):
    ctx = [0, 100, 511, 2000]
    pool, stats, bt, start, q = attend_case(71, ctx, [1] * 4, 24, 8, F16)
    out = kvx.attend_chunk(pool, ints(bt), ints(start), ints(ctx), q, stats=stats)
    lens = ints([c + 1 for c in ctx])
    err = (out.float() - kvx.decode(pool, ints(bt), lens, q, stats=stats).float()).abs()
    assert (err <= 1e-2 + 1e-3 * out.float().abs()).all()  # the decode's own bound


def test_attend_repeats_to_the_bit_on_any_stream_and_in_a_graph(kvx):
    ctx, new = [3000, 10], [6, 200]
    pool, stats, bt, start, q = attend_case(81, ctx, new, 24, 8, F16)
    args = (pool, ints(bt), ints(start), ints(ctx))
    ws = [kvx.attend_chunk_workspace(2, q.shape[0], 24, 8, bt.shape[1]).fill_(i) for i in (0, 255)]
    first = kvx.attend_chunk(*args, q, stats=stats, workspace=ws[0])
    assert torch.equal(first, kvx.attend_chunk(*args, q, stats=stats, workspace=ws[1]))  # whatever the scratch holds
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out, q2 = torch.zeros_like(q), q.clone()
    with torch.cuda.stream(side):
        kvx.attend_chunk(*args, q2, stats=stats, out=out, workspace=ws[1])
    side.synchronize()
    assert torch.equal(out, first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kvx.attend_chunk(*args, q2, stats=stats, out=out, workspace=ws[0])
    for seed in (1, 2):
        q2.copy_(normal(gen(seed), *q.shape))
        graph.replay()
        assert torch.equal(out, kvx.attend_chunk(*args, q2, stats=stats, workspace=ws[1]))


# -------------------------------------------------------------------- pages ---

class Model:
    """The bookkeeping in plain Python: page contents are tags."""

    def __init__(self, num_pages, rows, max_pages):
        self.refs, self.bt, self.lens = [0] * num_pages, [[-1] * max_pages for _ in range(rows)], [0] * rows
        self.tag = list(range(num_pages))

    def take(self):
        page = self.refs.index(0)
        self.refs[page] = 1
        return page

    def reserve(self, grow):
        for r, n in enumerate(grow):
            for lp in range((self.lens[r] + 15) // 16, (self.lens[r] + n + 15) // 16):
                if self.bt[r][lp] < 0:
                    self.bt[r][lp] = self.take()

    def fork(self, parents, children):
        for a, b in zip(parents, children):
            full = self.lens[a] // 16
            for lp in range(full):
                self.bt[b][lp] = self.bt[a][lp]
                self.refs[self.bt[a][lp]] += 1
            self.lens[b] = self.lens[a]
            if self.lens[a] % 16:
                self.bt[b][full] = self.take()
                self.tag[self.bt[b][full]] = self.tag[self.bt[a][full]]

    def free(self, rows):
        for r in rows:
            for lp, page in enumerate(self.bt[r]):
                if page >= 0:
                    self.refs[page] -= 1
                self.bt[r][lp] = -1
            self.lens[r] = 0

    def compact(self):
        live = sum(c > 0 for c in self.refs)
        holes = [p for p in range(live) if not self.refs[p]]
        moved = dict(zip((p for p in range(live, len(self.refs)) if self.refs[p]), holes))
        for a, b in moved.items():
            self.refs[b], self.refs[a], self.tag[b] = self.refs[a], 0, self.tag[a]
        self.bt = [[moved.get(p, p) for p in row] for row in self.bt]
        return live


def tagged_pools(num_pages, layers, hkv, kind):
    """Page p of layer l holds 31 p + l everywhere, its statistics p + l / 8."""
    value = (31 * torch.arange(num_pages, device="cuda")[None] + torch.arange(layers, device="cuda")[:, None])
    shape = (layers, num_pages, 2, hkv, 16, 128)
    if kind == "i8":
        pool = (value % 256 - 128).to(torch.int8)[..., None, None, None, None].expand(shape).contiguous()
        stats = (torch.arange(num_pages, device="cuda")[None] + torch.arange(layers, device="cuda")[:, None] / 8)
        return pool, stats[..., None, None, None].expand(shape[:4] + (4,)).contiguous()
    dtype = {"f16": F16, "f32": F32}[kind]
    return (value % 2048).to(dtype)[..., None, None, None, None].expand(shape).contiguous(), None


def assert_books(pages, model, pool, stats, kind):
    assert pages.refcounts.tolist() == model.refs
    assert pages.block_table.tolist() == model.bt
    assert pages.seq_lens.tolist() == model.lens
    fresh, fstats = tagged_pools(len(model.refs), pool.shape[0], pool.shape[3], kind)
    held = [p for p, c in enumerate(model.refs) if c]  # a free page's contents are nobody's
    tag = [model.tag[p] for p in held]
    assert torch.equal(pool[:, held], fresh[:, tag])
    if stats is not None:
        assert torch.equal(stats[:, held], fstats[:, tag])


@pytest.mark.parametrize("kind,hkv,layers", [("i8", 1, 3), ("f16", 8, 2), ("f32", 3, 1), ("i8", 8, 130)])
@pytest.mark.parametrize("num_pages,rows,max_pages", [(40, 6, 9), (700, 33, 20)])
def test_pages_life(kvx, kind, hkv, layers, num_pages, rows, max_pages):
    """A random life of reserve, grow, fork, free and compact against plain
    Python, whole numbers and page contents."""
    if layers > 100 and num_pages > 100:
        pytest.skip("130 layers once")
    rng = np.random.RandomState(num_pages + layers)
    pool, stats = tagged_pools(num_pages, layers, hkv, kind)
    pages = kvx.pages.Pages.empty(num_pages, rows, max_pages, list(pool), None if stats is None else list(stats))
    model = Model(num_pages, rows, max_pages)
    err, live = flag(), flag()
    for step in range(12):
        grow = [0] * rows
        room = sum(c == 0 for c in model.refs)
        for r in rng.permutation(rows)[: rows // 2 + 1]:
            n = int(rng.randint(0, 40))
            need = (model.lens[r] + n + 15) // 16 - (model.lens[r] + 15) // 16
            if need <= room // 2 and model.lens[r] + n <= 16 * max_pages:
                grow[r], room = n, room - need
        pages.reserve(ints(grow), error_flag=err)
        model.reserve(grow)
        pages.seq_lens += ints(grow)
        model.lens = [a + b for a, b in zip(model.lens, grow)]
        empty = [r for r in range(rows) if model.lens[r] == 0 and model.bt[r][0] < 0]
        full = [r for r in range(rows) if model.lens[r] > 0]
        n = min(len(empty), room, 1 + step % 4)
        if n and full:
            parents = [full[i] for i in rng.randint(0, len(full), n)]
            pages.fork(ints(parents), ints(empty[:n]), error_flag=err)
            model.fork(parents, empty[:n])
        assert_books(pages, model, pool, stats, kind)
        gone = [int(r) for r in rng.permutation(rows)[: 1 + rows // 4]]
        pages.free(ints(gone + gone[:1]), error_flag=err)  # a row given twice is freed once
        model.free(gone)
        if step % 3 == 2:
            pages.compact(num_live=live, error_flag=err)
            assert live.item() == model.compact()
        assert_books(pages, model, pool, stats, kind)
    assert err.item() == 0


def small(kvx, lens=(20, 0, 32, 0), num_pages=7):
    pool, stats = tagged_pools(num_pages, 2, 2, "i8")
    pages = kvx.pages.Pages.empty(num_pages, len(lens), 4, list(pool), list(stats))
    pages.reserve(ints(lens))
    pages.seq_lens.copy_(ints(lens))
    return pages, pool


@pytest.mark.parametrize("what,args,bit", [
    ("reserve", ([100, 0, 0, 0],), 4), ("reserve", ([0, 64, 32, 0],), 8), ("reserve", ([0, -1, 0, 0],), 2),
    ("fork", ([0], [4]), 2), ("fork", ([-1], [1]), 2), ("fork", ([0], [2]), 16), ("fork", ([0, 2], [1, 1]), 16),
    ("fork", ([0], [0]), 16), ("fork", ([0, 1], [1, 3]), 16), ("fork", ([0, 0, 0, 0], [1, 3, 1, 3]), 16)])
def test_pages_refused_calls_change_nothing(kvx, what, args, bit):
    pages, pool = small(kvx)
    before = [t.clone() for t in (pages.refcounts, pages.block_table, pages.seq_lens, pool)]
    err = flag()
    getattr(pages, what)(*(ints(a) for a in args), error_flag=err)
    assert err.item() & bit
    assert all(torch.equal(a, b) for a, b in zip(before, (pages.refcounts, pages.block_table, pages.seq_lens, pool)))
    getattr(pages, what)(*(ints(a) for a in args))  # without a flag


def test_pages_fork_without_room_changes_nothing(kvx):
    pages, pool = small(kvx, (20, 0, 16 * 4, 0), num_pages=6)
    err, before = flag(), pages.block_table.clone()
    pages.fork(ints([0]), ints([1]), error_flag=err)
    assert err.item() == 8 and torch.equal(pages.block_table, before) and pages.seq_lens.tolist() == [20, 0, 64, 0]
    err.zero_()
    pages.fork(ints([2]), ints([1]), error_flag=err)  # whole pages only: none needed
    assert err.item() == 0 and pages.refcounts.tolist() == [1, 1, 2, 2, 2, 2]


def test_pages_free_reports_what_is_not_there(kvx):
    pages, _ = small(kvx)
    err = flag()
    pages.free(ints([9, -1]), error_flag=err)
    assert err.item() == 2 and pages.refcounts.tolist() == [1, 1, 1, 1, 0, 0, 0]
    pages.block_table[1, 0], pages.block_table[1, 1] = 6, 77  # a free page, an unknown one
    err.zero_()
    pages.free(ints([1, 0]), error_flag=err)
    assert err.item() == 2 and pages.refcounts.tolist() == [0, 0, 1, 1, 0, 0, 0]


def test_pages_compact_reports_unknown_entries(kvx):
    pages, _ = small(kvx)
    pages.free(ints([0]))  # pages 2, 3 move to 0, 1
    pages.block_table[3, 0], pages.block_table[3, 1] = 5, 1000
    err, live = flag(), flag()
    pages.compact(num_live=live, error_flag=err)
    assert err.item() == 2 and live.item() == 2
    assert pages.block_table.tolist() == [[-1] * 4, [-1] * 4, [0, 1, -1, -1], [5, 1000, -1, -1]]
    pages.compact()
    assert pages.refcounts.tolist() == [1, 1, 0, 0, 0, 0, 0]


def test_pages_of_a_large_pool(kvx):
    """More pages than one step of the plan's scan, reference counts that do
    not start on a 16-byte boundary."""
    n = 40000
    rng = np.random.RandomState(5)
    model = Model(n, 3, 8000)
    held = rng.permutation(n)[:17000]
    for i, row in enumerate(np.array_split(held, 3)):
        model.bt[i][:len(row)] = row.tolist()
        model.lens[i] = 16 * len(row) - (3 if i else 0)
    for p in held:
        model.refs[p] = 1
    pool, _ = tagged_pools(n, 1, 1, "f16")
    refs = torch.zeros(n + 1, dtype=torch.int32, device="cuda")[1:]
    refs.copy_(ints(model.refs))
    pages = kvx.pages.Pages(refs, ints(model.bt), ints(model.lens), list(pool))
    live, grow = flag(), [100, 0, 5000]
    pages.reserve(ints(grow))
    model.reserve(grow)
    pages.compact(num_live=live)
    assert live.item() == model.compact()
    assert_books(pages, model, pool, None, "f16")


def test_pages_copy(kvx):
    for kind in ("i8", "f16", "f32"):
        pool, stats = tagged_pools(20, 3, 5, kind)
        pages = kvx.pages.Pages.empty(20, 1, 1, list(pool), None if stats is None else list(stats))
        want = pool.clone()
        err = flag()
        pages.copy(ints([3, 3, 7, 9]), ints([10, 0, 7, 11]), error_flag=err)
        want[:, [10, 0, 11]] = want[:, [3, 3, 9]]
        assert torch.equal(pool, want) and err.item() == 0
        pages.copy(ints([3, 20, -1]), ints([20, 1, 2]), error_flag=err)
        assert torch.equal(pool, want) and err.item() == 2
        if stats is not None:
            assert stats[2, 10, 0, 0, 0] == 3.25 and stats[2, 9, 0, 0, 0] == 9.25


# --------------------------------------------------------------- all at once ---

def test_a_serving_loop(kvx):
    """Prompts, a fork into samples, steps of drafted tokens, sequences that
    end, a compaction: every step's attention against 64 bits over the cache
    as it stands, and the same bits before and after the compaction."""
    g, hq, hkv, layers, rows, max_pages, num_pages = gen(99), 12, 4, 2, 6, 24, 90
    pool = torch.zeros(layers, num_pages, 2, hkv, 16, 128, dtype=torch.int8, device="cuda")
    stats = torch.zeros(layers, num_pages, 2, hkv, 4, device="cuda")
    pages = kvx.pages.Pages.empty(num_pages, rows, max_pages, list(pool), list(stats))
    table = kvx.rope_table(128, scaling="llama3", factor=8.0)
    err = flag()

    def step(new):
        start = [0]
        for n in new:
            start.append(start[-1] + n)
        ctx = pages.seq_lens.clone()
        pages.reserve(ints(new), error_flag=err)
        outs = []
        for layer in range(layers):
            packed = normal(g, start[-1], hq + 2 * hkv, 128)
            q, k, v = packed[:, :hq], packed[:, hq:hq + hkv], packed[:, hq + hkv:]
            qr = kvx.rope_append(pool[layer], pages.block_table, ints(start), ctx, k, v, q=q, table=table, stats=stats[layer],
                                 error_flag=err)
            out = kvx.attend_chunk(pool[layer], pages.block_table, ints(start), ctx, qr, stats=stats[layer], error_flag=err)
            assert_attended(out, attend64(pool[layer], stats[layer], pages.block_table.cpu().numpy(), start, ctx.tolist(), qr))
            outs.append((qr, out))
        pages.seq_lens += ints(new)
        return start, ctx, outs

    step([100, 33, 16, 0, 0, 0])
    pages.fork(ints([0, 0, 1]), ints([3, 4, 5]), error_flag=err)
    step([4, 1, 0, 4, 4, 1])
    pages.free(ints([0, 2]), error_flag=err)
    start, ctx, outs = step([0, 3, 0, 1, 17, 2])
    live = flag()
    pages.compact(num_live=live, error_flag=err)
    assert live.item() == int((pages.refcounts > 0).sum()) == int((pages.refcounts[: live.item()] > 0).sum())
    for layer, (qr, out) in enumerate(outs):
        again = kvx.attend_chunk(pool[layer], pages.block_table, ints(start), ctx, qr, stats=stats[layer], error_flag=err)
        assert torch.equal(again, out)
    step([7, 1, 0, 1, 1, 1])
    assert err.item() == 0


@pytest.mark.parametrize("prompt", [1, 9, 90])
def test_calls_in_a_row_see_each_other(kvx, prompt):
    """Appends, decodes (which start early and read their pages and queries
    before the launch before them has ended), attention and forks on one
    stream: the bits of the same calls with a wait after each."""
    g, hq, hkv, layers, rows, max_pages = gen(55), 24, 8, 12, 32, 40
    pool0 = torch.randint(-128, 128, (layers, rows * max_pages, 2, hkv, 16, 128), generator=g, dtype=torch.int8, device="cuda")
    stats0 = torch.rand(layers, rows * max_pages, 2, hkv, 4, generator=g, device="cuda") * 0.02
    packed = normal(g, layers, rows * prompt, hq + 2 * hkv, 128)
    lens0 = [0 if prompt > 16 and i % 2 else 37 * i % 500 for i in range(rows)]
    start, table = ints(range(0, rows * prompt + 1, prompt)), kvx.rope_table(128)
    last = torch.arange(prompt - 1, rows * prompt, prompt, device="cuda")
    results = []
    for wait in (torch.cuda.synchronize, lambda: None):
        pool, stats = pool0.clone(), stats0.clone()
        pages = kvx.pages.Pages.empty(rows * max_pages, rows, max_pages, list(pool), list(stats))
        pages.reserve(ints([n + prompt for n in lens0]))
        ctx, outs = ints(lens0), []
        after = ctx + prompt
        qr = torch.empty(rows * prompt, hq, 128, dtype=F16, device="cuda")
        torch.cuda.synchronize()
        for layer in range(layers):
            x = packed[layer]
            kvx.rope_append(pool[layer], pages.block_table, start, ctx, x[:, hq:hq + hkv], x[:, hq + hkv:], q=x[:, :hq], q_out=qr,
                            table=table, stats=stats[layer])
            wait()
            if prompt == 1:
                outs.append(kvx.decode(pool[layer], pages.block_table, after, qr, stats=stats[layer]))
                wait()
            out = kvx.attend_chunk(pool[layer], pages.block_table, start, ctx, qr, stats=stats[layer])
            wait()
            outs.append(out)
            outs.append(kvx.decode(pool[layer], pages.block_table, after, out if prompt == 1 else out[last], stats=stats[layer]))
            wait()
        pages.seq_lens += after
        pages.free(ints([3]))
        wait()
        pages.fork(ints([0]), ints([3]))
        wait()
        outs.append(kvx.decode(pool[0], pages.block_table, pages.seq_lens, packed[0, :rows, :hq].contiguous(), stats=stats[0]))
        torch.cuda.synchronize()
        results.append(outs)
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_a_captured_decode_step(kvx):
    """One step (append, attend, reserve of the next) as a CUDA graph: replays
    give what eager calls give."""
    g, rows = gen(7), 3
    sets = []
    for _ in range(2):
        pool, stats = tagged_pools(40, 1, 2, "i8")
        pages = kvx.pages.Pages.empty(40, rows, 8, list(pool), list(stats))
        pages.reserve(ints([20, 1, 47]))
        sets.append((pool, stats, pages))
    packed = normal(g, rows, 12, 128)
    table = kvx.rope_table(128)
    one, start = ints([1, 1, 1]), ints([0, 1, 2, 3])
    ws = kvx.attend_chunk_workspace(rows, rows, 8, 2, 8)

    def decode(pool, stats, pages, out):
        pages.reserve(one)
        qr = kvx.rope_append(pool[0], pages.block_table, start, pages.seq_lens, packed[:, 8:10], packed[:, 10:], q=packed[:, :8],
                             table=table, stats=stats[0])
        kvx.attend_chunk(pool[0], pages.block_table, start, pages.seq_lens, qr, stats=stats[0], out=out, workspace=ws)
        pages.seq_lens.add_(one)

    outs = [torch.zeros(rows, 8, 128, dtype=F16, device="cuda") for _ in sets]
    decode(*sets[0], outs[0])
    decode(*sets[1], outs[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        decode(*sets[1], outs[1])
    for i in range(20):
        packed.copy_(normal(gen(100 + i), *packed.shape))
        decode(*sets[0], outs[0])
        graph.replay()
        assert torch.equal(outs[0], outs[1])
    for a, b in zip(sets[0][:2], sets[1][:2]):
        assert torch.equal(a, b)
    assert torch.equal(sets[0][2].block_table, sets[1][2].block_table)
