"""Limits of the 8-bit serving operators against 64 bits: blocks of one value,
blocks with outliers, distant keys, sums over many keys, statistics far apart,
explicit streams, failures of a launch, lengths next to the largest int."""
import ctypes as C
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_operators import (E16, E32, F16, F32, F64, TINY16, assert_attended, assert_turned, attend64, attend_case,  # noqa: E402
                                flag, gen, ints, kvx, layout_of, normal, small)

assert kvx  # the fixture


# ------------------------------------------------- blocks of one value ---

def as_scale_zero(stats):
    """The same values: a block of one value v is stored as scale 1, codes
    -128, zero point v; scale 0, zero point v says it without a product."""
    one = (stats[..., 0] == stats[..., 1])[..., None] & torch.tensor([False, False, True, False], device="cuda")
    return torch.where(one, 0.0, stats)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("ctx,new", [([0], [2]), ([0, 0], [1, 5]), ([30], [3]), ([0], [33]), ([40, 500], [90, 128]), ([700], [300])])
def test_attend_over_blocks_of_one_value(kvx, dtype, ctx, new):
    """V all zero, or one value, or K of padding (zeros) in some pages, as the
    append stores them."""
    bt, num_pages, start = layout_of(ctx, new, 5)
    total = [c + n for c, n in zip(ctx, new)]
    g = gen(91)
    for value in (0.0, 3.25, -700.0):
        pool = torch.zeros(num_pages, 2, 2, 16, 128, dtype=torch.int8, device="cuda")
        stats = torch.zeros(num_pages, 2, 2, 4, device="cuda")
        k = normal(g, sum(total), 2, 128, dtype=dtype)
        k[::2] *= (torch.arange(len(k[::2]), device="cuda") // 40 % 2)[:, None, None]
        k[16:32] = 0  # whole pages of zeros among the others
        v = torch.full_like(k, value)
        kvx.rope_append(pool, ints(bt), ints(np.concatenate(([0], np.cumsum(total)))), ints([0] * len(ctx)), k, v, stats=stats)
        q = normal(g, int(start[-1]), 8, 128, dtype=dtype)
        out = kvx.attend_chunk(pool, ints(bt), ints(start), ints(ctx), q, stats=stats)
        # sums of p and of p v round alike: 64 steps bound them by far
        tol = abs(value) * (64 * 2.0 ** -23 + (E16 if dtype == F16 else E32))
        assert ((out.double() - value).abs() <= tol).all(), f"{value}: off by {(out.double() - value).abs().max():.3e}"
        assert_attended(out, attend64(pool, as_scale_zero(stats), bt, start, ctx, q))


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("ctx,new", [([60], [3]), ([40, 500], [90, 128])])
def test_attend_over_keys_of_one_value(kvx, dtype, ctx, new):
    """K of zeros everywhere: the mean of V; and in every other page only."""
    pool, stats, bt, start, q = attend_case(92, ctx, new, 8, 2, dtype)
    zeros = torch.tensor([0.0, 0.0, 1.0, 0.0], device="cuda")
    for step in (1, 2):
        stats[::step, 0] = zeros
        pool[::step, 0] = -128
        out = kvx.attend_chunk(pool, ints(bt), ints(start), ints(ctx), q * 16, stats=stats)
        assert_attended(out, attend64(pool, as_scale_zero(stats), bt, start, ctx, q * 16))


# ------------------------------------------------- precision of P V ---

def one_hot_q(g, rows, hq, dtype):
    """Queries with one element, a power of two: a score has no more than a
    few roundings, so that those of P V show."""
    q = torch.zeros(rows, hq, 128, dtype=dtype, device="cuda")
    at = torch.randint(0, 128, (rows, hq, 1), generator=g, device="cuda")
    size = torch.exp2(torch.randint(-2, 4, (rows, hq, 1), generator=g, device="cuda").float())
    sign = torch.randint(0, 2, (rows, hq, 1), generator=g, device="cuda") * 2 - 1
    return q.scatter_(2, at, (size * sign).to(dtype))


def assert_attended_closely(got, ref, floor=0.0):
    """With one_hot_q.  A score: two products, a sum, the maximum taken from
    it, each half a step of 2^-23 of what it adds up to (noise, twice with the
    maximum; in powers of two 1.45 times that), and the exponential 2^-21;
    once more through the sum.  A weight in high and low part is off by 2^-21,
    the sum of the second product by 64 steps of 2^-23 (truncated, or a random
    walk of more).  Then the output's rounding."""
    out, size, noise = ref
    eps = 16 * 2.0 ** -24 * noise + 2.0 ** -21
    tol = (2 * eps + 64 * 2.0 ** -23 + 2.0 ** -21) * size + floor
    tol = tol + ((E16 * (out.abs() + tol) + TINY16) if got.dtype == F16 else E32 * out.abs())
    bad = ~((got.double() - out).abs() <= tol)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} elements off, worst {(got.double() - out).abs().max():.3e}, "
                           f"{((got.double() - out).abs() / tol).max():.1f} of the bound")


def outlier_case(seed, ctx, new, hq, hkv, dtype):
    """1 % of V a hundred times the rest: the scale is the outliers'."""
    def spread(g, pages, hkv):
        s = torch.ones(pages, 2, hkv, 16, 128, device="cuda")
        s[:, 1][torch.rand(pages, hkv, 16, 128, generator=g, device="cuda") < 0.01] = 100.0
        return s
    pool, stats, bt, start, _ = attend_case(seed, ctx, new, hq, hkv, dtype, spread)
    return pool, stats, bt, start, one_hot_q(gen(seed), int(start[-1]), hq, dtype)


CLOSE = [([0], [2]), ([1], [1]), ([31], [2]), ([127], [1]), ([500], [4]), ([0], [40]), ([100], [33]), ([500, 3], [128, 300]), ([2000], [100])]


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("hq,hkv", [(8, 2), (24, 8)])
@pytest.mark.parametrize("ctx,new", CLOSE)
def test_attend_over_blocks_with_outliers(kvx, dtype, ctx, new, hq, hkv):
    pool, stats, bt, start, q = outlier_case(93 + sum(new), ctx, new, hq, hkv, dtype)
    out = kvx.attend_chunk(pool, ints(bt), ints(start), ints(ctx), q, stats=stats)
    assert_attended_closely(out, attend64(pool, stats, bt, start, ctx, q))


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("hq,hkv", [(8, 2), (24, 8), (32, 2)])
def test_attend_agrees_with_decode_over_outliers(kvx, dtype, hq, hkv):
    """A token attended alone and as the last of 40: what the calls round, no
    more; and decoded, within the decode's own bound."""
    ctx = [0, 31, 100, 511, 2000]
    pool, stats, bt, start, q = outlier_case(97, ctx, [1] * len(ctx), hq, hkv, dtype)
    args = pool, ints(bt)
    single = kvx.attend_chunk(*args, ints(start), ints(ctx), q, stats=stats)
    decoded = kvx.decode(*args, ints([c + 1 for c in ctx]), q, stats=stats)
    # the same token as the last of 40 (the others' queries do not matter)
    group = [max(c - 39, 0) for c in ctx]
    counts = [c + 1 - a for c, a in zip(ctx, group)]
    many_start = np.concatenate(([0], np.cumsum(counts))).astype(np.int32)
    many_q = torch.zeros(int(many_start[-1]), hq, 128, dtype=dtype, device="cuda")
    last = torch.tensor(many_start[1:] - 1, dtype=torch.int64, device="cuda")
    many_q[last] = q
    many = kvx.attend_chunk(*args, ints(many_start), ints(group), many_q, stats=stats)[last]
    ref = attend64(pool, stats, bt, start, ctx, q)
    for got in (single, many):
        assert_attended_closely(got, ref)
        assert ((got - decoded).float().abs() <= 1e-2 + 1e-3 * decoded.float().abs()).all()


# ------------------------------------------------- distant keys ---

@pytest.mark.parametrize("new", [1, 60])
@pytest.mark.parametrize("far,bits", [(13, 20), (24, 14), (30, 8)])
def test_attend_distant_keys_count(kvx, new, far, bits):
    """Key 0 takes nearly all of the weight and has a V of nearly nothing;
    30,000 others have 2^-far of it each and V of 1.37.  Scores are exact; a
    weight times the scale of V still has that many bits."""
    ctx, hq, hkv = 30000, 8, 2
    bt, num_pages, start = layout_of([ctx], [new], 7)
    g = gen(98)
    pool = torch.randint(-128, 128, (num_pages, 2, hkv, 16, 128), generator=g, device="cuda", dtype=torch.int8)
    stats = torch.zeros(num_pages, 2, hkv, 4, device="cuda")
    first = int(bt[0, 0])
    pool[:, 0, :, :, 0] = -128  # K: element 0 is 0 but for key 0's
    pool[first, 0, :, 0, 0] = 127
    stats[:, 0] = torch.tensor([0.0, 2.55, 2.55 / 255, 0.0], device="cuda")
    stats[first, 0] = torch.tensor([0.0, far, far / 255, 0.0], device="cuda")
    pool[:, 1, :, :, :64] = 127
    stats[:, 1] = torch.tensor([-1.37, 1.37, 2.74 / 255, -1.37], device="cuda")
    stats[first, 1] *= 2.0 ** -20
    q = torch.zeros(new, hq, 128, dtype=F32, device="cuda")
    q[..., 0] = 1.0
    out = kvx.attend_chunk(pool, ints(bt), ints([0, new]), ints([ctx]), q, stats=stats, sm_scale=math.log(2.0))
    ref = attend64(pool, stats, bt, [0, new], [ctx], q, scale=math.log(2.0))
    others = ctx * 2.0 ** -far
    # key 0's own V, up to 1.37 * 2^-20, is 3.5 % of the others' 2^-30 * 30,000 * 1.37
    assert ref[0][0, 0, 0].item() == pytest.approx(1.37 * others / (1 + others), rel=4e-2)
    assert_attended_closely(out, ref, floor=2.0 ** -bits * ref[0][0, 0, 0].item())


# ------------------------------------------------- sums over many keys ---

@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("batch,ctx,new,hq,hkv", [(1, 30000, 1184, 16, 2), (1, 30000, 40, 16, 2), (300, 30000, 1, 8, 2), (150, 31000, 17, 8, 1),
                                                       (1, 60000, 2368, 16, 2), (148, 120000, 16, 8, 1)])
def test_attend_sums_of_one_sign(kvx, dtype, batch, ctx, new, hq, hkv):
    """Flat scores and a V with one element at the top of its block's range in
    every token, one at the bottom: sums that only grow, over 30,000 to 120,000
    keys in one piece (as many row tiles as SMs; of 256 and of 128 rows), in
    several, in the few rows' kernel."""
    pages = (ctx + new + 15) // 16
    g = gen(99)
    pool = torch.randint(-128, 128, (pages, 2, hkv, 16, 128), generator=g, device="cuda", dtype=torch.int8)
    pool[:, 1, ..., 0], pool[:, 1, ..., 1] = 127, -128
    size = torch.rand(pages, 2, hkv, generator=g, device="cuda") / 4 + 0.75
    stats = torch.stack((-size, size, 2 * size / 255, -size), -1).contiguous()
    bt = ints(list(range(pages))).expand(batch, pages).contiguous()
    q = torch.zeros(batch * new, hq, 128, dtype=dtype, device="cuda")
    start = ints([new * i for i in range(batch + 1)])
    out = kvx.attend_chunk(pool, bt, start, ints([ctx] * batch), q, stats=stats)
    st = stats[:, 1].double()
    v = st[..., 3, None, None] + (pool[:, 1].double() + 128) * st[..., 2, None, None]  # [pages][hkv][16][128]
    v = v.permute(0, 2, 1, 3).reshape(-1, hkv, 128)[:ctx + new]
    want = (v.cumsum(0) / torch.arange(1, len(v) + 1, device="cuda")[:, None, None])[ctx:]
    want = want.repeat_interleave(hq // hkv, 1).repeat(batch, 1, 1)
    # An MMA takes up to 2^-21 off the sum it adds to; off a sum that grows
    # evenly, half of that on average: 2^-22 each.  Up to 32 (fp32: 8) key tiles
    # of 128 go into one sum, 16 (fp32: 8) MMAs each.
    off = 512 * 2.0 ** -22 if dtype == F16 else 64 * 2.0 ** -22
    err = (out.double() - want).abs()
    print(f"{dtype} {batch} x {new}: worst {err.max().item():.3e}, elements 0, 1: {err[..., :2].max().item():.3e}")
    assert ((out >= (want - off).to(dtype)) & (out <= (want + off).to(dtype))).all(), f"worst {err.max():.3e}"


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("batch,ctx,new,hq,hkv", [(1, 9000, 1184, 16, 2), (1, 9000, 2368, 16, 2), (148, 12000, 16, 8, 1), (1, 70000, 100, 8, 2)])
def test_attend_long_rows_in_place_with_rising_and_falling_scores(kvx, dtype, batch, ctx, new, hq, hkv):
    """Sums that were moved on and then scaled down, by a little and by more
    than a type holds, in the output's own place (out is q) and in pieces."""
    pool, stats, bt, start, q = attend_case(100 + batch, [ctx], [new], hq, hkv, dtype)
    pages = torch.tensor(bt[0][bt[0] >= 0], dtype=torch.int64, device="cuda")
    for head in range(hkv):
        ramp = torch.linspace(-3, 3, len(pages), device="cuda") * (1 if head == 0 else -1)
        if head == 0:  # and one step up of hundreds, in the middle
            ramp[len(pages) // 2:] += 200.0
        stats[pages, 0, head, 3] += ramp
    q = torch.cat([q] * batch)
    q[:, :, 0] += 3  # the ramps count the same way in every row
    bts, starts = np.concatenate([bt] * batch), np.arange(batch + 1, dtype=np.int32) * new
    args = pool, ints(bts), ints(starts), ints([ctx] * batch)
    out = kvx.attend_chunk(*args, q, stats=stats)
    got = q.clone()
    kvx.attend_chunk(*args, got, stats=stats, out=got)
    assert torch.equal(got, out)
    ref = attend64(pool, stats, bt, start, [ctx], q[:new])
    for s in range(0, batch, 49):
        assert_attended(out[s * new:(s + 1) * new], ref)


# ------------------------------------------------- statistics far apart ---

@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("ratio", [18, 24, 60])
@pytest.mark.parametrize("ctx,new", [([0, 0, 0], [40, 300, 3]), ([14, 12], [4, 90])])
def test_attend_larger_pages_behind_do_not_reach_a_row(kvx, dtype, ratio, ctx, new):
    """Rows that see a page of V, and behind it, out of their sight, pages of
    2^ratio times its range."""
    pool, stats, bt, start, q = attend_case(63 + ratio, ctx, new, 8, 2, dtype)
    for row in bt:
        for page in row[1:]:
            if page >= 0:
                stats[int(page), 1, :, 2:] *= 2.0 ** ratio
    out = kvx.attend_chunk(pool, ints(bt), ints(start), ints(ctx), q, stats=stats)
    ref = attend64(pool, stats, bt, start, ctx, q)
    rows = torch.cat([torch.arange(int(a), min(int(a) + 16 - c, int(b))) for a, b, c in zip(start, start[1:], ctx)]).cuda()
    assert_attended(out[rows], tuple(x[rows] for x in ref))


# ------------------------------------------------- keys of tiny ranges ---

@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("scale,size", [(2.0 ** -100, 1.0), (2.0 ** -100, 2.0 ** -45), (2.0 ** -70, 2.0 ** -60), (0.0, 2.0 ** -45), (2.0 ** -126, 1.0)])
def test_attend_over_keys_of_tiny_ranges(kvx, dtype, scale, size):
    """K blocks of a range next to nothing, and queries as small: the masked
    keys of a page stay masked."""
    ctx, new = [20, 300, 7], [60, 130, 3]
    pool, stats, bt, start, q = attend_case(64, ctx, new, 8, 2, dtype)
    stats[:, 0, :, 2] *= scale
    q = (q.float() * size).to(dtype)
    out = kvx.attend_chunk(pool, ints(bt), ints(start), ints(ctx), q, stats=stats)
    assert_attended(out, attend64(pool, stats, bt, start, ctx, q))


# ------------------------------------------------- streams ---

LONG = 200_000_000  # cycles: 0.1 s on a stream


def test_attend_output_on_an_explicit_stream(kvx):
    """The rows that the call fills with zeros itself are filled before its
    kernels, on their stream."""
    ctx, new = [300, 10], [6, 50]
    pool, stats, bt, start, q = attend_case(101, ctx, new, 8, 2, F16)
    args = pool, ints(bt), ints(start), ints(ctx), q
    want = kvx.attend_chunk(*args, stats=stats)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(LONG)
    got = [kvx.attend_chunk(*args, stats=stats, stream=s) for s in (side, side.cuda_stream)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in got)


def test_attend_scratch_of_two_explicit_streams(kvx, monkeypatch):
    """Scratch that a call makes itself is not given to another stream while
    the call may still use it."""
    ctx, new = [300, 10], [6, 50]
    pool, stats, bt, start, q = attend_case(102, ctx, new, 8, 2, F16)
    args = pool, ints(bt), ints(start), ints(ctx), q
    outs = [torch.zeros_like(q) for _ in range(3)]
    at, real = [], kvx.attend_chunk_workspace

    def noted(*a, **kw):
        w = real(*a, **kw)
        at.append((w.data_ptr(), w.numel()))
        return w
    monkeypatch.setattr(kvx, "attend_chunk_workspace", noted)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for s, o in zip(streams, outs):
        with torch.cuda.stream(s):
            torch.cuda._sleep(LONG)
        kvx.attend_chunk(*args, stats=stats, out=o, stream=s)
    kvx.attend_chunk(*args, stats=stats, out=outs[2])
    torch.cuda.synchronize()
    assert all(torch.equal(o, outs[2]) for o in outs)
    at.sort()
    assert len(at) == 3 and all(a + n <= b for (a, n), (b, _) in zip(at, at[1:]))


def test_rope_and_append_outputs_on_an_explicit_stream(kvx):
    """Outputs that the calls make themselves do not lie in memory that
    another stream's pending work still writes."""
    q, k = normal(gen(103), 64, 24, 128), normal(gen(104), 64, 8, 128)
    pos, table = ints(list(range(64))), kvx.rope_table(128)
    pool = torch.zeros(4, 2, 8, 16, 128, dtype=torch.int8, device="cuda")
    stats = torch.zeros(4, 2, 8, 4, device="cuda")
    bt, start, first = ints([[0, 1, 2, 3]]), ints([0, 64]), ints([0])
    want_q, want_k = kvx.rope(q, k, pos, table)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(LONG)
    for x in (q, k, q):  # freed with their fill still to come
        torch.empty_like(x).fill_(7.0)
    got_q, got_k = kvx.rope(q, k, pos, table, stream=side)
    got = kvx.rope_append(pool, bt, start, first, k, k, q=q, table=table, stats=stats, stream=side)
    torch.cuda.synchronize()
    assert torch.equal(got_q, want_q) and torch.equal(got_k, want_k) and torch.equal(got, want_q)


# ------------------------------------------------- a launch that fails ---

@pytest.mark.parametrize("tokens", [3, 5000])
def test_append_reports_a_launch_that_fails(kvx, tokens):
    """Launches into a stream whose capture has been made invalid fail on the
    host; the call says so, and works again afterwards."""
    k = normal(gen(105), tokens, 1, 128)
    q = normal(gen(106), tokens, 2, 128)
    q_out = torch.empty_like(q)
    pages = (tokens + 15) // 16
    pool = torch.zeros(pages, 2, 1, 16, 128, dtype=torch.int8, device="cuda")
    stats = torch.zeros(pages, 2, 1, 4, device="cuda")
    bt, start, first = ints([list(range(pages))]), ints([0, tokens]), ints([0])
    side = torch.cuda.Stream()

    def call():
        kvx.rope_append(pool, bt, start, first, k, k, q=q, q_out=q_out, stats=stats, stream=side)
    call()
    torch.cuda.synchronize()
    rt = C.CDLL("libcudart.so.12")
    stream, graph = C.c_void_p(side.cuda_stream), C.c_void_p()
    assert rt.cudaStreamBeginCapture(stream, 2) == 0  # relaxed
    try:
        assert rt.cudaStreamSynchronize(stream) != 0  # not allowed: the capture is void
        with pytest.raises(kvx.KvxError) as e:
            call()
        assert e.value.status == -3
    finally:
        rt.cudaStreamEndCapture(stream, C.byref(graph))
        rt.cudaGetLastError()
    call()
    torch.cuda.synchronize()
    assert torch.equal(q_out, q)


# ------------------------------------------------- lengths ---

@pytest.mark.parametrize("length", [2 ** 31 - 1, 2 ** 31 - 15, 2 ** 31 - 16, 65])
def test_pages_refuse_lengths_next_to_the_largest_int(kvx, length):
    pages, pool = small(kvx)
    pages.seq_lens[0] = length
    before = [t.clone() for t in (pages.refcounts, pages.block_table, pages.seq_lens, pool)]
    for what, args in (("fork", ([0], [1])), ("reserve", ([1, 0, 0, 0],))):
        err = flag()
        getattr(pages, what)(*(ints(a) for a in args), error_flag=err)
        assert err.item() == 4
        assert all(torch.equal(a, b) for a, b in zip(before, (pages.refcounts, pages.block_table, pages.seq_lens, pool)))


# ------------------------------------------------- gradients ---

class Turn(torch.autograd.Function):
    """kvx.rope as an operation that autograd records."""

    @staticmethod
    def forward(ctx, q, k, rope, pos, table):
        ctx.rope, ctx.pos, ctx.table = rope, pos, table
        return rope(q, k, pos, table)

    @staticmethod
    def backward(ctx, gq, gk):
        return (*ctx.rope(gq, gk, ctx.pos, ctx.table, inverse=True), None, None, None)


def test_rope_in_an_autograd_function(kvx):
    """The documented way: grad mode is off in both directions.  The gradient
    of a weighted sum against the formula's: R^T w, by the inverse."""
    g = gen(107)
    q, k = normal(g, 9, 4, 128, dtype=F32).requires_grad_(), normal(g, 9, 2, 128, dtype=F32).requires_grad_()
    wq, wk = normal(g, 9, 4, 128, dtype=F32), normal(g, 9, 2, 128, dtype=F32)
    pos, table = ints(list(range(100, 109))), kvx.rope_table(96, scaling="yarn", factor=4.0, high=32.0)
    with pytest.raises(ValueError):
        kvx.rope(q, k, pos, table)
    yq, yk = Turn.apply(q, k, kvx.rope, pos, table)
    ((yq * wq).sum() + (yk * wk).sum()).backward()
    for x, w in ((q, wq), (k, wk)):
        assert_turned(x.grad, w, pos, table, inverse=True)


# ------------------------------------------------- documented use ---

@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("ctx,new,hq,hkv", [([0], [1001], 24, 8), ([0, 0], [700, 700], 24, 8), ([0] + [600] * 9 + [0] * 6, [300] + [1] * 9 + [0] * 6, 16, 4)])
@pytest.mark.parametrize("width", [64, 2048])
def test_attend_with_a_table_wider_than_the_lengths(kvx, dtype, ctx, new, hq, hkv, width):
    """A block table of the longest context, rows of sequences that are not
    active among them: prompts, and a prompt beside single tokens."""
    pool, stats, bt, start, q = attend_case(108, ctx, new, hq, hkv, dtype)
    wide = np.full((len(ctx), width), -1, np.int32)
    wide[:, :bt.shape[1]] = bt[:, :width]
    err = flag()
    out = kvx.attend_chunk(pool, ints(wide), ints(start), ints(ctx), q, stats=stats, error_flag=err)
    assert err.item() == 0
    assert_attended(out, attend64(pool, stats, bt, start, ctx, q))


@pytest.mark.parametrize("dtype", [F16, F32])
def test_append_of_prompts_to_float_pools(kvx, dtype):
    """Prompt-sized chunks behind other lengths, 64 q-heads: the bits of the
    rotation, then of the append."""
    ctx, new = [0, 37, 16], [2731, 700, 1]
    bt, num_pages, start = layout_of(ctx, new, 9)
    g = gen(109)
    q, k, v = (normal(g, int(start[-1]), h, 128, dtype=dtype) for h in (64, 8, 8))
    pool = normal(g, num_pages, 2, 8, 16, 128, dtype=dtype)
    want = pool.clone()
    table = kvx.rope_table(128, scaling="llama3", factor=8.0)
    pos = torch.cat([torch.arange(c, c + n) for c, n in zip(ctx, new)]).int().cuda()
    tq, tk = kvx.rope(q, k, pos, table)
    for s, (c, n) in enumerate(zip(ctx, new)):
        a, b = int(start[s]), int(start[s + 1])
        kvx.append_chunk(want, ints(bt[s:s + 1]), ints([c]), tk[None, a:b].contiguous(), v[None, a:b].contiguous())
    qo = kvx.rope_append(pool, ints(bt), ints(start), ints(ctx), k, v, q=q, table=table)
    assert torch.equal(qo, tq) and torch.equal(pool, want)
