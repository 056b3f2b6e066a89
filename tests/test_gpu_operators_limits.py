"""Limits of the 8-bit serving operators against 64 bits: blocks of one value,
blocks with outliers, distant keys, sums over many keys, statistics far apart,
explicit streams, failures of a launch, lengths next to the largest int."""
import ctypes as C
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_operators import (E16, E32, F16, F32, F64, TINY16, assert_attended, attend64, attend_case, flag, gen, ints,  # noqa: E402
                                kvx, layout_of, normal, small)

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
