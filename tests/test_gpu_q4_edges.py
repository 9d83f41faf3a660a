"""4-bit products where they can lose what counts: vectors with a few large values
beside small ones, tiny vectors, values that are not finite, on every tile of the
matrix-core kernel and in the decode kernel.

Tolerances, u = 2^-24. The matrix-core kernel (every product with the outputs' rows
first, layout 1) takes a value as two f16 numbers after a power of two that puts the
largest of its 128 columns at 2^6 or more: off by 2^-23 of it, or by half a step of
2^-24, 2^-31 of that largest; where the power is kept within 2^64 of the one that put
the vector's largest there, by 2^-(25 + 64 + 6) of that. The decode kernel takes integers of at most 2^30 for a block whose largest value
is at least 2^29 of them: off by half a step, 2^-30 of the block's largest. A row with a single weight of 1 gives the value itself: both, and a unit
for the sum of the two parts; nothing of the other columns' sizes.
"""
import numpy as np
import pytest

import mmhip as mm
import step_ends_reference as ref
from step_reference import At, Buffers, U

pytestmark = pytest.mark.gpu

TYPES = [mm.Q4_0, mm.IQ4_NL]
# A (vectors, rows, columns) for each tile of the matrix-core kernel on 256 CUs: vectors in 16s, weight tiles a wave, waves
# that share x, groups of columns.
TILES = {"1118": (6, 64, 4128), "1124": (20, 64, 2176), "1144": (16, 8200, 672), "1244": (40, 5500, 2048),
         "1242": (40, 5500, 672), "2182": (40, 11000, 672), "1241": (16, 65600, 352), "2281": (40, 22000, 352),
         "4281": (250, 10250, 352)}


def product(ctx, raw, t, x, rows, layout):
    """[batch, rows]"""
    batch, cols = x.shape
    wt = ctx.upload(raw, t, rows, cols)
    with Buffers(ctx) as d:
        dy = d.put(np.full(batch * rows, 7.0, np.float32))
        ctx.qmm_dev(wt, 0, d.put(x), dy, batch, layout)
        ctx.synchronize()
        y = dy.to_numpy(np.float32, batch * rows)
    wt.free()
    return y.reshape(batch, rows) if layout == 0 else np.ascontiguousarray(y.reshape(rows, batch).T)


def picking(t, rows, cols):
    """Weights of which row r has a single 1, at column at[r] (Q4_0), or 1 in the block around it (IQ4_NL, which has no 0)."""
    at = np.arange(rows) * 37 % cols
    blk = np.zeros((rows, cols // 32, 18), np.uint8)
    one = np.array([1.0], np.float16).view(np.uint8)
    if t == mm.Q4_0:
        blk[..., :2], blk[..., 2:] = one, 0x88
        j = at % 32
        blk[np.arange(rows), at // 32, 2 + j % 16] = np.where(j < 16, 0x89, 0x98)
    else:
        blk[..., 2:] = 0x88
        blk[np.arange(rows), at // 32, :2] = one
    return blk.reshape(-1), at


def largest_of(x, n):
    """|x|'s largest in each run of n columns, for every column."""
    pad = -(-x.shape[1] // n) * n
    b = np.zeros((len(x), pad))
    b[:, :x.shape[1]] = np.abs(x)
    return np.repeat(b.reshape(len(x), -1, n).max(-1), n, 1)[:, :x.shape[1]]


def check_picked(y, x, t, at, run, step):
    """y against the values (or block sums) that the rows pick; run columns share a step of `step` of their largest."""
    x = x.astype(np.float64)
    off = 2 * U * np.abs(x) + step * largest_of(x, run) + 2.0 ** -95 * np.abs(x).max(1, keepdims=True)
    if t == mm.Q4_0:
        want, tol = x[:, at], off[:, at] + U * np.abs(x[:, at])
    else:  # 32 values: 64 parts summed, each sum rounded by a unit at most
        want = x.reshape(len(x), -1, 32).sum(-1)[:, at // 32]
        tol = (off + 66 * U * np.abs(x)).reshape(len(x), -1, 32).sum(-1)[:, at // 32]
    err, tol = np.abs(y - want), tol + 2.0 ** -149
    assert (err <= tol).all(), (err / tol).max()


def uneven(rng, batch, cols):
    """Vectors with one value 10^3 to 10^25 times as large as the rest, first ones among them, and some with several."""
    x = rng.standard_normal((batch, cols)).astype(np.float32)
    where = [3, 40, 63, 64, 100, cols - 1, cols // 2, 130]
    size = [1e3, 1e4, 1e5, 1e6, 1e9, 1e25]
    for b in range(1, batch):
        x[b, where[b % 8]] = size[b % 6] * (-1) ** (b // 3)
        if b % 5 == 0:
            x[b, where[(b + 3) % 8]] = -size[(b + 1) % 6]
        if b % 7 == 0:
            x[b, :64] *= np.float32(1e-6)
        if b % 11 == 0:
            x[b, 64:192] = 0
    return x


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("tile", sorted(TILES))
def test_large_values_cost_others_nothing(ctx, t, tile):
    batch, rows, cols = TILES[tile]
    x = uneven(np.random.default_rng(batch), batch, cols)
    raw, at = picking(t, rows, cols)
    check_picked(product(ctx, raw, t, x, rows, 1), x, t, at, 128, 2.0 ** -31)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("batch", [1, 3, 4, 21])
def test_large_values_in_the_decode_kernel(ctx, t, batch):
    rows, cols = 500, 2080
    x = uneven(np.random.default_rng(batch), batch, cols)
    raw, at = picking(t, rows, cols)
    check_picked(product(ctx, raw, t, x, rows, 0), x, t, at, 32, 2.0 ** -30)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("layout,batch", [(0, 1), (0, 4), (0, 22), (1, 1), (1, 22), (1, 70)])
@pytest.mark.parametrize("size", [1e-30, 1e-36, 1e-38, 1e-42])
def test_tiny_vectors(ctx, t, layout, batch, size):
    """Down to f32's subnormal numbers, of which the last has 10 bits: nothing is flushed."""
    rng = np.random.default_rng(batch)
    rows, cols = 300, 1056
    x = (rng.standard_normal((batch, cols)) * size).astype(np.float32)
    x[:, 32:64] = 0
    x[:, 64:128] *= np.float32(1e-2)
    x[batch // 2, :256] = 0
    raw, at = picking(t, rows, cols)
    check_picked(product(ctx, raw, t, x, rows, layout), x, t, at, 128 if layout else 32, 2.0 ** (-31 if layout else -30))


def definition(x, w):
    """The sums of w x, and of |w x|: x [batch, cols], w [rows, cols] in 64 bits, of which some are not finite."""
    at = ~(np.isfinite(x).all(0) & np.isfinite(w).all(0))
    fx, fw = np.where(at, 0.0, x), np.where(at, 0.0, w)
    y, s = fx @ fw.T, np.abs(fx) @ np.abs(fw).T
    for c in np.flatnonzero(at):
        term = x[:, c, None] * w[:, c]
        y, s = y + term, s + np.abs(term)
    return y, s


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("tile", sorted(TILES) + ["decode1", "decode4", "fours"])
def test_what_is_not_finite_follows_the_definition(ctx, t, tile):
    """Infinite values times weights of either sign and 0, infinite and NaN scales, sums that only 64 bits hold: the
    definition's infinity or NaN in their results, and nothing of them in the others."""
    batch, rows, cols = TILES.get(tile) or {"decode1": (1, 700, 2080), "decode4": (4, 700, 2080), "fours": (22, 700, 544)}[tile]
    rng = np.random.default_rng(rows)
    raw = mm.make_weight(rng, t, rows, cols).reshape(rows, cols // 32, 18)
    big = np.array([65504.0], np.float16).view(np.uint8)
    raw[3, 1, :2] = np.array([np.inf], np.float16).view(np.uint8)
    raw[20 % rows, 2, :2] = np.array([-np.inf], np.float16).view(np.uint8)
    raw[37 % rows, 0, :2] = np.array([np.nan], np.float16).view(np.uint8)
    raw[40:44, :, :2], raw[40:44, :, 2:] = big, rng.integers(0, 256, (4, 1, 16))  # rows of alike blocks
    x = rng.standard_normal((batch, cols)).astype(np.float32)
    odd = [lambda v: v.__setitem__(5, np.inf), lambda v: v.__setitem__(cols - 1, -np.inf), lambda v: v.__setitem__(64, np.nan),
           lambda v: v.__setitem__([70, 90], np.inf), lambda v: v.__setitem__([3, 99], [np.inf, -np.inf]),
           # the first half's values again with the other sign: sums beyond f32 that cancel in rows of alike blocks
           lambda v: (v.__setitem__(slice(None), 0), v.__setitem__(slice(0, 32), 3e38), v.__setitem__(slice(64, 96), -3e38))]
    with np.errstate(invalid="ignore"):
        for b in range(batch):
            if batch == 1 or b % 3 == 1:
                odd[(b // 3 + rows) % 6](x[b])
    w = ref.values_4bit(raw, t).reshape(rows, cols)
    y = product(ctx, raw.reshape(-1), t, x, rows, 1 if tile in TILES else 0)
    with np.errstate(over="ignore", invalid="ignore"):
        want, s = definition(x.astype(np.float64), w)
        want32 = want.astype(np.float32)
    fine = np.isfinite(want32)
    assert np.array_equal(np.isnan(y), np.isnan(want32))
    assert np.array_equal(y[~fine & ~np.isnan(y)], want32[~fine & ~np.isnan(want32)])
    tol = (cols / 32 + 200) * U * s + 2.0 ** -30 * cols * np.abs(x).max(1, keepdims=True, where=np.isfinite(x), initial=0) * np.max(
        np.where(np.isfinite(w), np.abs(w), 0), 1)
    with np.errstate(invalid="ignore"):
        err = np.where(fine, np.abs(y - want), 0)
    bad = fine & ~(err <= tol)
    assert (fine.any() or batch == 1) and not bad.any(), [(i, y[tuple(i)], want[tuple(i)], s[tuple(i)], tol[tuple(i)]) for i in np.argwhere(bad)[:9]]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("layout,batch", [(0, 1), (0, 3), (0, 24), (1, 1), (1, 24), (1, 100)])
def test_all_bits_of_a_value(ctx, t, layout, batch):
    """One value of 23 bits in each block: it comes out as it is. (Two f16 numbers hold it: of the values' 4096 .. 8191 the
    nearest multiple of 4, and what that leaves, at most 2 in steps of 2^-10; a block's integers hold 30 bits.)"""
    rng = np.random.default_rng(batch)
    rows, cols = 320, 1056
    x = np.zeros((batch, cols), np.float32)
    x[:, rng.integers(0, 32, cols // 32) + np.arange(0, cols, 32)] = (
        rng.integers(1 << 22, 1 << 23, (batch, cols // 32)) * np.float32(2.0 ** -22) * rng.choice([-1, 1], (batch, cols // 32)))
    raw, at = picking(mm.IQ4_NL, rows, cols)  # whole blocks of ones
    if t == mm.Q4_0:
        raw = raw.reshape(rows, -1, 18)
        raw[..., 2:] = 0x99
        raw = raw.reshape(-1)
    assert np.array_equal(product(ctx, raw, t, x, rows, layout), x.reshape(batch, -1, 32).sum(-1)[:, at // 32])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("batch", [2, 4, 5, 7, 15, 16, 17, 32, 33, 40])
@pytest.mark.parametrize("rows,cols", [(17, 96), (100, 544), (64, 2176), (500, 4128)])
def test_fours_are_as_exact_as_one_vector(ctx, t, batch, rows, cols):
    """Shapes of up to two workgroups per CU. A block's sum: two roundings of the digits' sums, one of both together, one
    with its scale, one with the others, the last one in up to cols / 32 blocks, eight waves' parts and three chunks one after
    the other; the values themselves are off by 2^-30 of their block's largest."""
    rng = np.random.default_rng(batch * 31 + rows)
    raw = mm.make_weight(rng, t, rows, cols)
    w = np.abs(ref.values_4bit(raw, t).reshape(rows, cols))
    x = rng.standard_normal((batch, cols)).astype(np.float32)
    x[:, rng.integers(0, cols, cols // 32)] *= 300
    y = product(ctx, raw, t, x, rows, 0)
    x = x.astype(np.float64)
    want = x @ ref.values_4bit(raw, t).reshape(rows, cols).T
    tol = (cols / 32 + 4 + 8 + 3) * U * (np.abs(x) @ w.T) + (2.0 ** -30 + 2.0 ** -38) * (largest_of(x, 32) @ w.T)
    err = np.abs(y - want)
    assert (err <= tol).all(), (err / tol).max()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("batch", [1, 20, 70])
@pytest.mark.parametrize("size", [1e-38, 1.0, 1e30, 1e38])
def test_sizes_of_vectors_and_scales_on_the_matrix_cores(ctx, t, batch, size):
    """Scales of 0, of f16's largest and smallest, beside vectors of all sizes; results beyond f32 are infinite."""
    rng = np.random.default_rng(9)
    rows, cols = 500, 1056
    raw = mm.make_weight(rng, t, rows, cols).reshape(rows, cols // 32, 18)
    for r, d in ((3, 65504.0), (5, 6e-8), (7, 0.0)):
        raw[r, 4:6, :2] = np.array([d], np.float16).view(np.uint8)
    w = ref.values_4bit(raw, t).reshape(rows, cols)
    x = (rng.standard_normal((batch, cols)) * size).clip(-3e38, 3e38).astype(np.float32)
    x[:, 32:64] = 0
    x[:, 64:96] *= np.float32(1e-3)
    y = product(ctx, raw.reshape(-1), t, x, rows, 1)
    x = x.astype(np.float64)
    want, s = x @ w.T, np.abs(x) @ np.abs(w).T
    # each of a block's 64 products and its sums is rounded by a unit at most, as each block's sum; subnormal results by 2^-150
    tol = (cols / 32 + 200) * U * s + 2.0 ** -31 * (largest_of(x, 128) @ np.abs(w).T) + 2.0 ** -149
    with np.errstate(over="ignore"):
        inf = np.abs(want.astype(np.float32)) == np.inf
    sure = np.abs(np.abs(want) - 2.0 ** 128) > tol
    assert np.array_equal((np.abs(y) == np.inf)[sure], inf[sure])
    ok = ~inf & np.isfinite(y)
    assert (np.abs(y.astype(np.float64) - want)[ok] <= tol[ok]).all()


@pytest.mark.parametrize("t", [mm.Q4_0, mm.IQ4_NL, mm.Q8_0, mm.F32])
def test_ranges_of_matrices_that_wrap(ctx, t):
    """A first matrix whose sum with their number goes round 2^64 is refused like any other beyond the stack."""
    wt = ctx.upload(mm.make_weight(np.random.default_rng(1), t, 16, 64, 3), t, 16, 64, 3)
    with Buffers(ctx) as d:
        x, y = d.new(64 * 4, 0), d.put(np.full(3 * 16, 7.0, np.float32))
        for first, n in ((2 ** 64 - 1, 1), (2 ** 64 - 2, 3), (2, 2 ** 64 - 1), (3, 1), (0, 4), (2 ** 63, 2 ** 63)):
            with pytest.raises(mm.MmhipError, match="out of range") as e:
                ctx.gemv_batched_dev(wt, first, n, x, 0, y, 16)
            assert e.value.code == mm.ERR_INVALID
        ctx.synchronize()
        assert (y.to_numpy(np.float32, 48) == 7).all()
    wt.free()
