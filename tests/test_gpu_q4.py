"""4-bit weights with group scales (Q4_0, IQ4_NL) through the library's
products, against 64-bit ones of the exact weights.

Tolerances, u = 2^-24, S = sum |w x| of a result: few vectors (one to four here) enter as
integers of 31 bits (2^-31 of a block's largest), a block's sum is rounded once,
and cols / 32 blocks and a few partial sums are added: (cols / 32 + 12) u S. More
vectors enter the matrix cores as two f16 numbers that leave 2^-23 of a value at
most (2 u), and each of a block's 64 products and its sums is rounded at most by a
unit, 2 u: (cols / 32 + 200) u S.
"""
import numpy as np
import pytest

import mmhip as mm
import step_ends_reference as ref
from step_reference import At, Buffers, Graph, U

pytestmark = pytest.mark.gpu

TYPES = [mm.Q4_0, mm.IQ4_NL]


def weights(rng, t, rows, cols, count=1):
    raw = mm.make_weight(rng, t, rows, cols, count)
    return raw, ref.values_4bit(raw, t).reshape(count, rows, cols)


def check(y, w, x, few=True):
    """y [..., rows] against w [rows, cols] times x [..., cols]."""
    x = x.astype(np.float64)
    want, s = x @ w.T, np.abs(x) @ np.abs(w).T
    tol = (w.shape[1] / 32 + (12 if few else 200)) * U * s + (2.0 ** -31 * 32 * np.abs(x).max() * np.abs(w).max() * w.shape[1] / 32)
    err = np.abs(y - want)
    assert (err <= tol).all(), (err / tol).max()


# ---- dequantisation -------------------------------------------------------

@pytest.mark.parametrize("t", TYPES)
def test_every_scale_and_code(ctx, t):
    """All 65536 scales, every code: the bits of f16 times an integer, NaN where the scale is one."""
    blk = np.zeros((65536, 18), np.uint8)
    blk[:, :2] = np.arange(65536, dtype=np.uint16).view(np.uint8).reshape(-1, 2)
    blk[:, 2:] = (np.arange(16) | (np.arange(16)[::-1] << 4)).astype(np.uint8)
    got = ctx.dequantize(blk.reshape(-1), t, 65536 * 32)
    with np.errstate(invalid="ignore"):
        want = ref.values_4bit(blk, t).astype(np.float32).ravel()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[~np.isnan(want)], want[~np.isnan(want)])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n", [1, 3, 16, 17, 31, 32, 33, 999])
def test_dequantised_lengths(ctx, t, n):
    rng = np.random.default_rng(n)
    raw = mm.make_weight(rng, t, 1, (n + 31) // 32 * 32)
    want = ref.values_4bit(raw, t).ravel()[:n].astype(np.float32)
    with Buffers(ctx) as d:
        out = d.put(np.full(n + 5, 7.0, np.float32))
        ctx.dequantize_dev(At(out, 4), d.put(raw), t, n)  # not 16-byte aligned
        ctx.synchronize()
        got = out.to_numpy(np.float32, n + 5)
    assert np.array_equal(got[1:n + 1], want) and (got[n + 1:] == 7).all() and got[0] == 7


# ---- one vector -----------------------------------------------------------

@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 32), (15, 96), (16, 128), (17, 160), (33, 512), (40, 544), (768, 2048), (100, 2112),
                                       (64, 8192), (48, 8224), (35, 20480), (5000, 64), (70000, 32), (4111, 768)])
def test_one_vector(ctx, t, rows, cols):
    rng = np.random.default_rng(rows * 7 + cols)
    raw, w = weights(rng, t, rows, cols)
    x = rng.standard_normal(cols).astype(np.float32)
    x[rng.integers(0, cols, cols // 32)] *= 1000
    wt = ctx.upload(raw, t, rows, cols)
    with Buffers(ctx) as d:
        dx, dy = d.put(np.concatenate([[0], x]).astype(np.float32)), d.put(np.full(rows + 9, 7.0, np.float32))
        ys = []
        for _ in range(2):
            ctx.gemv_batched_dev(wt, 0, 1, At(dx, 4), 0, At(dy, 4), 0)
            ctx.synchronize()
            ys.append(dy.to_numpy(np.float32, rows + 9))
    wt.free()
    assert np.array_equal(ys[0], ys[1]) and (ys[0][rows + 1:] == 7).all() and ys[0][0] == 7
    check(ys[0][1:rows + 1], w[0], x)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("shared", [False, True])
def test_several_matrices(ctx, t, shared):
    rng = np.random.default_rng(3)
    n, rows, cols = 9, 70, 1184
    raw, w = weights(rng, t, rows, cols, n)
    x = rng.standard_normal((n, cols + 3)).astype(np.float32)
    wt = ctx.upload(raw, t, rows, cols, n)
    with Buffers(ctx) as d:
        dy = d.put(np.full((n, rows + 2), 7.0, np.float32))
        ctx.gemv_batched_dev(wt, 2, 6, d.put(x), 0 if shared else cols + 3, dy, rows + 2)
        ctx.synchronize()
        y = dy.to_numpy(np.float32, n * (rows + 2)).reshape(n, rows + 2)
        with pytest.raises(mm.MmhipError):
            ctx.gemv_batched_dev(wt, 4, 6, d.put(x), 0, dy, rows + 2)
    wt.free()
    for i in range(6):
        check(y[i, :rows], w[2 + i], x[0 if shared else i, :cols])
    assert (y[6:] == 7).all() and (y[:, rows:] == 7).all()


@pytest.mark.parametrize("t", TYPES)
def test_groups_in_one_launch(ctx, t):
    """Groups of other shapes and strides in one launch."""
    rng = np.random.default_rng(4)
    shapes = [(3, 150, 512), (5, 64, 2080), (1, 16, 96)]
    with Buffers(ctx) as d:
        groups, all_w, xs, ys = [], [], [], []
        for n, rows, cols in shapes:
            raw, w = weights(rng, t, rows, cols, n)
            x = rng.standard_normal((n, cols)).astype(np.float32)
            all_w.append((ctx.upload(raw, t, rows, cols, n), w))
            xs.append(x)
            ys.append(d.new(n * rows * 4))
            groups.append((all_w[-1][0], 0, n, d.put(x), cols, ys[-1], rows))
        ctx.gemv_grouped_dev(groups)
        ctx.synchronize()
        for (n, rows, cols), (wt, w), x, y in zip(shapes, all_w, xs, ys):
            got = y.to_numpy(np.float32, n * rows).reshape(n, rows)
            for i in range(n):
                check(got[i], w[i], x[i])
        other = ctx.upload(mm.make_weight(rng, mm.Q8_0, 16, 64), mm.Q8_0, 16, 64)
        with pytest.raises(mm.MmhipError):
            ctx.gemv_grouped_dev([groups[0], (other, 0, 1, ys[0], 0, ys[1], 16)])  # two types
        other.free()
        for wt, _ in all_w:
            wt.free()


# ---- several vectors ------------------------------------------------------

@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("batch", [1, 2, 3, 4, 5, 7, 15, 16, 17, 32, 33, 77, 130])
@pytest.mark.parametrize("rows,cols", [(17, 96), (100, 544), (64, 2176)])
def test_several_vectors(ctx, t, layout, batch, rows, cols):
    rng = np.random.default_rng(batch * 31 + rows)
    raw, w = weights(rng, t, rows, cols)
    x = rng.standard_normal((batch, cols)).astype(np.float32)
    x[:, rng.integers(0, cols, cols // 32)] *= 300
    wt = ctx.upload(raw, t, rows, cols)
    with Buffers(ctx) as d:
        dx, dy = d.put(x), d.put(np.full(batch * rows + 9, 7.0, np.float32))
        ys = []
        for call in (ctx.qmm_dev, ctx.qmm_dev_noalloc):
            call(wt, 0, dx, dy, batch, layout)
            ctx.synchronize()
            ys.append(dy.to_numpy(np.float32, batch * rows + 9))
    wt.free()
    assert np.array_equal(ys[0], ys[1]) and (ys[0][batch * rows:] == 7).all()
    y = ys[0][:batch * rows]
    check(y.reshape(batch, rows) if layout == 0 else y.reshape(rows, batch).T, w[0], x, few=False)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("batch,rows,cols", [(256, 1000, 768), (300, 4100, 256), (64, 16400, 128), (4, 40000, 64), (1000, 130, 8224),
                                             (16, 70001, 96), (29, 40000, 160), (37, 30000, 288), (250, 10250, 544), (513, 5000, 96), (40, 16000, 544), (100, 6000, 96),
                                             (77, 7001, 2176), (64, 768, 4352), (64, 1000, 768),
                                             (100, 1000, 2176), (77, 4000, 2112)])
def test_large_products(ctx, t, batch, rows, cols):
    rng = np.random.default_rng(batch)
    raw, w = weights(rng, t, rows, cols, 2)
    x = rng.standard_normal((batch, cols)).astype(np.float32)
    wt = ctx.upload(raw, t, rows, cols, 2)
    with Buffers(ctx) as d:
        dy = d.new(batch * rows * 4)
        ctx.qmm_dev(wt, 1, d.put(x), dy, batch)
        ctx.synchronize()
        y = dy.to_numpy(np.float32, batch * rows).reshape(batch, rows)
    wt.free()
    check(y, w[1], x, few=False)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("batch,rows,cols", [(2, 50, 160), (20, 50, 160), (300, 4100, 160), (50, 30000, 96)])
def test_vectors_at_any_float(ctx, t, batch, rows, cols):
    """Inputs and outputs that stand four bytes behind what larger accesses like; nothing around the output is written."""
    rng = np.random.default_rng(batch)
    raw, w = weights(rng, t, rows, cols)
    x = rng.standard_normal((batch, cols)).astype(np.float32)
    wt = ctx.upload(raw, t, rows, cols)
    with Buffers(ctx) as d:
        dx, dy = d.put(np.concatenate([[np.float32(np.nan)], x.ravel()])), d.put(np.full(batch * rows + 9, 7.0, np.float32))
        ctx.qmm_dev(wt, 0, At(dx, 4), At(dy, 4), batch)
        ctx.synchronize()
        y = dy.to_numpy(np.float32, batch * rows + 9)
    wt.free()
    assert y[0] == 7 and (y[batch * rows + 1:] == 7).all()
    check(y[1:batch * rows + 1].reshape(batch, rows), w[0], x, few=False)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("layout", [0, 1])
def test_results_behind_four_gigabytes(ctx, t, layout):
    """The last ones of [70000 x 32] times 20000 vectors (5.6 GB)."""
    rng = np.random.default_rng(5)
    batch, rows, cols = 20000, 70000, 32
    raw, w = weights(rng, t, rows, cols)
    x = rng.standard_normal((batch, cols)).astype(np.float32)
    wt = ctx.upload(raw, t, rows, cols)
    with Buffers(ctx) as d:
        y = mm.DeviceArray(ctx, batch * rows * 4)
        d.held.append(y)
        ctx.qmm_dev(wt, 0, d.put(x), y, batch, layout)
        ctx.synchronize()
        line = rows if layout == 0 else batch
        take = d.new(4 * line)
        # the last line, as a row of a table of lines
        lines = batch if layout == 0 else rows
        ctx.embed_dev(take, y, mm.F32, lines, line, d.put(np.array([lines - 1], np.uint32)), 1)
        ctx.synchronize()
        last = take.to_numpy(np.float32, line)
    wt.free()
    if layout == 0:
        check(last[None], w[0], x[-1:], few=False)
    else:
        check(last[:, None], w[0][-1:], x, few=False)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("batch,rows,cols", [(6, 40, 640), (64, 500, 640), (70, 3000, 640), (70, 9000, 640), (40, 30000, 640), (64, 768, 4352), (77, 4000, 2112)])
@pytest.mark.parametrize("where", [100, 321, 600])
def test_values_that_outgrow_the_first(ctx, t, batch, rows, cols, where):
    """Values up to 1e6 and 1e30 times as large as a vector's first 64, which set its power of two; first ones of 0."""
    rng = np.random.default_rng(where)
    raw, w = weights(rng, t, rows, cols)
    x = rng.standard_normal((batch, cols)).astype(np.float32)
    x[0, where] = 1e6
    x[1, where] = -1e30
    x[2, :where] = 0
    x[3, :where] *= np.float32(1e-30)
    x[4, where:where + 32] *= 4000
    wt = ctx.upload(raw, t, rows, cols)
    with Buffers(ctx) as d:
        dy = d.new(batch * rows * 4)
        ctx.qmm_dev(wt, 0, d.put(x), dy, batch)
        ctx.synchronize()
        y = dy.to_numpy(np.float32, batch * rows).reshape(batch, rows)
    wt.free()
    x = x.astype(np.float64)
    want, s = x @ w[0].T, np.abs(x) @ np.abs(w[0]).T
    # a value below 2^-39 of the vector's largest may be off by that much
    tol = (cols / 32 + 200) * U * s + 2.0 ** -38 * np.abs(x).max(1, keepdims=True) * np.abs(w[0]).sum(1)
    assert (np.abs(y - want) <= tol).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("batch", [1, 3, 40])
def test_seam(ctx, t, batch):
    """The host entry points."""
    rng = np.random.default_rng(batch)
    raw, w = weights(rng, t, 333, 640)
    x = rng.standard_normal((batch, 640)).astype(np.float32)
    check(ctx.batch_mat_mul(raw, t, x, 333, batch, 640), w[0], x, few=False)
    check(ctx.mat_vec_mul(raw, t, x[0], 333, 640), w[0], x[0])


# ---- values where it can go wrong -----------------------------------------

@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("batch", [1, 4, 20])
@pytest.mark.parametrize("size", [1e-38, 1e-30, 1.0, 1e30])
def test_sizes_of_values(ctx, t, batch, size):
    """Tiny and large vectors, a block of zeros, blocks of very different size beside each other."""
    rng = np.random.default_rng(5)
    rows, cols = 40, 704
    raw, w = weights(rng, t, rows, cols)
    x = (rng.standard_normal((batch, cols)) * size).astype(np.float32)
    x[:, 32:64] = 0
    x[:, 64:96] *= np.float32(1e-3)
    wt = ctx.upload(raw, t, rows, cols)
    with Buffers(ctx) as d:
        dy = d.new(batch * rows * 4)
        ctx.qmm_dev(wt, 0, d.put(x), dy, batch)
        ctx.synchronize()
        y = dy.to_numpy(np.float32, batch * rows).reshape(batch, rows)
    wt.free()
    x64 = x.astype(np.float64)
    want, s = x64 @ w[0].T, np.abs(x64) @ np.abs(w[0]).T
    # below f32's normal numbers (2^-126) sums and parts may be flushed: a unit of that size each
    tol = (cols / 32 + 200) * U * s + cols * np.abs(w).max() * 2.0 ** -122
    assert (np.abs(y - want) <= tol).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("batch", [1, 2, 4, 20])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_one_vector_that_is_not_finite(ctx, t, batch, bad):
    """It poisons its own results, not the other vectors'."""
    rng = np.random.default_rng(6)
    rows, cols = 70, 256
    raw, w = weights(rng, t, rows, cols)
    x = rng.standard_normal((batch, cols)).astype(np.float32)
    x[batch // 2, 77] = bad
    wt = ctx.upload(raw, t, rows, cols)
    with Buffers(ctx) as d:
        dy = d.new(batch * rows * 4)
        ctx.qmm_dev(wt, 0, d.put(x), dy, batch)
        ctx.synchronize()
        y = dy.to_numpy(np.float32, batch * rows).reshape(batch, rows)
    wt.free()
    assert not np.isfinite(y[batch // 2]).any()
    rest = np.arange(batch) != batch // 2
    if rest.any():
        check(y[rest], w[0], x[rest], few=False)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("batch", [1, 4, 20])
def test_scales_that_are_large_tiny_or_not_finite(ctx, t, batch):
    rng = np.random.default_rng(7)
    rows, cols = 36, 256
    raw = mm.make_weight(rng, t, rows, cols).reshape(rows, cols // 32, 18)
    for r, d in ((3, 65504.0), (5, 6e-8), (7, 0.0), (9, np.nan), (11, np.inf)):
        raw[r, 4, :2] = np.array([d], np.float16).view(np.uint8)
    w = ref.values_4bit(raw, t).reshape(rows, cols)
    x = rng.standard_normal((batch, cols)).astype(np.float32)
    wt = ctx.upload(raw.reshape(-1), t, rows, cols)
    with Buffers(ctx) as d:
        dy = d.new(batch * rows * 4)
        ctx.qmm_dev(wt, 0, d.put(x), dy, batch)
        ctx.synchronize()
        y = dy.to_numpy(np.float32, batch * rows).reshape(batch, rows)
    wt.free()
    assert not np.isfinite(y[:, [9, 11]]).any()
    fine = np.isfinite(w).all(1)
    x64 = x.astype(np.float64)
    want, s = x64 @ w[fine].T, np.abs(x64) @ np.abs(w[fine]).T
    assert (np.abs(y[:, fine] - want) <= (cols / 32 + 200) * U * s).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("batch", [1, 4, 24])
def test_all_bits_of_a_vector_count(ctx, t, batch):
    """Products that cancel down to the vectors' last bits: weights of one size, x and -x (1 - 2^-23) side by side. Every
    block's sum is a few last bits, so nothing is rounded and the result is exact to 2^-20 of itself."""
    rng = np.random.default_rng(8)
    rows, cols = 32, 128
    blk = np.zeros((rows, cols // 32, 18), np.uint8)
    blk[..., :2] = np.array([1.0], np.float16).view(np.uint8)
    blk[..., 2:] = 0x99 if t == mm.Q4_0 else 0x88  # weight 1 in both
    x = np.empty((batch, cols), np.float32)
    x[:, ::2] = rng.integers(1 << 22, 1 << 23, (batch, cols // 2)) * np.float32(2.0 ** -22)
    x[:, 1::2] = -(x[:, ::2] - np.float32(2.0 ** -22))
    want = x.astype(np.float64).sum(1)
    wt = ctx.upload(blk.reshape(-1), t, rows, cols)
    with Buffers(ctx) as d:
        dy = d.new(batch * rows * 4)
        ctx.qmm_dev(wt, 0, d.put(x), dy, batch)
        ctx.synchronize()
        y = dy.to_numpy(np.float32, batch * rows).reshape(batch, rows)
    wt.free()
    # the bf16 parts' products are summed by size, up to 32 x 2 in a block: 2^-23 x 64 per block where they cancel
    tol = 2.0 ** -20 * want[:, None] if batch <= 4 else cols / 32 * 64 * 2.0 ** -23
    assert (np.abs(y - want[:, None]) <= tol).all()


# ---- graphs, files, refusals ----------------------------------------------

@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("batch", [1, 4, 40])
def test_captured_and_replayed(ctx, t, batch):
    rng = np.random.default_rng(9)
    rows, cols = 500, 1056
    raw, w = weights(rng, t, rows, cols)
    wt = ctx.upload(raw, t, rows, cols)
    with Buffers(ctx) as d:
        dx, dy, de = d.new(batch * cols * 4), d.new(batch * rows * 4), d.new(batch * rows * 4)
        call = (lambda y: ctx.qmm_dev(wt, 0, dx, y, batch)) if batch > 1 else (lambda y: ctx.gemv_batched_dev(wt, 0, 1, dx, 0, y, 0))
        call(dy)  # the kernels are loaded outside the capture
        ctx.synchronize()
        g = Graph(ctx, lambda: call(dy))
        try:
            for _ in range(3):
                x = rng.standard_normal((batch, cols)).astype(np.float32)
                mm.check(ctx.lib.mmhip_memcpy_h2d(ctx.handle, dx.ptr, x.ctypes.data, x.nbytes), "h2d")
                g.replay()
                call(de)
                ctx.synchronize()
                a, b = dy.to_numpy(np.float32, batch * rows), de.to_numpy(np.float32, batch * rows)
                assert np.array_equal(a, b)
                check(a.reshape(batch, rows), w[0], x, few=False)
        finally:
            g.free()
            wt.free()


def test_from_a_file(ctx, tmp_path):
    import gguf_writer as gw
    rng = np.random.default_rng(10)
    a, wa = weights(rng, mm.Q4_0, 48, 96)
    b, wb = weights(rng, mm.Q4_0, 20, 96)
    c, wc = weights(rng, mm.IQ4_NL, 30, 64)
    path = tmp_path / "f.gguf"
    gw.write(path, [], [("a.weight", [96, 48], mm.Q4_0, a), ("b.weight", [96, 20], mm.Q4_0, b), ("c.weight", [64, 30], mm.IQ4_NL, c)])
    x = rng.standard_normal(96).astype(np.float32)
    with mm.Gguf(path) as g, Buffers(ctx) as d:
        ab, wt = ctx.upload_gguf_rows(g, ["a.weight", "b.weight"]), ctx.upload_gguf(g, "c.weight")
        dx, dy = d.put(x), d.new(68 * 4)
        ctx.gemv_batched_dev(ab, 0, 1, dx, 0, dy, 0)
        ctx.synchronize()
        check(dy.to_numpy(np.float32, 68), np.concatenate([wa[0], wb[0]]), x)
        ctx.gemv_batched_dev(wt, 0, 1, dx, 0, dy, 0)
        ctx.synchronize()
        check(dy.to_numpy(np.float32, 30), wc[0], x[:64])
        ab.free()
        wt.free()


@pytest.mark.parametrize("t", TYPES)
def test_refusals(ctx, t):
    raw = np.zeros(18 * 64, np.uint8)
    for rows, cols, code in ((4, 33, mm.ERR_INVALID), (4, 16, mm.ERR_INVALID), (0, 32, mm.ERR_INVALID), (1, 1 << 23, mm.ERR_UNSUPPORTED)):
        with pytest.raises(mm.MmhipError) as e:
            ctx.upload(raw, t, rows, cols)
        assert e.value.code == code
    h = np.zeros((2, 64, 64), np.float32)
    with pytest.raises(mm.MmhipError) as e:
        mm.MoeLayer(ctx, hidden=64, inter=64, n_experts=2, expert_type=t, router=np.zeros((2, 64), np.float32),
                    gate=h.view(np.uint8), up=h.view(np.uint8), down=h.view(np.uint8))
    assert e.value.code == mm.ERR_UNSUPPORTED
