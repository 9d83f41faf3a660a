"""The operators between a decode step's products on the device, against plain
64-bit forms (tests/step_reference.py).

Tolerances, u = 2^-24 (half a step of f32): the norm's value is three f32
roundings (the root, two products), 3 u; a rotated value the rounding of two
cosines, two products and a sum, at most 4 u (|a| + |b|) times the magnitude,
plus the angle's error of 1e-9 up to 2^20 positions and 2e-6 beyond; f16 results
half a step (2^-11) more. Attention: queries and probabilities of 22 bits and
sums in f32 put random errors of about 2^-22 times a few on each probability;
against values of random sign they reach the output's 2-norm at that size, and
1e-5 leaves a factor of ten; lse, 1e-5. Log probabilities: a sum of exponentials
in f32 in chunks of at most 64 terms joined in a tree is good to about 100 u in
the worst order, 6e-6, and the entropy to that times the terms' size.
"""
import math

import numpy as np
import pytest

import mmhip as mm
import step_reference as ref
from step_reference import At, Buffers, Graph, Pool, U

pytestmark = pytest.mark.gpu

F16_HALF_STEP = 2.0 ** -11


def f32(b, n):
    return b.to_numpy(np.float32, n)


def same_bits(a, b):
    a, b = np.ascontiguousarray(a), np.ascontiguousarray(b)
    assert a.dtype == b.dtype and a.shape == b.shape
    view = {4: np.uint32, 2: np.uint16, 1: np.uint8}[a.dtype.itemsize]
    assert np.array_equal(a.view(view), b.view(view))


# ---- root-mean-square norm ------------------------------------------------

def run_norm(ctx, x, w, eps, res=None, y_type=mm.F32, want_sum=False, in_place=False, pad=0, off=0):
    """(y, sum): strided by `pad` extra columns and shifted by `off` floats; the padding has to stay as it was."""
    n, cols = x.shape
    ld = cols + pad
    with Buffers(ctx) as d:
        def rows(a):
            buf = np.full((n, ld), np.nan, np.float32)
            buf[:, :cols] = a
            return At(d.put(np.concatenate([np.zeros(off, np.float32), buf.ravel()])), 4 * off)
        dx, dw = rows(x), At(d.put(np.concatenate([np.zeros(off, np.float32), w])), 4 * off)
        dr = rows(res) if res is not None else None
        size = {mm.F32: 4, mm.F16: 2}.get(y_type)
        dy = d.new(n * ld * size if size else n * ((cols + 31) // 32) * 34)
        ds = dr if in_place else d.new(n * ld * 4) if want_sum else None
        ctx.rms_norm_dev(dy, dx, dw, n, cols, eps=eps, y_type=y_type, y_stride=ld, x_stride=ld, residual=dr,
                         residual_stride=ld, sum_out=ds, sum_stride=ld)
        ctx.synchronize()
        if size:
            raw = dy.to_numpy(np.float32 if size == 4 else np.float16, n * ld).reshape(n, ld)
            assert np.isnan(raw[:, cols:]).all()
            y = raw[:, :cols].copy()
        else:
            y = dy.to_numpy(np.uint8, n * ((cols + 31) // 32) * 34).reshape(n, -1, 34)
        s = None
        if ds is not None:
            base = ds.buf if isinstance(ds, At) else ds
            s = f32(base, (off if isinstance(ds, At) else 0) + n * ld)[-n * ld:].reshape(n, ld)[:, :cols].copy()
        return y, s


@pytest.mark.parametrize("n,cols", [(1, 2048), (3, 768), (5, 512), (2, 33), (4, 1), (1, 31), (2, 1025), (7, 2050),
                                    (1, 4099), (2, 10000), (300, 96)])
@pytest.mark.parametrize("residual", [False, True])
def test_norm(ctx, n, cols, residual):
    rng = np.random.default_rng(n * 10007 + cols)
    x, w = rng.standard_normal((n, cols)).astype(np.float32), rng.standard_normal(cols).astype(np.float32)
    res = (4 * rng.standard_normal((n, cols))).astype(np.float32) if residual else None
    s = x + res if residual else x
    want = ref.rms_norm64(s, w, np.float64(np.float32(1e-5)))
    y, got_s = run_norm(ctx, x, w, 1e-5, res, want_sum=residual)
    assert (np.abs(y - want) <= 3.1 * U * np.abs(want)).all()
    if residual:
        same_bits(got_s, s)
    # other buffers, strides and alignments: the same bits
    for kw in (dict(pad=3), dict(off=1), dict(pad=4, off=2), dict(in_place=residual, pad=1)):
        y2, s2 = run_norm(ctx, x, w, 1e-5, res, want_sum=residual, **kw)
        same_bits(y2, y)
        if residual:
            same_bits(s2, s)
    h, _ = run_norm(ctx, x, w, 1e-5, res, y_type=mm.F16, pad=1)
    same_bits(h, y.astype(np.float16))
    q, _ = run_norm(ctx, x, w, 1e-5, res, y_type=mm.Q8_0)
    for r in range(n):
        assert np.array_equal(q[r].reshape(-1), ctx.quantize_q8_0(y[r])), r


@pytest.mark.parametrize("n,cols", [(3, 1024), (2, 1028), (3, 4096), (2, 4095), (2, 4100), (1, 20000)])
def test_norm_widths(ctx, n, cols):
    """Either side of the widths at which a row is held differently."""
    test_norm(ctx, n, cols, True)


def test_norm_in_place(ctx):
    """y on x, y on the residual, the sum on x: each gives what separate buffers give."""
    rng = np.random.default_rng(3)
    for n, cols in ((3, 2048), (2, 9001)):
        x, r = (rng.standard_normal((n, cols)).astype(np.float32) for _ in range(2))
        w = rng.standard_normal(cols).astype(np.float32)
        y, s = run_norm(ctx, x, w, 1e-6, r, want_sum=True)
        with Buffers(ctx) as d:
            dw = d.put(w)
            a, b, c = d.put(x), d.put(r), d.new(n * cols * 4)
            ctx.rms_norm_dev(a, a, dw, n, cols, eps=1e-6, residual=b)
            same_bits(f32(a, n * cols).reshape(n, cols), y)
            a = d.put(x)
            ctx.rms_norm_dev(b, a, dw, n, cols, eps=1e-6, residual=b, sum_out=a)
            same_bits(f32(b, n * cols).reshape(n, cols), y)
            same_bits(f32(a, n * cols).reshape(n, cols), s)
            a, b = d.put(x), d.put(r)
            ctx.rms_norm_dev(c, a, dw, n, cols, eps=1e-6, residual=b, sum_out=a)
            same_bits(f32(c, n * cols).reshape(n, cols), y)
            same_bits(f32(a, n * cols).reshape(n, cols), s)
            a = d.put(x)
            ctx.rms_norm_dev(a, a, dw, n, cols, eps=1e-6)
            same_bits(f32(a, n * cols).reshape(n, cols), run_norm(ctx, x, w, 1e-6)[0])


def test_norm_values(ctx):
    """Zeros, huge and tiny rows (their squares leave f32's range), infinities and NaN."""
    cols = 300
    x = np.zeros((6, cols), np.float32)
    x[1], x[2] = 1e30, 1e-30
    x[3, 7], x[4, 9] = np.inf, np.nan
    x[5] = np.linspace(-3e38, 3e38, cols)
    w = np.full(cols, 1.5, np.float32)
    y, _ = run_norm(ctx, x, w, 1e-5)
    assert (y[0] == 0).all()
    want = ref.rms_norm64(x, w, np.float64(np.float32(1e-5)))
    for r in (1, 2, 5):
        assert (np.abs(y[r] - want[r]) <= 3.1 * U * np.abs(want[r]) + 1e-45).all(), r
    assert np.isnan(y[3, 7]) and (np.delete(y[3], 7) == 0).all()
    assert np.isnan(y[4]).all()
    y0, _ = run_norm(ctx, x[:1], w, 0.0)
    assert np.isnan(y0).all()


# ---- rotary positions -----------------------------------------------------

ROPES = [dict(dims=64, base=1e6), dict(dims=64, base=1e4, scaling="linear", factor=4.0),
         dict(dims=64, base=1e6, scaling="yarn", factor=16.0, original_context=8192), dict(dims=2, base=1e4),
         dict(dims=256, base=5e5), dict(dims=6, base=100.0, magnitude=0.25)]


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("kw", ROPES)
@pytest.mark.parametrize("tokens,heads,head_dim,first", [(1, 20, 192, 128), (5, 3, 64, 0), (33, 1, 300, 17)])
def test_rope(ctx, layout, kw, tokens, heads, head_dim, first):
    dims = kw["dims"]
    head_dim = max(head_dim, first + dims)
    rng = np.random.default_rng(dims + tokens)
    x = rng.standard_normal((tokens, heads, head_dim)).astype(np.float32)
    pos = rng.integers(0, 1 << 20, tokens).astype(np.uint32)
    pos[0] = 0 if tokens > 1 else 131071
    freqs = ref.frequencies64(**dict(kw, base=float(np.float32(kw["base"]))))
    rope = mm.Rope(ctx, layout=layout, **kw)
    mag = mm.rope_frequencies(rope.params)[1]
    part = slice(first, first + dims)
    want = ref.rope64(x[..., part], pos, layout, freqs, mag)
    n = dims // 2
    a = np.abs(x[..., part].astype(np.float64))
    pair = a[..., 0::2] + a[..., 1::2] if layout == "interleaved" else a[..., :n] + a[..., n:]
    room = np.repeat(pair, 2, -1) if layout == "interleaved" else np.concatenate([pair, pair], -1)
    hs, ts = head_dim + 2, heads * (head_dim + 2) + 5
    with Buffers(ctx) as d:
        try:
            dx, dp, dy = d.put(x), d.put(pos), d.new(tokens * ts * 4)
            ctx.rope_dev(rope, dy, dx, dp, tokens, heads, head_dim, first, y_strides=(ts, hs))
            ctx.synchronize()
            raw = f32(dy, tokens * ts).reshape(tokens, ts)
            heads_out = raw[:, :heads * hs].reshape(tokens, heads, hs)
            assert np.isnan(raw[:, heads * hs:]).all() and np.isnan(heads_out[..., head_dim:]).all()
            y = heads_out[..., :head_dim]
            assert (np.abs(y[..., part] - want) <= (4 * U + 1e-9) * mag * room).all()
            same_bits(np.delete(y, np.r_[part], -1), np.delete(x, np.r_[part], -1))
            ctx.rope_dev(rope, dx, dx, dp, tokens, heads, head_dim, first)  # in place: the same bits
            ctx.synchronize()
            same_bits(f32(dx, x.size).reshape(x.shape), y.copy())
        finally:
            rope.free()


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dims,heads,head_dim,first", [(64, 20, 192, 128), (64, 130, 72, 4), (8, 700, 8, 0), (256, 9, 260, 4),
                                                       (128, 3, 1024, 512)])
def test_rope_aligned(ctx, layout, dims, heads, head_dim, first):
    """Buffers of 16-byte aligned rows and heads, copied and in place, with more pairs than a workgroup has threads: the
    bits of buffers that are one float off."""
    rng = np.random.default_rng(heads)
    tokens = 3
    x = rng.standard_normal((tokens, heads, head_dim)).astype(np.float32)
    pos = np.array([0, 77, 131071], np.uint32)
    rope = mm.Rope(ctx, dims=dims, base=1e5, layout=layout)
    with Buffers(ctx) as d:
        try:
            dp, dx, dy = d.put(pos), d.put(x), d.new(x.size * 4)
            ctx.rope_dev(rope, dy, dx, dp, tokens, heads, head_dim, first)
            ctx.synchronize()
            y = f32(dy, x.size).reshape(x.shape)
            same_bits(np.delete(y, np.r_[first:first + dims], -1), np.delete(x, np.r_[first:first + dims], -1))
            part = slice(first, first + dims)
            want = ref.rope64(x[..., part], pos, layout, ref.frequencies64(dims, 1e5))
            assert (np.abs(y[..., part] - want) <= (4 * U + 1e-9) * 2 * np.abs(x).max()).all()
            odd, off = d.put(np.concatenate([np.zeros(1, np.float32), x.ravel()])), d.new(x.size * 4 + 4)
            ctx.rope_dev(rope, At(off, 4), At(odd, 4), dp, tokens, heads, head_dim, first)
            ctx.rope_dev(rope, dx, dx, dp, tokens, heads, head_dim, first)
            ctx.synchronize()
            same_bits(f32(off, x.size + 1)[1:].reshape(x.shape).copy(), y)
            same_bits(f32(dx, x.size).reshape(x.shape), y)
            with pytest.raises(mm.MmhipError, match="heads"):
                ctx.rope_dev(rope, dy, dx, dp, 1, 1 << 24, head_dim, first)
        finally:
            rope.free()


def test_rope_far_positions(ctx):
    rng = np.random.default_rng(9)
    pos = np.array([0, 2 ** 20 - 1, 2 ** 24 + 1, 2 ** 31 - 1, 2 ** 32 - 1], np.uint32)
    x = rng.standard_normal((5, 2, 64)).astype(np.float32)
    rope = mm.Rope(ctx, dims=64, base=1e4, layout="half")
    # the angle modulo a turn, in integers: frequencies as multiples of 2^-80 of a turn
    turns = [int(round(f / (2 * math.pi) * 2.0 ** 50)) << 30 for f in ref.frequencies64(64, 1e4)]
    with Buffers(ctx) as d:
        try:
            dx = d.put(x)
            ctx.rope_dev(rope, dx, dx, d.put(pos), 5, 2, 64)
            ctx.synchronize()
            y = f32(dx, x.size).reshape(x.shape)
        finally:
            rope.free()
    for t, p in enumerate(pos):
        ang = np.array([(int(p) * k) % (1 << 80) / 2.0 ** 80 * 2 * math.pi for k in turns])
        c, s = np.cos(ang), np.sin(ang)
        a, b = x[t, :, :32].astype(np.float64), x[t, :, 32:].astype(np.float64)
        # 2^-51 of a turn on the rounded frequencies above, times the position
        tol = (4 * U + 2e-6 + float(p) * 2 * math.pi * 2.0 ** -51 * 2) * (np.abs(a) + np.abs(b))
        assert (np.abs(y[t, :, :32] - (a * c - b * s)) <= tol).all(), p
        assert (np.abs(y[t, :, 32:] - (a * s + b * c)) <= tol).all(), p


# ---- the paged cache's writer ---------------------------------------------

@pytest.mark.parametrize("ggml_type", [mm.F16, mm.Q8_0])
@pytest.mark.parametrize("rank,pe,pt,layout", [(512, 64, 16, "interleaved"), (512, 64, 64, "half"), (32, 0, 16, "half"),
                                               (96, 32, 128, "interleaved"), (480, 64, 16, "half")])
def test_store(ctx, ggml_type, rank, pe, pt, layout):
    """Each stored row is the norm's, the rope's and the codec's result for it; every other byte stays."""
    rng = np.random.default_rng(rank + pe + pt)
    width, n_pages, n, pad = rank + pe, 7, 23, 5
    pool = Pool(rng, ggml_type, rank, pe, pt, n_pages)
    kv = (2 * rng.standard_normal((n, width + pad))).astype(np.float32)
    kv[3] = 0.0
    w = rng.standard_normal(rank).astype(np.float32)
    slots = rng.permutation(n_pages * pt)[:n].astype(np.int32)
    slots[5], slots[11] = -1, -7
    slots[0] = n_pages * pt - 1 if n_pages * pt - 1 not in slots else slots[0]
    pos = rng.integers(0, 200000, n).astype(np.uint32)
    rope = mm.Rope(ctx, dims=pe, base=1e6, layout=layout) if pe else None
    try:
        for norm, turn in ((True, True), (False, True), (True, False), (False, False)):
            turn = turn and pe > 0
            rows = kv[:, :width].copy()
            if norm:
                rows[:, :rank] = run_norm(ctx, np.ascontiguousarray(kv[:, :rank]), w, 1e-5)[0]
            with Buffers(ctx) as d:
                dp = d.put(pos)
                if turn:
                    dr = d.put(rows[:, rank:])
                    ctx.rope_dev(rope, dr, dr, dp, n, 1, pe)
                    ctx.synchronize()
                    rows[:, rank:] = f32(dr, n * pe).reshape(n, pe)
                dpool = d.put(pool.bytes)
                cache = mm.KvCache(dpool, ggml_type, rank=rank, rope_dims=pe, page_tokens=pt, n_pages=n_pages)
                ctx.kv_store_dev(cache, d.put(kv), d.put(slots), n, kv_stride=width + pad,
                                 norm_weight=d.put(w) if norm else None, rope=rope if turn else None, positions=dp)
                ctx.synchronize()
                got = dpool.to_numpy(np.uint8, pool.bytes.size).reshape(pool.bytes.shape)
            want = pool.bytes.copy()
            for t, s in enumerate(slots):
                if s < 0:
                    continue
                page, at = s // pt, s % pt
                if ggml_type == mm.F16:
                    want[page].view(np.float16).reshape(pt, width)[at] = rows[t].astype(np.float16)
                else:
                    blocks = ctx.quantize_q8_0(rows[t]).reshape(-1, 34)
                    want[page, at * width:(at + 1) * width] = blocks[:, 2:].reshape(-1)
                    scales = want[page, pt * width:].reshape(pt, width // 32, 2)
                    scales[at] = blocks[:, :2]
            assert np.array_equal(got, want), (norm, turn)
    finally:
        if rope:
            rope.free()


def test_store_bad_slots(ctx):
    """Slots that the pool does not have are left out and reported once; the others are stored."""
    rng = np.random.default_rng(2)
    pool = Pool(rng, mm.F16, 64, 32, 16, 3)
    kv = rng.standard_normal((4, 96)).astype(np.float32)
    with Buffers(ctx) as d:
        guard = d.put(np.concatenate([pool.bytes.ravel(), np.full(4096, 0xAB, np.uint8)]))
        cache = mm.KvCache(guard, mm.F16, rank=64, rope_dims=32, page_tokens=16, n_pages=3)
        ctx.kv_store_dev(cache, d.put(kv), d.put(np.array([5, 48, 2 ** 31 - 1, 47], np.int32)), 4)
        with pytest.raises(mm.MmhipError, match="slot") as e:
            ctx.synchronize()
        assert e.value.code == mm.ERR_INVALID
        ctx.synchronize()
        got = guard.to_numpy(np.uint8, guard.nbytes)
        want = pool.bytes.copy()
        want[0].view(np.float16).reshape(16, 96)[5] = kv[0].astype(np.float16)
        want[2].view(np.float16).reshape(16, 96)[15] = kv[3].astype(np.float16)
        assert np.array_equal(got[:want.size], want.ravel()) and (got[want.size:] == 0xAB).all()


# ---- attention over the paged cache ---------------------------------------

def run_attention(ctx, pool, q, q_pe, tables, lens, scale, table_of=None, pad=0, lse=True, expect=None, n_tables=None):
    """(out, lse) through strided queries and outputs whose padding has to stay as it was."""
    n, h, rank = q.shape
    pe = pool.rope
    with Buffers(ctx) as d:
        def rows(a, width):
            buf = np.full((n, h, width + pad), np.nan, np.float32)
            buf[..., :width] = a
            return d.put(buf)
        cache = mm.KvCache(d.put(pool.bytes), pool.type, rank=rank, rope_dims=pe, page_tokens=pool.page_tokens,
                           n_pages=pool.n_pages)
        do, dl = d.new(n * h * (rank + pad) * 4), d.new(n * h * 4) if lse else None
        need = ctx.mla_attention_workspace(n, h, rank)
        work = d.new(need)
        args = ctx.mla_attention_args(
            cache, q=rows(q, rank), q_pe=rows(q_pe, pe) if pe else None, out=do, lse=dl, lens=d.put(lens.astype(np.uint32)),
            tables=d.put(tables.astype(np.int32)), n_tables=n_tables or len(tables), table_pages=tables.shape[1],
            table_of=None if table_of is None else d.put(table_of.astype(np.uint32)), n_tokens=n, n_heads=h, scale=scale,
            workspace=work, q_strides=(h * (rank + pad), rank + pad), q_pe_strides=(h * (pe + pad), pe + pad),
            out_strides=(h * (rank + pad), rank + pad))
        ctx.mla_attention_dev(args)
        if expect:
            with pytest.raises(mm.MmhipError, match=expect):
                ctx.synchronize()
        ctx.synchronize()
        out = f32(do, n * h * (rank + pad)).reshape(n, h, rank + pad)
        assert np.isnan(out[..., rank:]).all()
        first = out[..., :rank].copy()
        got = f32(dl, n * h).reshape(n, h) if lse else None
        ctx.mla_attention_dev(args)  # again, on the workspace as it was left: the same bits
        if expect:
            with pytest.raises(mm.MmhipError, match=expect):
                ctx.synchronize()
        ctx.synchronize()
        again = f32(do, n * h * (rank + pad)).reshape(n, h, rank + pad)[..., :rank].copy()
        same_bits(again, first)
        return first, got


def check_attention(out, lse, want, want_lse):
    assert np.isfinite(out).all()
    live = np.isfinite(want_lse)
    assert (out[~live] == 0).all() and (lse[~live] == -np.inf).all()
    err = np.linalg.norm(out - want, axis=-1)
    size = np.linalg.norm(want, axis=-1)
    assert (err <= 1e-5 * size).all(), float((err[live] / size[live]).max())
    assert (np.abs(lse[live] - want_lse[live]) <= 1e-5 * np.maximum(1, np.abs(want_lse[live]))).all()


def tables_for(rng, lens, pt, n_pages, more=2):
    """A table per token: its own pages in no order, entries behind them that name no page."""
    p = max(1, max((int(n) + pt - 1) // pt for n in lens)) + more
    t = np.full((len(lens), p), -1, np.int32)
    ids, at = rng.permutation(n_pages), 0
    for i, n in enumerate(lens):
        k = (int(n) + pt - 1) // pt
        t[i, :k] = ids[at:at + k]
        at += k
    assert at <= n_pages
    return t


def queries(rng, n, h, rank, pe, sigma=1.0):
    q = (rng.standard_normal((n, h, rank)) * sigma).astype(np.float32)
    return q, ((rng.standard_normal((n, h, pe)) * sigma).astype(np.float32) if pe else None)


LENS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 500, 1025]


@pytest.mark.parametrize("ggml_type", [mm.F16, mm.Q8_0])
@pytest.mark.parametrize("heads", [1, 5, 16, 17, 20, 32, 33, 40])
def test_attention_lengths_and_heads(ctx, ggml_type, heads):
    """Tokens of all lengths in one call; the rest of each last page holds NaN."""
    rng = np.random.default_rng(heads)
    lens = np.array(LENS if heads in (1, 20) else LENS[::3])
    pt, n_pages = 16, int(((lens + 15) // 16).sum()) + 3
    pool = Pool(rng, ggml_type, 512, 64, pt, n_pages)
    tables = tables_for(rng, lens, pt, n_pages)
    for i, n in enumerate(lens):
        for at in range(n % pt, pt if n % pt else 0):
            pool.spoil(tables[i, n // pt], at)
    q, q_pe = queries(rng, len(lens), heads, 512, 64)
    want = ref.attention64(q, q_pe, pool.values, tables, np.arange(len(lens)), lens, pt, 192 ** -0.5, 512)
    check_attention(*run_attention(ctx, pool, q, q_pe, tables, lens, 192 ** -0.5), *want)


@pytest.mark.parametrize("ggml_type", [mm.F16, mm.Q8_0])
@pytest.mark.parametrize("rank,pe,pt", [(512, 0, 16), (32, 64, 16), (64, 32, 32), (480, 64, 16), (96, 0, 1024),
                                        (256, 32, 64), (288, 64, 128)])
def test_attention_sizes(ctx, ggml_type, rank, pe, pt):
    rng = np.random.default_rng(rank + pe)
    lens = np.array([77, 0, 300, 1, 160])
    n_pages = int(((lens + pt - 1) // pt).sum()) + 1
    pool = Pool(rng, ggml_type, rank, pe, pt, n_pages)
    tables = tables_for(rng, lens, pt, n_pages, more=0)
    q, q_pe = queries(rng, 5, 7, rank, pe)
    scale = (rank + pe) ** -0.5 * 1.5
    want = ref.attention64(q, q_pe, pool.values, tables, np.arange(5), lens, pt, scale, rank)
    check_attention(*run_attention(ctx, pool, q, q_pe, tables, lens, scale, pad=3), *want)


@pytest.mark.parametrize("ggml_type", [mm.F16, mm.Q8_0])
@pytest.mark.parametrize("tokens,length", [(1, 20001), (3, 6000), (40, 700)])
def test_attention_shared_table(ctx, ggml_type, tokens, length):
    """A chunk of one context (one table, lengths one apart), and one long context split over the chip."""
    rng = np.random.default_rng(tokens)
    pt = 16
    n_pages = (length + pt - 1) // pt + 2
    pool = Pool(rng, ggml_type, 512, 64, pt, n_pages)
    tables = tables_for(rng, [length], pt, n_pages)
    lens = np.arange(length - tokens + 1, length + 1)
    q, q_pe = queries(rng, tokens, 20, 512, 64)
    rows = np.zeros(tokens, np.int64)
    want = ref.attention64(q, q_pe, pool.values, tables, rows, lens, pt, 192 ** -0.5, 512)
    check_attention(*run_attention(ctx, pool, q, q_pe, tables, lens, 192 ** -0.5, table_of=rows), *want)


@pytest.mark.parametrize("ggml_type", [mm.F16, mm.Q8_0])
@pytest.mark.parametrize("heads", [7, 20, 33])
def test_attention_unaligned_rows(ctx, ggml_type, heads):
    """Queries and outputs whose rows are not 16-byte aligned, of whole and of split tokens: the bits of aligned ones."""
    rng = np.random.default_rng(heads)
    pt, lens = 16, np.array([3, 1700, 0, 40, 16])
    n_pages = 200
    pool = Pool(rng, ggml_type, 512, 64, pt, n_pages)
    tables = tables_for(rng, lens, pt, n_pages)
    q, q_pe = queries(rng, len(lens), heads, 512, 64)
    a = run_attention(ctx, pool, q, q_pe, tables, lens, 0.07)
    b = run_attention(ctx, pool, q, q_pe, tables, lens, 0.07, pad=1)
    same_bits(a[0], b[0])
    same_bits(a[1], b[1])
    check_attention(*a, *ref.attention64(q, q_pe, pool.values, tables, np.arange(len(lens)), lens, pt, 0.07, 512))


@pytest.mark.parametrize("ggml_type", [mm.F16, mm.Q8_0])
def test_attention_many_ragged_tokens(ctx, ggml_type):
    """More tokens than the chip has workgroups, most of them short, empty ones between, a few long."""
    rng = np.random.default_rng(31)
    n, pt = 700, 16
    lens = np.where(rng.random(n) < 0.2, 0, np.exp(rng.uniform(0, np.log(200), n)).astype(np.int64))
    lens[::97] = 900
    lens[-1] = 0
    n_pages = 400
    pool = Pool(rng, ggml_type, 512, 64, pt, n_pages)
    tables = rng.integers(0, n_pages, (50, 60)).astype(np.int32)
    rows = rng.integers(0, 50, n)
    q, q_pe = queries(rng, n, 3, 512, 64)
    want = ref.attention64(q, q_pe, pool.values, tables, rows, lens, pt, 192 ** -0.5, 512)
    check_attention(*run_attention(ctx, pool, q, q_pe, tables, lens, 192 ** -0.5, table_of=rows), *want)


@pytest.mark.parametrize("ggml_type", [mm.F16, mm.Q8_0])
@pytest.mark.parametrize("sigma", [0.0, 1e-3, 12.0, 1e4])
def test_attention_score_sizes(ctx, ggml_type, sigma):
    """Even probabilities, and scores so far apart that one position takes all: small queries, large ones, and scores
    that rise and fall over the positions, so that the running maximum changes late and early."""
    rng = np.random.default_rng(5)
    pt, length = 16, 1000
    n_pages = (length + pt - 1) // pt
    pool = Pool(rng, ggml_type, 512, 64, pt, n_pages)
    tables = tables_for(rng, [length], pt, n_pages)
    q, q_pe = queries(rng, 4, 20, 512, 64, sigma)
    lens = np.array([length, length - 1, 333, 1])
    rows = np.zeros(4, np.int64)
    want, want_lse = ref.attention64(q, q_pe, pool.values, tables, rows, lens, pt, 192 ** -0.5, 512)
    out, lse = run_attention(ctx, pool, q, q_pe, tables, lens, 192 ** -0.5, table_of=rows)
    # A score's own error grows with its size (22 bits of the query, sums in f32): the sum's terms of random sign are
    # |q| |c| scale ~ 1.7 sigma each way, their rounding a few u of that.
    tol = 1e-5 * max(1.0, sigma)
    if sigma < 1000:
        err = np.linalg.norm(out - want, axis=-1) / np.linalg.norm(want, axis=-1)
        assert err.max() <= tol
    # lse of one position is that score, which may be small where its terms are not: 576 additions, each rounded by at
    # most u times a partial sum, whose size is up to 2 * 1.7 sigma; uniform errors of independent sign add up to
    # sqrt(576 / 3) u * 3.4 sigma = 2.8e-6 sigma (one standard deviation), four of them 1.2e-5 sigma.
    assert (np.abs(lse - want_lse) <= 1e-5 * np.maximum(1, np.abs(want_lse)) + 1.2e-5 * sigma).all()


@pytest.mark.parametrize("ggml_type", [mm.F16, mm.Q8_0])
def test_attention_bad_tables(ctx, ggml_type):
    """Pages that the pool does not have count as masked, lengths beyond a table end with it, rows that do not exist see
    nothing; each is reported."""
    rng = np.random.default_rng(8)
    pt, n_pages = 16, 12
    pool = Pool(rng, ggml_type, 512, 64, pt, n_pages)
    tables = rng.permutation(n_pages).reshape(2, 6).astype(np.int32)
    q, q_pe = queries(rng, 2, 20, 512, 64)
    scale = 192 ** -0.5
    ids = np.arange(2)
    holes = tables.copy()
    holes[0, 2], holes[0, 5], holes[1, 0], holes[1, 1] = n_pages, -5, 2 ** 31 - 1, -2 ** 31
    lens = np.array([96, 90])
    want = ref.attention64(q, q_pe, pool.values, holes, ids, lens, pt, scale, 512)
    check_attention(*run_attention(ctx, pool, q, q_pe, holes, lens, scale, expect="page"), *want)
    gone = np.full((2, 6), -1, np.int32)
    gone[1] = tables[1]
    want = ref.attention64(q, q_pe, pool.values, gone, ids, lens, pt, scale, 512)
    check_attention(*run_attention(ctx, pool, q, q_pe, gone, lens, scale, expect="page"), *want)
    long = np.array([50, 2 ** 32 - 1])
    want = ref.attention64(q, q_pe, pool.values, tables, ids, long, pt, scale, 512)
    check_attention(*run_attention(ctx, pool, q, q_pe, tables, long, scale, expect="length"), *want)
    rows = np.array([1, 2])
    want = ref.attention64(q, q_pe, pool.values, tables, rows, lens, pt, scale, 512)
    check_attention(*run_attention(ctx, pool, q, q_pe, tables, lens, scale, table_of=rows, expect="row"), *want)


@pytest.mark.parametrize("ggml_type", [mm.F16, mm.Q8_0])
def test_attention_not_a_number(ctx, ggml_type):
    """A NaN in a seen row's latent part reaches its tokens' outputs, and no other token's."""
    rng = np.random.default_rng(12)
    pool = Pool(rng, ggml_type, 512, 64, 16, 8)
    tables = np.arange(8, dtype=np.int32).reshape(2, 4)
    pool.spoil(1, 3)
    q, q_pe = queries(rng, 2, 20, 512, 64)
    lens = np.array([64, 64])
    out, lse = run_attention(ctx, pool, q, q_pe, tables, lens, 0.07)
    assert np.isnan(out[0]).all() and np.isnan(lse[0]).all()
    want, want_lse = ref.attention64(q, q_pe, pool.values, tables, np.arange(2), lens, 16, 0.07, 512)
    check_attention(out[1:], lse[1:], want[1:], want_lse[1:])
    q[0, 0, 5] = np.nan
    q[1, 2, 7] = np.inf
    pool = Pool(rng, ggml_type, 512, 64, 16, 8)
    out, lse = run_attention(ctx, pool, q, q_pe, tables, lens, 0.07)
    assert np.isnan(out[0, 0]).all() and np.isfinite(out[0, 1:]).all()
    assert np.isnan(out[1, 2]).all() and np.isfinite(np.delete(out[1], 2, 0)).all()


@pytest.mark.parametrize("ggml_type", [mm.F16, mm.Q8_0])
def test_attention_far_into_a_pool(ctx, ggml_type):
    """Pages whose bytes lie beyond 2^32 (the pool is larger; only the last pages are written)."""
    rng = np.random.default_rng(4)
    pt = 1024
    page = mm.KvCache.page_bytes(ggml_type, 512, 64, pt)
    n_pages = (5 << 30) // page + 2
    pool = Pool(rng, ggml_type, 512, 64, pt, 2)
    q, q_pe = queries(rng, 1, 20, 512, 64)
    lens = np.array([1500])
    want = ref.attention64(q, q_pe, pool.values, np.array([[1, 0]]), [0], lens, pt, 0.07, 512)
    with Buffers(ctx) as d:
        big = mm.DeviceArray(ctx, n_pages * page)
        d.held.append(big)
        at = (n_pages - 2) * page
        mm.check(ctx.lib.mmhip_memcpy_h2d(ctx.handle, big.ptr + at, pool.bytes.ctypes.data, pool.bytes.nbytes), "h2d")
        cache = mm.KvCache(big, ggml_type, rank=512, rope_dims=64, page_tokens=pt, n_pages=n_pages)
        # one of the rows is written there by the cache's writer
        row = pool.values[1, 9].astype(np.float32)
        ctx.kv_store_dev(cache, d.put(row), d.put(np.array([(n_pages - 1) * pt + 9], np.int32)), 1)
        do, dl = d.new(20 * 512 * 4), d.new(80)
        ctx.mla_attention_dev(ctx.mla_attention_args(
            cache, q=d.put(q), q_pe=d.put(q_pe), out=do, lse=dl, lens=d.put(lens.astype(np.uint32)),
            tables=d.put(np.array([n_pages - 1, n_pages - 2], np.int32)), n_tables=1, table_pages=2, n_tokens=1,
            n_heads=20, scale=0.07, workspace=d.new(ctx.mla_attention_workspace(1, 20, 512))))
        ctx.synchronize()
        check_attention(f32(do, 20 * 512).reshape(1, 20, 512), f32(dl, 20).reshape(1, 20), *want)


def test_attention_refuses_a_small_workspace(ctx):
    need = ctx.mla_attention_workspace(4, 20, 512)
    if need == 0:
        return
    with Buffers(ctx) as d:
        b = d.new(1 << 20, 0)
        cache = mm.KvCache(b, mm.F16, rank=512, rope_dims=64, page_tokens=16, n_pages=4)
        kw = dict(q=b, q_pe=b, out=d.new(4 * 20 * 512 * 4), lens=d.put(np.zeros(4, np.uint32)), tables=d.put(np.zeros(4, np.int32)),
                  n_tables=4, table_pages=1, n_tokens=4, n_heads=20, scale=0.1)
        work = d.new(need + 16)
        for w in (At(work, 0, need - 1), At(work, 8, need)):
            with pytest.raises(mm.MmhipError, match="workspace"):
                ctx.mla_attention_dev(ctx.mla_attention_args(cache, workspace=w, **kw))
        ctx.mla_attention_dev(ctx.mla_attention_args(cache, workspace=At(work, 16, need), **kw))
        ctx.synchronize()


# ---- log probabilities ----------------------------------------------------

def run_logprobs(ctx, x, tokens=None, top=0, pad=0, off=0, entropy=True, top_logp=True, expect=None):
    n, v = x.shape
    g = 0 if tokens is None else tokens.shape[1]
    with Buffers(ctx) as d:
        buf = np.full((n, v + pad), 1e30, np.float32)  # what lies between the rows is larger than all of them
        buf[:, :v] = x
        dx = At(d.put(np.concatenate([np.full(off, 1e30, np.float32), buf.ravel(), np.full(8, 1e30, np.float32)])), 4 * off)
        lp, en, ids, tlp = d.new(n * g * 4), d.new(n * 4), d.new(n * top * 4), d.new(n * top * 4)
        kw = dict(stride=v + pad, tokens=None if tokens is None else d.put(tokens.astype(np.uint32)), n_given=g,
                  token_logprobs=lp, entropy=en if entropy else None, top=top, top_ids=ids,
                  top_logprobs=tlp if top_logp else None, workspace=d.new(ctx.logprobs_workspace(n, v, top)))
        ctx.logprobs_dev(dx, n, v, **kw)
        ctx.logprobs_dev(dx, n, v, **kw)
        if expect:
            with pytest.raises(mm.MmhipError, match=expect):
                ctx.synchronize()
        ctx.synchronize()
        return (f32(lp, n * g).reshape(n, g), f32(en, n), ids.to_numpy(np.uint32, n * top).reshape(n, top),
                f32(tlp, n * top).reshape(n, top))


def check_logprobs(x, tokens, top, got):
    lp, h = ref.logprobs64(x)
    ids = ref.top_ids(x, top)
    near = lambda a, b: (np.isnan(a) & np.isnan(b)) | (a == b) | (np.abs(a - b) <= 6e-6 + 2 * U * np.abs(b))  # noqa: E731
    with np.errstate(invalid="ignore"):
        if tokens is not None:
            assert near(got[0], np.take_along_axis(lp, tokens.astype(np.int64), 1)).all()
        assert np.array_equal(np.isnan(got[1]), np.isnan(h))
        ok = ~np.isnan(h)
        assert (np.abs(got[1] - h)[ok] <= 6e-6 * (1 + np.abs(h[ok]) * 2)).all()
        assert np.array_equal(got[2], ids)
        assert near(got[3], np.take_along_axis(lp, ids.astype(np.int64), 1)).all()


@pytest.mark.parametrize("n,v", [(1, 154880), (3, 32000), (2, 4097), (5, 1000), (2, 33), (1, 1), (70, 2048), (2, 8191),
                                 (1, 1 << 20)])
@pytest.mark.parametrize("top", [0, 1, 5, 20, 32])
def test_logprobs(ctx, n, v, top):
    top = min(top, v)
    rng = np.random.default_rng(v + top)
    x = (rng.standard_normal((n, v)) * 3).astype(np.float32)
    x[:, rng.integers(0, v, 3)] += 8
    tokens = rng.integers(0, v, (n, 3))
    got = run_logprobs(ctx, x, tokens, top)
    check_logprobs(x, tokens, top, got)
    for kw in (dict(pad=4), dict(pad=1, off=1), dict(off=3)):  # the same bits wherever the rows lie
        for a, b in zip(run_logprobs(ctx, x, tokens, top, **kw), got):
            same_bits(a, b)


@pytest.mark.parametrize("v", [300, 5000, 154880])
def test_logprobs_ties_and_masks(ctx, v):
    rng = np.random.default_rng(v)
    x = np.zeros((8, v), np.float32)
    x[1] = rng.integers(0, 3, v)                       # many equal largest
    x[2] = -np.inf
    x[2, v - 1] = -1e38                                # all but one masked
    x[3] = np.where(rng.random(v) < 0.95, -np.inf, rng.standard_normal(v))
    x[3, 11] = 0.0
    x[4] = np.sort(rng.standard_normal(v))             # rising: the largest lie together at the end
    x[5] = -np.sort(rng.standard_normal(v))
    x[6] = np.finfo(np.float32).min                    # masked with the lowest value
    x[6, 100:140] = rng.standard_normal(40)
    x[7] = np.where(np.arange(v) % 2 == 0, -0.0, 0.0)  # zeros of both signs are equal
    tokens = np.stack([np.zeros(8, np.int64), np.full(8, v - 1), np.full(8, 11)], 1)
    got = run_logprobs(ctx, x, tokens, 32)
    check_logprobs(x, tokens, 32, got)
    assert np.array_equal(got[2][0], np.arange(32)) and np.array_equal(got[2][7], np.arange(32))


def test_logprobs_without_probabilities(ctx):
    """NaN, +infinity and nothing but -infinity in a row: NaN, with ids that still follow the logits."""
    v = 3000
    rng = np.random.default_rng(1)
    x = rng.standard_normal((6, v)).astype(np.float32)
    x[0, 1234] = np.nan
    x[1, 77] = np.inf
    x[2] = -np.inf
    x[3] = np.nan
    x[4, ::2] = np.nan
    x[4, 1] = np.inf
    x[4, 3:] = np.nan
    tokens = np.array([[0, 1234, 77]] * 6)
    got = run_logprobs(ctx, x, tokens, 8)
    for r in range(5):
        assert np.isnan(got[0][r]).all() and np.isnan(got[1][r]) and np.isnan(got[3][r]).all(), r
    assert np.array_equal(got[2], ref.top_ids(x, 8))
    check_logprobs(x[5:], tokens[5:], 8, tuple(g[5:] for g in got))


@pytest.mark.parametrize("n,v", [(1100, 12300), (300, 20000), (1, (1 << 22) + 5)])
@pytest.mark.parametrize("top", [1, 32])
def test_logprobs_long_pieces(ctx, n, v, top):
    """Rows whose pieces take several steps, the largest found so far going from one to the next: rising, falling and
    equal logits, the largest in the last step, masks, NaN late in a row."""
    rng = np.random.default_rng(n + top)
    x = (rng.standard_normal((n, v)) * 3).astype(np.float32)
    for r in range(n):
        kind = r % 11
        if kind == 1:
            x[r].sort()
        elif kind == 2:
            x[r] = np.sort(x[r])[::-1]
        elif kind == 3:
            x[r] = 2.5
        elif kind == 4:
            x[r] = np.rint(x[r] / 4)
        elif kind == 5:
            x[r, :-20] = -np.inf
        elif kind == 6:
            x[r, -7:] = np.nan
        elif kind == 7:
            x[r, 40:] = np.finfo(np.float32).min
        elif kind == 8:
            x[r, :-3] = np.nan
        elif kind == 9:
            x[r, v // 2] = np.inf
        elif kind == 10:
            x[r] = np.where(np.arange(v) < v - 33, -np.inf, -0.0)
    tokens = rng.integers(0, v, (n, 2))
    check_logprobs(x, tokens, top, run_logprobs(ctx, x, tokens, top))


def test_logprobs_refuses_a_small_workspace(ctx):
    need = ctx.logprobs_workspace(3, 5000, 7)
    assert need > 0
    with Buffers(ctx) as d:
        x, out = d.put(np.zeros((3, 5000), np.float32)), d.new(3 * 7 * 4)
        work = d.new(need + 16)
        for w in (At(work, 0, need - 1), At(work, 8, need)):
            with pytest.raises(mm.MmhipError, match="workspace"):
                ctx.logprobs_dev(x, 3, 5000, top=7, top_ids=out, workspace=w)
        ctx.logprobs_dev(x, 3, 5000, top=7, top_ids=out, workspace=At(work, 16, need))
        ctx.synchronize()
        assert np.array_equal(out.to_numpy(np.uint32, 21).reshape(3, 7), np.tile(np.arange(7), (3, 1)))


def test_logprobs_outputs_left_out(ctx):
    rng = np.random.default_rng(6)
    x = rng.standard_normal((3, 5000)).astype(np.float32)
    tokens = rng.integers(0, 5000, (3, 1))
    whole = run_logprobs(ctx, x, tokens, 7)
    part = run_logprobs(ctx, x, tokens, 7, entropy=False, top_logp=False)
    same_bits(part[0], whole[0])
    assert np.array_equal(part[2], whole[2]) and np.isnan(part[1]).all() and np.isnan(part[3]).all()
    lone = run_logprobs(ctx, x, None, 0)
    same_bits(lone[1], whole[1])


def test_logprobs_bad_tokens(ctx):
    rng = np.random.default_rng(6)
    x = rng.standard_normal((2, 100)).astype(np.float32)
    tokens = np.array([[5, 100], [2 ** 32 - 1, 99]])
    got = run_logprobs(ctx, x, tokens, 3, expect="vocabulary")
    lp, _ = ref.logprobs64(x)
    assert np.isnan(got[0][0, 1]) and np.isnan(got[0][1, 0])
    assert abs(got[0][0, 0] - lp[0, 5]) <= 6e-6 and abs(got[0][1, 1] - lp[1, 99]) <= 6e-6


# ---- together -------------------------------------------------------------

class Step:
    """A decode step's part between products for `n` conversations: norm, rope of the queries, the cache's write,
    attention, and the log probabilities of logits in hand."""

    def __init__(self, ctx, d, rng, ggml_type, lens, vocab=5000):
        self.ctx, self.n, self.lens = ctx, len(lens), np.array(lens)
        n, pt = self.n, 16
        self.n_pages = int(((self.lens + pt - 1) // pt).sum()) + 1
        self.pool = Pool(rng, ggml_type, 512, 64, pt, self.n_pages)
        self.tables = tables_for(rng, self.lens, pt, self.n_pages)
        last = self.lens - 1
        self.slots = self.tables[np.arange(n), last // pt] * pt + last % pt
        self.rope = mm.Rope(ctx, dims=64, base=1e6)
        self.w, self.wkv = (rng.standard_normal(k).astype(np.float32) for k in (2048, 512))
        self.d = {k: d.new(4 * v) for k, v in dict(hidden=n * 2048, res=n * 2048, normed=n * 2048, q=n * 20 * 192,
                                                   q_lat=n * 20 * 512, kv=n * 576, out=n * 20 * 512, lse=n * 20,
                                                   logits=n * vocab, lp=n, en=n, ids=n * 5, tlp=n * 5).items()}
        self.dw, self.dwkv = d.put(self.w), d.put(self.wkv)
        self.dpool, self.dpos = d.put(self.pool.bytes), d.put(last.astype(np.uint32))
        self.dslots, self.dtok = d.put(self.slots.astype(np.int32)), d.put(np.arange(n, dtype=np.uint32))
        self.cache = mm.KvCache(self.dpool, ggml_type, rank=512, rope_dims=64, page_tokens=pt, n_pages=self.n_pages)
        self.args = ctx.mla_attention_args(
            self.cache, q=self.d["q_lat"], q_pe=self.d["q"], q_pe_offset=128 * 4, q_pe_strides=(20 * 192, 192),
            out=self.d["out"], lse=self.d["lse"], lens=d.put(self.lens.astype(np.uint32)), tables=d.put(self.tables),
            n_tables=n, table_pages=self.tables.shape[1], n_tokens=n, n_heads=20, scale=192 ** -0.5,
            workspace=d.new(ctx.mla_attention_workspace(n, 20, 512)))
        self.vocab, self.work = vocab, d.new(ctx.logprobs_workspace(n, vocab, 5))

    def fill(self, rng):
        self.x = {k: rng.standard_normal(s).astype(np.float32) for k, s in dict(
            hidden=(self.n, 2048), res=(self.n, 2048), q=(self.n, 20, 192), q_lat=(self.n, 20, 512), kv=(self.n, 576),
            logits=(self.n, self.vocab)).items()}
        for k, v in self.x.items():
            mm.check(self.ctx.lib.mmhip_memcpy_h2d(self.ctx.handle, self.d[k].ptr, v.ctypes.data, v.nbytes), "h2d")

    def run(self):
        c, d, n = self.ctx, self.d, self.n
        c.rms_norm_dev(d["normed"], d["hidden"], self.dw, n, 2048, residual=d["res"], sum_out=d["res"])
        c.rope_dev(self.rope, d["q"], d["q"], self.dpos, n, 20, 192, first=128)
        c.kv_store_dev(self.cache, d["kv"], self.dslots, n, norm_weight=self.dwkv, rope=self.rope, positions=self.dpos)
        c.mla_attention_dev(self.args)
        c.logprobs_dev(d["logits"], n, self.vocab, tokens=self.dtok, n_given=1, token_logprobs=d["lp"], entropy=d["en"],
                       top=5, top_ids=d["ids"], top_logprobs=d["tlp"], workspace=self.work)

    def results(self):
        self.ctx.synchronize()
        n = self.n
        return dict(normed=f32(self.d["normed"], n * 2048), res=f32(self.d["res"], n * 2048), q=f32(self.d["q"], n * 20 * 192),
                    pool=self.dpool.to_numpy(np.uint8, self.pool.bytes.size), out=f32(self.d["out"], n * 20 * 512),
                    lse=f32(self.d["lse"], n * 20), lp=f32(self.d["lp"], n), en=f32(self.d["en"], n),
                    ids=self.d["ids"].to_numpy(np.uint32, n * 5), tlp=f32(self.d["tlp"], n * 5))

    def check(self, got):
        """The whole step in 64 bits, from the inputs to the attention's output."""
        x, n = self.x, self.n
        s = x["hidden"] + x["res"]
        want = ref.rms_norm64(s, self.w, np.float64(np.float32(1e-5)))
        assert (np.abs(got["normed"].reshape(want.shape) - want) <= 3.1 * U * np.abs(want)).all()
        same_bits(got["res"].reshape(s.shape), s)
        pos, freqs = self.lens - 1, ref.frequencies64(64, 1e6)
        q_pe = ref.rope64(x["q"][..., 128:], pos, "interleaved", freqs)
        row = np.concatenate([ref.rms_norm64(x["kv"][:, :512], self.wkv, np.float64(np.float32(1e-5))),
                              ref.rope64(x["kv"][:, None, 512:], pos, "interleaved", freqs)[:, 0]], 1).astype(np.float32)
        values = self.pool.values.copy()
        for t, sl in enumerate(self.slots):
            if self.pool.type == mm.F16:
                values[sl // 16, sl % 16] = row[t].astype(np.float16)
            else:
                c, d = ref.q8_blocks(row[t])
                values[sl // 16, sl % 16] = (c.reshape(-1, 32) * d.astype(np.float64)[:, None]).ravel()
        want, lse = ref.attention64(x["q_lat"], q_pe, values, self.tables, np.arange(n), self.lens, 16, 192 ** -0.5, 512)
        # the stored row may differ by one step of its own format from the one rounded here: one position in lens[t]
        err = np.linalg.norm(got["out"].reshape(want.shape) - want, axis=-1) / np.linalg.norm(want, axis=-1)
        assert err.max() <= 1e-3
        tokens = np.arange(n)[:, None]
        check_logprobs(x["logits"], tokens, 5, (got["lp"].reshape(n, 1), got["en"], got["ids"].reshape(n, 5),
                                                got["tlp"].reshape(n, 5)))


@pytest.mark.parametrize("ggml_type", [mm.F16, mm.Q8_0])
def test_step_together(ctx, ggml_type):
    rng = np.random.default_rng(77)
    with Buffers(ctx) as d:
        step = Step(ctx, d, rng, ggml_type, [200, 17, 1, 64, 333])
        step.fill(rng)
        step.run()
        step.check(step.results())
        step.rope.free()


@pytest.mark.parametrize("ggml_type", [mm.F16, mm.Q8_0])
def test_step_captured_and_replayed(ctx, ggml_type):
    """A captured step replayed on other inputs, the program's own calls between the replays: the bits of the calls made
    one by one."""
    rng = np.random.default_rng(78)
    with Buffers(ctx) as d:
        step, eager = (Step(ctx, d, np.random.default_rng(5), ggml_type, [700, 17, 1, 1300]) for _ in range(2))
        step.fill(rng)
        step.run()  # the kernels are loaded outside the capture
        ctx.synchronize()
        g = Graph(ctx, step.run)
        try:
            for i in range(4):
                state = rng.bit_generator.state
                step.fill(rng)
                rng.bit_generator.state = state
                eager.fill(rng)
                g.replay()
                eager.run()
                a, b = step.results(), eager.results()
                for k in a:
                    same_bits(a[k], b[k])
        finally:
            g.free()
            step.rope.free()
            eager.rope.free()


def test_two_contexts_at_once(mm, ctx):
    """Two contexts' steps queued together on one device: each as alone."""
    with mm.Context(0) as other, Buffers(ctx) as d, Buffers(other) as e:
        pair = [Step(ctx, d, np.random.default_rng(5), mm.F16, [3000, 17, 900, 1300] * 8),
                Step(other, e, np.random.default_rng(6), mm.Q8_0, [2500, 64, 1, 800] * 8)]
        for i, s in enumerate(pair):
            s.fill(np.random.default_rng(40 + i))
            s.run()
        alone = [s.results() for s in pair]
        for i, s in enumerate(pair):
            s.fill(np.random.default_rng(40 + i))
        for _ in range(3):  # the norm's residual is its own sum: only the first pass has the same inputs for it
            for s in pair:
                s.ctx.mla_attention_dev(s.args)
                s.ctx.logprobs_dev(s.d["logits"], s.n, s.vocab, tokens=s.dtok, n_given=1, token_logprobs=s.d["lp"],
                                   entropy=s.d["en"], top=5, top_ids=s.d["ids"], top_logprobs=s.d["tlp"], workspace=s.work)
        for s in pair:
            s.run()
        for s, want in zip(pair, alone):
            got = s.results()
            for k in ("out", "lse", "lp", "en", "ids", "tlp", "pool"):
                same_bits(got[k], want[k])
            s.rope.free()
