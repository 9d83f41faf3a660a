"""The operators between a decode step's products where their numbers or their
dispatch can go wrong: infinite cached values, block scales of all sizes, the
precision of the operands, large finite queries, every kernel the attention can
take. Against the plain 64-bit forms of tests/step_reference.py; u = 2^-24, half a
step of f32."""
import numpy as np
import pytest

import mmhip as mm
import step_reference as ref
from step_reference import Buffers, Graph, Pool, U
from test_gpu_step_ops import check_attention, f32, queries, run_attention, run_logprobs, same_bits, tables_for

pytestmark = pytest.mark.gpu


def parts(pool):
    """Views of a pool's codes [pages, rows, width] and scales [pages, rows, width / 32]."""
    w, pt = pool.width, pool.page_tokens
    codes = pool.bytes[:, :pt * w].view(np.int8).reshape(pool.n_pages, pt, w)
    scales = pool.bytes[:, pt * w:].view(np.float16).reshape(pool.n_pages, pt, w // 32)
    return codes, scales


def revalue(pool):
    """The values that the pool's bytes stand for now."""
    if pool.type == mm.F16:
        pool.values = pool.bytes.view(np.float16).reshape(pool.values.shape).astype(np.float64)
    else:
        codes, scales = parts(pool)
        with np.errstate(invalid="ignore"):
            pool.values = (codes.reshape(*codes.shape[:2], -1, 32).astype(np.float64) * scales.astype(np.float64)[..., None]) \
                .reshape(codes.shape)


# ---- operands of 24 bits --------------------------------------------------

@pytest.mark.parametrize("ggml_type", [mm.F16, mm.Q8_0])
@pytest.mark.parametrize("heads", [5, 20, 33])
def test_attention_uses_every_bit_of_a_query(ctx, ggml_type, heads):
    """A query of 2 - 2^-23 against -2: the score is -2^-23 times the cached value, all of it the query's last bit. (Its
    terms are below 2^17 and are added with three roundings of at most half a step, 2^-8 each.)"""
    rng = np.random.default_rng(1)
    pool = Pool(rng, ggml_type, 512, 64, 16, 1)
    c = 65504.0 if ggml_type == mm.F16 else 127 * 512.0
    if ggml_type == mm.F16:
        pool.bytes.view(np.float16)[...] = 0
        pool.bytes.view(np.float16).reshape(16, 576)[0, [40, 41]] = c
    else:
        codes, scales = parts(pool)
        codes[...], scales[...] = 0, 512.0
        codes[0, 0, [40, 41]] = 127
    q, q_pe = np.zeros((1, heads, 512), np.float32), np.zeros((1, heads, 64), np.float32)
    q[..., 40], q[..., 41] = np.float32(2 - 2.0 ** -23), -2.0
    lse = run_attention(ctx, pool, q, q_pe, np.zeros((1, 1)), np.array([1]), 1.0)[1]
    assert (np.abs(lse + c * 2.0 ** -23) <= 3 * 2.0 ** -8).all(), lse


@pytest.mark.parametrize("ggml_type", [mm.F16, mm.Q8_0])
@pytest.mark.parametrize("heads", [5, 20, 33])
@pytest.mark.parametrize("length", [32, 900])
def test_attention_probabilities_add_up_to_one(ctx, ggml_type, heads, length):
    """Where every cached value is 1.25, so is the output, up to roundings to nearest (running sums, the division): as
    much as forty whole ones on a value's way, without a side. The mean over N values then has a deviation of at most
    sqrt(40 / 3 / N) u; 4 of these for N = 4000 are 0.23 u, and 0.4 u is allowed. Probabilities cut to 22 bits are 1.25 u
    too small."""
    rng = np.random.default_rng(heads + length)
    pt, n_pages, n = 16, (length + 15) // 16, (4000 + heads - 1) // heads
    pool = Pool(rng, ggml_type, 512, 64, pt, n_pages)
    if ggml_type == mm.F16:
        pool.bytes.view(np.float16).reshape(n_pages, pt, 576)[..., :512] = 1.25
    else:
        codes, scales = parts(pool)
        codes[..., :512], scales[..., :16] = 80, 2.0 ** -6
    q, q_pe = np.zeros((n, heads, 512), np.float32), rng.standard_normal((n, heads, 64)).astype(np.float32)
    out, _ = run_attention(ctx, pool, q, q_pe, np.arange(n_pages)[None], np.full(n, length), 0.1, table_of=np.zeros(n, np.int64))
    assert (np.abs(out - 1.25) <= 1e-5 * 1.25).all()
    mean = (out.astype(np.float64) / 1.25 - 1).mean()
    assert abs(mean) <= 0.4 * U, mean / U


# ---- block scales of all sizes --------------------------------------------

@pytest.mark.parametrize("heads", [5, 20, 33])
@pytest.mark.parametrize("rank,pe", [(512, 64), (480, 64)])
@pytest.mark.parametrize("length,where", [(60, "early"), (60, "late"), (3000, "early"), (3000, "late"), (3000, "spread")])
def test_attention_block_scales(ctx, heads, rank, pe, length, where):
    """Block scales from 2^-14 to f16's largest in one context. For the first token the rotary part gives weight to some
    rows of small scales alone, the same to each: its output is their mean, where a value loses nothing to what else is
    cached. (38 rows count, of equal probabilities: as many additions, the probability's rounding and the division, less
    than 64 u of the column's largest.) For the second token every row counts: 1e-5 of the output's norm per block of
    columns, as everywhere."""
    rng = np.random.default_rng(heads + length + rank)
    pt, n_pages = 16, (length + 15) // 16
    pool = Pool(rng, mm.Q8_0, rank, pe, pt, n_pages)
    codes, scales = parts(pool)
    nb = rank // 32
    row = np.arange(n_pages * pt).reshape(n_pages, pt)
    big = {"early": row < 20, "late": row >= length - 20, "spread": row % 13 == 5}[where]
    small = np.isin(row, rng.choice(row[~big & (row < length)], 38, replace=False))
    scales[..., :nb] = np.exp2(rng.uniform(-14, -3, (n_pages, pt, nb)))
    scales[small, :nb] = np.exp2(rng.uniform(-14, -11, (38, nb)))
    mixed = rng.random((n_pages, pt, nb)) < 0.5  # not every block of such a row
    scales[..., :nb] = np.where(big[..., None] & mixed, np.exp2(rng.uniform(8, 15.9, (n_pages, pt, nb))), scales[..., :nb])
    # the first rotary value: 1 for the small rows, -1 for all others
    codes[..., rank:], scales[..., nb:] = 0, 2.0 ** -6
    codes[..., rank] = np.where(small, 64, -64)
    revalue(pool)
    q, q_pe = np.zeros((2, heads, rank), np.float32), np.zeros((2, heads, pe), np.float32)
    q_pe[0, :, 0] = 200.0  # 400 between the two kinds
    q_pe[1] = rng.standard_normal((heads, pe))
    lens, ids = np.array([length, length]), np.zeros(2, np.int64)
    tables = np.arange(n_pages)[None]
    want, want_lse = ref.attention64(q, q_pe, pool.values, tables, ids, lens, pt, 1.0, rank)
    out, lse = run_attention(ctx, pool, q, q_pe, tables, lens, 1.0, table_of=ids)
    assert np.isfinite(out).all()
    most = np.abs(pool.values[small, :rank]).max(0)
    assert (np.abs(out[0] - want[0]) <= 64 * U * most).all()
    err = np.linalg.norm((out[1] - want[1]).reshape(heads, nb, 32), axis=-1)
    assert (err <= 1e-5 * np.linalg.norm(want[1].reshape(heads, nb, 32), axis=-1)).all()
    assert (np.abs(lse - want_lse) <= 1e-5 * np.maximum(1, np.abs(want_lse))).all()


# ---- infinities -----------------------------------------------------------

def infinite_row(pool, page, at, col, sign):
    """A value of the row (a whole block of it in Q8_0, all of one sign) becomes infinite."""
    if pool.type == mm.F16:
        pool.bytes.view(np.float16).reshape(pool.n_pages, pool.page_tokens, -1)[page, at, col] = sign * np.inf
        return [col]
    codes, scales = parts(pool)
    b = col // 32
    codes[page, at, 32 * b:32 * b + 32] = sign * 5
    scales[page, at, b] = np.inf
    return list(range(32 * b, 32 * b + 32))


@pytest.mark.parametrize("ggml_type", [mm.F16, mm.Q8_0])
@pytest.mark.parametrize("heads", [5, 16, 17, 20, 24, 33])
@pytest.mark.parametrize("rank,pe,length", [(512, 64, 50), (512, 64, 2000), (96, 32, 50)])
def test_attention_infinite_rotary_values(ctx, ggml_type, heads, rank, pe, length):
    """A score of -infinity only drops its position, one of +infinity gives NaN, whatever the query's bits: the values of
    every other head are those of the formula."""
    rng = np.random.default_rng(heads + rank)
    pt, n_pages = 16, (length + 15) // 16
    pool = Pool(rng, ggml_type, rank, pe, pt, n_pages)
    q, q_pe = queries(rng, 2, heads, rank, pe)
    q_pe[:, ::2] = np.where(q_pe[:, ::2] < 0, -0.5, 0.5)  # bits that fit f16: nothing is left for a second part
    for at, col in ((3, rank + pe - 3), (17, rank + 1), (length - 1, rank + pe - 20)):
        cols = [c - rank for c in infinite_row(pool, at // pt, at % pt, col, -1)]
        q_pe[..., cols] = np.abs(q_pe[..., cols])
    revalue(pool)
    up = np.zeros(heads, bool)
    up[[1, heads - 1]] = True
    q_pe[1, up] *= -1  # the second token's heads 1 and last: +infinity (some rows also -infinity)
    lens, ids, tables = np.array([length, length]), np.zeros(2, np.int64), np.arange(n_pages)[None]
    with np.errstate(invalid="ignore"):
        want, want_lse = ref.attention64(q, q_pe, pool.values, tables, ids, lens, pt, 0.07, rank)
    out, lse = run_attention(ctx, pool, q, q_pe, tables, lens, 0.07, table_of=ids)
    assert np.isnan(want[1, up]).all() and np.isfinite(want[0]).all() and np.isfinite(want[1, ~up]).all()
    assert np.isnan(out[1, up]).all() and np.isnan(lse[1, up]).all()
    check_attention(out[0], lse[0], want[0], want_lse[0])
    check_attention(out[1, ~up], lse[1, ~up], want[1, ~up], want_lse[1, ~up])


@pytest.mark.parametrize("ggml_type", [mm.F16, mm.Q8_0])
@pytest.mark.parametrize("heads", [5, 20, 33])
def test_attention_infinite_latent_values(ctx, ggml_type, heads):
    """An infinite latent value whose score is -infinity: NaN in its own columns (0 times infinity), the formula's values
    in all others."""
    rng = np.random.default_rng(heads)
    pool = Pool(rng, ggml_type, 512, 64, 16, 4)
    q, q_pe = queries(rng, 1, heads, 512, 64)
    cols = infinite_row(pool, 2, 5, 300, 1)
    revalue(pool)
    q[..., cols] = -np.abs(q[..., cols])
    q[:, ::2, cols] = -0.25
    lens, tables = np.array([64]), np.arange(4)[None]
    with np.errstate(invalid="ignore"):
        want, want_lse = ref.attention64(q, q_pe, pool.values, tables, [0], lens, 16, 0.07, 512)
    out, lse = run_attention(ctx, pool, q, q_pe, tables, lens, 0.07)
    assert np.isnan(out[..., cols]).all()
    keep = np.setdiff1d(np.arange(512), cols)
    check_attention(out[..., keep], lse, want[..., keep], want_lse)


@pytest.mark.parametrize("ggml_type", [mm.F16, mm.Q8_0])
def test_attention_without_a_finite_score(ctx, ggml_type):
    """Every score -infinity: like nothing seen, out 0 and lse -infinity; the other heads as always."""
    rng = np.random.default_rng(3)
    pool = Pool(rng, ggml_type, 512, 64, 16, 2)
    q, q_pe = queries(rng, 1, 20, 512, 64)
    for at in range(20):
        cols = [c - 512 for c in infinite_row(pool, at // 16, at % 16, 515, 1)]
    q_pe[..., cols] = -np.abs(q_pe[..., cols])
    q_pe[:, 7:9, cols] *= -1
    out, lse = run_attention(ctx, pool, q, q_pe, np.array([[0, 1]]), np.array([20]), 0.07)
    rest = np.r_[0:7, 9:20]
    assert (out[0, rest] == 0).all() and (lse[0, rest] == -np.inf).all()
    assert np.isnan(out[0, 7:9]).all() and np.isnan(lse[0, 7:9]).all()


# ---- sizes of queries -----------------------------------------------------

@pytest.mark.parametrize("ggml_type", [mm.F16, mm.Q8_0])
@pytest.mark.parametrize("size", [1e-30, 1e32, 1e36])
def test_attention_query_sizes(ctx, ggml_type, size):
    """Finite queries of any size, as long as the scores stay in f32's range."""
    rng = np.random.default_rng(2)
    pool = Pool(rng, ggml_type, 512, 64, 16, 8)
    q, q_pe = (np.clip(a, -4, 4) for a in queries(rng, 2, 20, 512, 64))
    q, q_pe = (a * np.float32(size) for a in (q, q_pe))
    scale = float(np.float32(0.07 / size))
    lens, tables = np.array([128, 77]), np.arange(8)[None]
    ids = np.zeros(2, np.int64)
    want = ref.attention64(q, q_pe, pool.values, tables, ids, lens, 16, scale, 512)
    check_attention(*run_attention(ctx, pool, q, q_pe, tables, lens, scale, table_of=ids), *want)


# ---- every kernel ---------------------------------------------------------

@pytest.mark.parametrize("ggml_type", [mm.F16, mm.Q8_0])
@pytest.mark.parametrize("heads", [17, 24, 33, 70])
@pytest.mark.parametrize("rank,pe,pt", [(512, 0, 16), (512, 32, 32), (480, 64, 16), (256, 32, 64), (96, 0, 16), (32, 64, 16)])
def test_attention_sizes_and_heads(ctx, ggml_type, heads, rank, pe, pt):
    """Two product tiles, a packed one, several head tiles, each at ranks and rotary parts that leave waves partly or
    wholly without columns; a table per token, and one table of all (which f16 rows are read otherwise for)."""
    rng = np.random.default_rng(heads + rank + pe)
    lens = np.array([77, 0, 300, 1, 160])
    n_pages = int(((lens + pt - 1) // pt).sum()) + 1
    pool = Pool(rng, ggml_type, rank, pe, pt, n_pages)
    q, q_pe = queries(rng, 5, heads, rank, pe)
    scale = (rank + pe) ** -0.5 * 1.5
    tables = tables_for(rng, lens, pt, n_pages, more=0)
    want = ref.attention64(q, q_pe, pool.values, tables, np.arange(5), lens, pt, scale, rank)
    check_attention(*run_attention(ctx, pool, q, q_pe, tables, lens, scale, pad=3), *want)
    tables, rows = tables[2:3], np.zeros(5, np.int64)
    want = ref.attention64(q, q_pe, pool.values, tables, rows, lens, pt, scale, rank)
    check_attention(*run_attention(ctx, pool, q, q_pe, tables, lens, scale, table_of=rows), *want)


@pytest.mark.parametrize("ggml_type", [mm.F16, mm.Q8_0])
@pytest.mark.parametrize("heads,rank,pe", [(20, 512, 64), (40, 512, 64), (20, 512, 32), (40, 96, 32)])
@pytest.mark.parametrize("n", [65, 300])
def test_attention_many_tokens_and_heads(ctx, ggml_type, heads, rank, pe, n):
    """More tokens than a wave has lanes (and than a workgroup has threads), with a packed tile and with two head tiles."""
    rng = np.random.default_rng(n + heads)
    pt, n_pages = 16, 300
    lens = np.where(rng.random(n) < 0.2, 0, np.exp(rng.uniform(0, np.log(150), n)).astype(np.int64))
    lens[::41] = 700
    pool = Pool(rng, ggml_type, rank, pe, pt, n_pages)
    tables = rng.integers(0, n_pages, (20, 44)).astype(np.int32)
    rows = rng.integers(0, 20, n)
    q, q_pe = queries(rng, n, heads, rank, pe)
    want = ref.attention64(q, q_pe, pool.values, tables, rows, lens, pt, 0.08, rank)
    check_attention(*run_attention(ctx, pool, q, q_pe, tables, lens, 0.08, table_of=rows), *want)


# ---- log probabilities ----------------------------------------------------

def test_logprobs_have_no_side(ctx):
    """One large logit and 32767 about 10.4 below it, which together weigh as much: log probabilities near -0.7, whose
    own rounding is at most u / 2, to either side. Over 512 rows the mean's deviation is below 0.05 u, that of the sums,
    some ten roundings, below 0.1 u; 0.5 u is allowed. An exponent off by 1.3e-8 of its size (log2 e rounded to f32) puts
    all of them 1.1 u too low, a logarithm that is cut off 0.5 u too high."""
    rng = np.random.default_rng(10)
    n, v = 512, 32768
    x = (-10.4 + rng.uniform(-0.5, 0.5, (n, v)) + rng.uniform(-0.2, 0.2, (n, 1))).astype(np.float32)
    x[:, 5] = 0.0
    got = run_logprobs(ctx, x, np.full((n, 1), 5), 0)
    lp, h = ref.logprobs64(x)
    assert (np.abs(got[0][:, 0] - lp[:, 5]) <= 6e-6).all()
    assert abs((got[0][:, 0] - lp[:, 5]).mean()) <= 0.5 * U, (got[0][:, 0] - lp[:, 5]).mean() / U


# ---- two contexts ---------------------------------------------------------

def test_two_contexts_as_each_alone(mm, ctx):
    """Each context's step from its own run, finished before the other begins: the bits of both queued together."""
    from test_gpu_step_ops import Step
    with mm.Context(0) as other, Buffers(ctx) as d, Buffers(other) as e:
        pair = [Step(ctx, d, np.random.default_rng(5), mm.F16, [3000, 17, 900, 1300] * 8),
                Step(other, e, np.random.default_rng(6), mm.Q8_0, [2500, 64, 1, 800] * 8)]
        alone = []
        for i, s in enumerate(pair):
            s.fill(np.random.default_rng(40 + i))
            s.run()
            alone.append(s.results())
        for i, s in enumerate(pair):
            s.fill(np.random.default_rng(40 + i))
        for s in pair:
            s.run()
        for s, want in zip(pair, alone):
            got = s.results()
            for k in got:
                same_bits(got[k], want[k])
            s.rope.free()


# ---- a captured batch of fixed size ---------------------------------------

@pytest.mark.parametrize("ggml_type", [mm.F16, mm.Q8_0])
@pytest.mark.parametrize("n", [5, 70])
def test_captured_batch_with_other_sequences(ctx, ggml_type, n):
    """A captured cache write and attention, replayed with other slots, tables, lengths, positions and padding, the
    program's own calls between the replays: the bits of the calls made one by one, and the formula's values."""
    rng = np.random.default_rng(n)
    pt, pages_each, heads = 16, 40, 20
    n_pages = n * pages_each
    pool = Pool(rng, ggml_type, 512, 64, pt, n_pages)
    rope = mm.Rope(ctx, dims=64, base=1e6)
    with Buffers(ctx) as d:
        sides = []
        for _ in range(2):
            b = dict(pool=d.put(pool.bytes), kv=d.new(n * 576 * 4), slots=d.new(n * 4), pos=d.new(n * 4), lens=d.new(n * 4),
                     tables=d.new(n * pages_each * 4), q=d.new(n * heads * 512 * 4), q_pe=d.new(n * heads * 64 * 4),
                     out=d.new(n * heads * 512 * 4), lse=d.new(n * heads * 4),
                     work=d.new(ctx.mla_attention_workspace(n, heads, 512)))
            cache = mm.KvCache(b["pool"], ggml_type, rank=512, rope_dims=64, page_tokens=pt, n_pages=n_pages)
            args = ctx.mla_attention_args(cache, q=b["q"], q_pe=b["q_pe"], out=b["out"], lse=b["lse"], lens=b["lens"],
                                          tables=b["tables"], n_tables=n, table_pages=pages_each, n_tokens=n,
                                          n_heads=heads, scale=0.07, workspace=b["work"])
            sides.append((b, cache, args))

        def fill(b, seed):
            g = np.random.default_rng(seed)
            lens = np.where(g.random(n) < 0.3, 0, np.exp(g.uniform(0, np.log(pages_each * pt), n))).astype(np.uint32)
            tables = g.permutation(n_pages).reshape(n, pages_each).astype(np.int32)
            last = np.maximum(lens.astype(np.int64) - 1, 0)
            slots = np.where(lens > 0, tables[np.arange(n), last // pt] * pt + last % pt, -1).astype(np.int32)
            x = dict(kv=g.standard_normal((n, 576)), q=g.standard_normal((n, heads, 512)), q_pe=g.standard_normal((n, heads, 64)))
            x = {k: v.astype(np.float32) for k, v in x.items()}
            x.update(slots=slots, pos=last.astype(np.uint32), lens=lens, tables=tables)
            for k, v in x.items():
                mm.check(ctx.lib.mmhip_memcpy_h2d(ctx.handle, b[k].ptr, v.ctypes.data, v.nbytes), "h2d")
            return x

        def run(side):
            b, cache, args = side
            ctx.kv_store_dev(cache, b["kv"], b["slots"], n, rope=rope, positions=b["pos"])
            ctx.mla_attention_dev(args)

        fill(sides[0][0], 0)
        fill(sides[1][0], 0)
        for side in sides:
            run(side)  # the kernels are loaded outside the capture
        ctx.synchronize()
        g = Graph(ctx, lambda: run(sides[0]))
        try:
            for seed in (1, 2, 3):
                x = [fill(b, seed) for b, _, _ in sides][0]
                g.replay()
                run(sides[1])
                ctx.synchronize()
                got = [[b["out"].to_numpy(np.float32, n * heads * 512), b["lse"].to_numpy(np.float32, n * heads),
                        b["pool"].to_numpy(np.uint8, pool.bytes.size)] for b, _, _ in sides]
                for a, c in zip(*got):
                    same_bits(a, c)
                pool.bytes = got[0][2].reshape(pool.bytes.shape).copy()
                revalue(pool)
                want = ref.attention64(x["q"], x["q_pe"], pool.values, x["tables"], np.arange(n), x["lens"], pt, 0.07, 512)
                check_attention(got[0][0].reshape(n, heads, 512), got[0][1].reshape(n, heads), *want)
        finally:
            g.free()
            rope.free()
