"""What stands at a decode step's two ends on the device: embedding rows, the
page plan and sampling, against plain forms (tests/step_ends_reference.py), and
steps whose tokens lead to the next step's without the host.

An embedding value is exact before its scale and rounded once: equal bits. A plan
holds whole numbers: equal. A sampled token and the number of tokens kept are
whole numbers: equal, the weights' sums being good to 2^-44 of the largest weight
per token (2^-26 together for 2^18 tokens), far closer than a random number of 24
bits or a cut comes to a border in these inputs. Its probability is a quotient in
64 bits, rounded once: half a step of f32, 2^-24, and the sums' 2^-26.
"""
import numpy as np
import pytest

import mmhip as mm
import step_ends_reference as ref
from step_reference import At, Buffers, Graph, Pool, U

pytestmark = pytest.mark.gpu

NONE = mm.NO_TOKEN


def put_into(ctx, buf, arr):
    arr = np.ascontiguousarray(arr)
    mm.check(ctx.lib.mmhip_memcpy_h2d(ctx.handle, buf.ptr, arr.ctypes.data, arr.nbytes), "h2d")


# ---- embedding rows -------------------------------------------------------

def table_values(raw, t, rows, cols, orc):
    if t in (mm.Q4_0, mm.IQ4_NL):
        return ref.values_4bit(raw, t).reshape(rows, cols).astype(np.float32)
    if t == mm.F32:
        return raw.view(np.float32).reshape(rows, cols)
    bs, bb = mm.BLOCK_SIZE[t], mm.BLOCK_BYTES[t]
    per = (cols + bs - 1) // bs
    return np.stack([orc.dequantize(r, t, cols) for r in raw.reshape(rows, per * bb)])


@pytest.mark.parametrize("t", [mm.F32, mm.F16, mm.Q8_0, mm.Q4_0, mm.IQ4_NL, mm.IQ2_XXS])
@pytest.mark.parametrize("cols,n", [(1, 1), (32, 3), (37, 5), (256, 1), (768, 70), (2048, 9), (4352, 3)])
def test_embedding_rows(ctx, orc, t, cols, n):
    if cols % mm.BLOCK_SIZE[t] and t not in (mm.F32, mm.F16, mm.Q8_0):
        cols = -(-cols // mm.BLOCK_SIZE[t]) * mm.BLOCK_SIZE[t]
    rng = np.random.default_rng(cols + n)
    rows = 61
    raw = np.asarray(mm.make_weight(rng, t, rows, cols), np.uint8)
    want = table_values(raw, t, rows, cols, orc)
    for pad, off, scale in ((0, 0, 1.0), (3, 1, 45.25483)):
        tokens = rng.integers(0, rows, n).astype(np.uint32)
        tokens[n // 2] = tokens[0]  # the same row twice
        if n > 2:
            tokens[1], tokens[2] = NONE, rows - 1
        ld = cols + pad
        with Buffers(ctx) as d:
            y = d.put(np.full(off + n * ld, 7.0, np.float32))
            shift = 2 if t != mm.F32 else 4  # the table at its type's alignment only
            table = d.put(np.concatenate([np.zeros(shift, np.uint8), raw]))
            ctx.embed_dev(y, At(table, shift), t, rows, cols, d.put(tokens), n, scale=scale, y_stride=ld, y_offset=4 * off)
            ctx.synchronize()
            got = y.to_numpy(np.float32, off + n * ld)
        assert (got[:off] == 7).all()
        got = got[off:].reshape(n, ld)
        expect = np.full((n, ld), 7.0, np.float32)
        live = tokens != NONE
        expect[live, :cols] = want[tokens[live]] * np.float32(scale)
        assert np.array_equal(got, expect)


def test_embedding_tokens_outside_the_table(ctx):
    rng = np.random.default_rng(1)
    raw = mm.make_weight(rng, mm.Q4_0, 10, 64)
    tokens = np.array([3, 10, NONE, 0xFFFFFFFE, 9], np.uint32)
    with Buffers(ctx) as d:
        y = d.put(np.full((5, 64), 7.0, np.float32))
        ctx.embed_dev(y, d.put(raw), mm.Q4_0, 10, 64, d.put(tokens), 5)
        with pytest.raises(mm.MmhipError, match="embed") as e:
            ctx.synchronize()
        assert e.value.code == mm.ERR_INVALID
        ctx.synchronize()  # once
        got = y.to_numpy(np.float32, 320).reshape(5, 64)
    assert np.isnan(got[[1, 3]]).all() and (got[2] == 7).all() and np.isfinite(got[[0, 4]]).all()


def test_embedding_in_a_large_table(ctx):
    """Rows behind 2^32 bytes."""
    rows, cols = 2_200_000, 2048
    rng = np.random.default_rng(2)
    with Buffers(ctx) as d:
        table = mm.DeviceArray(ctx, rows * cols)  # f16 rows, the last ones filled
        d.held.append(table)
        rows //= 2
        last = rng.standard_normal((4, cols)).astype(np.float16)
        put_into(ctx, At(table, (rows - 4) * cols * 2), last)
        y = d.new(4 * cols * 4)
        ctx.embed_dev(y, table, mm.F16, rows, cols, d.put(np.arange(rows - 4, rows, dtype=np.uint32)), 4)
        ctx.synchronize()
        assert np.array_equal(y.to_numpy(np.float32, 4 * cols).reshape(4, cols), last.astype(np.float32))


# ---- page plans -----------------------------------------------------------

class Planner:
    """A plan's buffers; the tables' rows are apart, and guards stand behind every output."""

    GUARD = 5

    def __init__(self, ctx, d, *, n, table_pages, pt, n_pages, max_tokens, release=True, shared=True, last=True, aliased=False,
                 table_gap=3):
        self.ctx, self.n, self.tp, self.gap, self.n_pages, self.max_tokens, self.pt = ctx, n, table_pages, table_gap, n_pages, max_tokens, pt
        u = lambda k: d.new(4 * (k + self.GUARD))  # noqa: E731
        self.b = dict(lens=u(n), new=u(n), release=u(n), shared=u(n), next_lens=u(n), free=u(n_pages), free_count=u(1),
                      next_free=u(1), positions=u(max_tokens), slots=u(max_tokens), table_of=u(max_tokens), seen=u(max_tokens),
                      firsts=u(n + 1), granted=u(n), last=u(n), tables=u(n * (table_pages + table_gap)),
                      work=d.new(ctx.kv_plan_workspace(n)))
        b = self.b
        self.aliased, self.has_last = aliased, last
        if aliased:
            b["next_lens"], b["next_free"] = b["lens"], b["free_count"]
        self.args = ctx.kv_plan_args(
            n_requests=n, lens=b["lens"], new=b["new"], release=b["release"] if release else None,
            shared=b["shared"] if shared else None, next_lens=b["next_lens"], tables=b["tables"], table_pages=table_pages,
            table_stride=table_pages + table_gap, page_tokens=pt, n_pages=n_pages, free=b["free"], free_count=b["free_count"],
            next_free_count=b["next_free"], max_tokens=max_tokens, positions=b["positions"], slots=b["slots"],
            table_of=b["table_of"], seen=b["seen"], firsts=b["firsts"], granted=b["granted"], last=b["last"] if last else None,
            workspace=b["work"])

    def set(self, lens=None, new=None, release=None, shared=None, tables=None, free=None, count=None):
        for k, v in (("lens", lens), ("new", new), ("release", release), ("shared", shared), ("free", free)):
            if v is not None:
                put_into(self.ctx, self.b[k], np.asarray(v).astype(np.int64).astype(np.uint32))
        if count is not None:
            put_into(self.ctx, self.b["free_count"], np.array([count], np.uint32))
        if tables is not None:
            full = np.full((self.n, self.tp + self.gap), -77, np.int32)
            full[:, :self.tp] = tables
            put_into(self.ctx, self.b["tables"], full)

    def get(self):
        size = dict(positions=self.max_tokens, slots=self.max_tokens, table_of=self.max_tokens, seen=self.max_tokens,
                    firsts=self.n + 1, granted=self.n, last=self.n, next_lens=self.n, free=self.n_pages, next_free=1)
        out = {}
        for k, s in size.items():
            v = self.b[k].to_numpy(np.uint32, s + self.GUARD)
            assert (v[s:] == 0xFFFFFFFF).all(), k  # nothing behind an output is written
            out[k] = v[:s].view(np.int32) if k in ("slots", "free") else v[:s]
        t = self.b["tables"].to_numpy(np.int32, self.n * (self.tp + self.gap)).reshape(self.n, self.tp + self.gap)
        assert (t[:, self.tp:] == -77).all()
        out["tables"] = t[:, :self.tp]
        return out

    def check(self, want):
        got = self.get()
        for k, v in want.items():
            if k == "last" and not self.has_last:
                continue
            v = np.asarray(v)
            assert np.array_equal(got[k].astype(np.int64).reshape(v.shape) & 0xFFFFFFFF, v.astype(np.int64) & 0xFFFFFFFF), k


def random_plan(rng, n, pt, longest, spare):
    """Lengths, tables and a stack of free pages that belong together."""
    table_pages = -(-longest // pt) + 3
    lens = np.where(rng.random(n) < 0.2, 0, np.exp(rng.uniform(0, np.log(longest), n))).astype(np.int64)
    held = -(-lens // pt)
    n_pages = int(held.sum()) + spare
    ids = rng.permutation(n_pages)
    tables = np.full((n, table_pages), -5, np.int32)
    at = 0
    for r in range(n):
        tables[r, :held[r]] = ids[at:at + held[r]]
        at += held[r]
    free = np.full(n_pages, -9, np.int32)
    free[:spare] = ids[at:]
    return lens, tables, free, n_pages, table_pages


@pytest.mark.parametrize("n,pt,longest,max_tokens", [(1, 16, 40, 1), (1, 16, 40, 100), (3, 16, 5, 7), (64, 16, 300, 64),
                                                     (70, 64, 1000, 5000), (1000, 16, 60, 900), (1024, 32, 90, 4096),
                                                     (1025, 16, 50, 2000), (3000, 16, 40, 70000), (130, 1024, 5000, 9000)])
@pytest.mark.parametrize("room", ["plenty", "few_pages", "few_tokens"])
def test_plans(ctx, n, pt, longest, max_tokens, room):
    rng = np.random.default_rng(n + pt + len(room))
    lens, tables, free, n_pages, table_pages = random_plan(rng, n, pt, longest, 3 + n // 4 if room == "few_pages" else 4 * n + 70000 // pt)
    new = np.where(rng.random(n) < 0.6, 1, rng.integers(0, 3 * pt, n))
    if room != "few_tokens" and new.sum() > max_tokens:
        new = np.where(np.cumsum(new) <= max_tokens, new, 0)
    release, shared = rng.random(n) < 0.25, rng.integers(0, 3, n)
    new = np.minimum(new, table_pages * pt - np.where(release, 0, lens))  # every table is long enough
    over = room == "few_tokens" and new.sum() > max_tokens
    count = int((free != -9).sum())
    with Buffers(ctx) as d:
        p = Planner(ctx, d, n=n, table_pages=table_pages, pt=pt, n_pages=n_pages, max_tokens=max_tokens)
        p.set(lens, new, release, shared, tables, free, count)
        ctx.kv_plan_dev(p.args)
        if over:
            with pytest.raises(mm.MmhipError, match="max_tokens"):
                ctx.synchronize()
        ctx.synchronize()
        p.check(ref.plan(lens, new, tables, free, count, page_tokens=pt, n_pages=n_pages, max_tokens=max_tokens,
                         release=release, shared=shared))


@pytest.mark.parametrize("release,shared,last", [(False, False, False), (True, False, True)])
def test_plans_without_the_optional_buffers(ctx, release, shared, last):
    rng = np.random.default_rng(1)
    lens, tables, free, n_pages, table_pages = random_plan(rng, 40, 16, 100, 90)
    new, flags = rng.integers(0, 20, 40), rng.random(40) < 0.5
    new = np.minimum(new, table_pages * 16 - lens)
    with Buffers(ctx) as d:
        p = Planner(ctx, d, n=40, table_pages=table_pages, pt=16, n_pages=n_pages, max_tokens=900, release=release, shared=shared,
                    last=last)
        p.set(lens, new, flags, np.zeros(40), tables, free, 90)
        ctx.kv_plan_dev(p.args)
        ctx.synchronize()
        p.check(ref.plan(lens, new, tables, free, 90, page_tokens=16, n_pages=n_pages, max_tokens=900,
                         release=flags if release else None))


def test_plan_of_no_requests_and_no_tokens(ctx):
    with Buffers(ctx) as d:
        p = Planner(ctx, d, n=0, table_pages=4, pt=16, n_pages=9, max_tokens=6, release=False, shared=False, last=False)
        p.set(free=np.arange(9), count=4)
        ctx.kv_plan_dev(p.args)
        ctx.synchronize()
        got = p.get()
        assert got["firsts"].tolist() == [0] and got["next_free"].tolist() == [4] and (got["slots"] == -1).all()
        assert (got["seen"] == 0).all()
        p = Planner(ctx, d, n=2, table_pages=4, pt=16, n_pages=9, max_tokens=0)
        p.set([5, 0], [0, 0], [0, 0], [0, 0], np.zeros((2, 4)), np.arange(9), 4)
        ctx.kv_plan_dev(p.args)
        ctx.synchronize()
        got = p.get()
        assert got["next_lens"].tolist() == [5, 0] and got["granted"].tolist() == [0, 0] and (got["last"] == NONE).all()


@pytest.mark.parametrize("n,max_tokens", [(6, 60), (1500, 9000)])
def test_plans_with_wrong_numbers(ctx, n, max_tokens):
    """Nothing is written out of bounds, the requests that are right get what they should, and the fault is named."""
    pt, tp, n_pages = 16, 4, 20
    base = dict(lens=np.zeros(n), new=np.zeros(n), release=np.zeros(n), shared=np.zeros(n), tables=np.zeros((n, tp)),
                free=np.arange(n_pages), count=n_pages)

    def run(word, **kw):
        a = dict(base, **{k: np.array(v) for k, v in kw.items()})
        for k in ("lens", "new", "release", "shared"):
            a[k] = np.concatenate([a[k], np.zeros(n - len(a[k]))])
        with Buffers(ctx) as d:
            p = Planner(ctx, d, n=n, table_pages=tp, pt=pt, n_pages=n_pages, max_tokens=max_tokens)
            p.set(a["lens"], a["new"], a["release"], a["shared"], a["tables"], a["free"], int(a["count"]))
            ctx.kv_plan_dev(p.args)
            with pytest.raises(mm.MmhipError, match=word):
                ctx.synchronize()
            ctx.synchronize()
            return p.get()

    g = run("length beyond", lens=[60, 0, 64], new=[5, 3, 1])
    assert g["granted"][:3].tolist() == [0, 1, 0] and g["next_lens"][:3].tolist() == [60, 3, 64]
    g = run("length beyond", lens=[0xFFFFFFFF, 0], new=[0xFFFFFFFF, 2])
    assert g["granted"][:2].tolist() == [0, 1] and g["next_lens"][0] == 0xFFFFFFFF
    g = run("length beyond", lens=[500], release=[1], count=3)  # its table has four pages to give back
    assert g["next_free"].tolist() == [7] and g["next_lens"][0] == 0
    g = run("more free pages", count=21, new=[17])
    assert g["next_free"].tolist() == [18] and g["granted"][0] == 1
    g = run("more free pages", lens=[30, 40], release=[1, 1], new=[0, 0, 20], count=17)
    assert g["next_free"].tolist() == [18] and g["granted"][2] == 1
    g = run("page that the pool", free=np.where(np.arange(n_pages) == 19, 20, np.arange(n_pages)), new=[18, 2])
    assert (g["slots"][:16] == -1).all() and g["slots"][16:20].tolist() == [18 * 16, 18 * 16 + 1, 17 * 16, 17 * 16 + 1]
    g = run("page that the pool", lens=[3], new=[2, 1], tables=np.full((n, tp), -1))
    assert g["slots"][:3].tolist() == [-1, -1, 19 * 16]


@pytest.mark.parametrize("n,max_tokens", [(50, 200), (50, 5000)])
def test_plan_goes_on_from_itself(ctx, n, max_tokens):
    """Captured with its lengths and count in place, replayed for many steps: the plans made one after the other."""
    rng = np.random.default_rng(3)
    lens, tables, free, n_pages, table_pages = random_plan(rng, n, 16, 400, 300)
    tables = np.concatenate([tables, np.full((n, 20), -5, np.int32)], 1)
    count = 300
    with Buffers(ctx) as d:
        p = Planner(ctx, d, n=n, table_pages=tables.shape[1], pt=16, n_pages=n_pages, max_tokens=max_tokens, aliased=True)
        p.set(np.zeros(n), np.zeros(n), np.zeros(n), np.zeros(n), tables, free, 0)
        ctx.kv_plan_dev(p.args)  # the kernels are loaded outside the capture
        ctx.synchronize()
        g = Graph(ctx, lambda: ctx.kv_plan_dev(p.args))
        try:
            p.set(lens=lens, tables=tables, free=free, count=count)
            for _ in range(6):
                release = rng.random(n) < 0.1
                new = np.where(rng.random(n) < 0.7, 1, np.where(release, rng.integers(0, 60, n), 0))
                new = np.where(np.cumsum(new) <= max_tokens, new, 0)
                p.set(new=new, release=release)
                g.replay()
                ctx.synchronize()
                want = ref.plan(lens, new, tables, free, count, page_tokens=16, n_pages=n_pages, max_tokens=max_tokens,
                                release=release, shared=np.zeros(n))
                p.check(want)
                lens, tables, free, count = want["next_lens"], want["tables"], want["free"], want["next_free"][0]
                held = np.concatenate([tables[r, :-(-lens[r] // 16)] for r in range(n)] + [free[:count]])
                assert len(np.unique(held)) == len(held)  # no page belongs to two
        finally:
            g.free()


@pytest.mark.parametrize("n,max_tokens", [(17, 40), (17, 5000)])
def test_more_pages_given_back_than_there_are(ctx, n, max_tokens):
    """Lengths of 2^32 - 16 in tables of 2^28 - 1 entries, 2^32 of them together: those that the stack holds come back."""
    pt, tp, n_pages, count = 16, (1 << 28) - 1, 20, 4
    with Buffers(ctx) as d:
        tables = mm.DeviceArray(ctx, n * tp * 4)  # only what comes back is read
        d.held.append(tables)
        put_into(ctx, tables, np.arange(100, 140, dtype=np.int32))
        put_into(ctx, At(tables, (n - 1) * tp * 4), np.arange(200, 210, dtype=np.int32))
        ints = lambda k: d.put(np.zeros(k, np.uint32))  # noqa: E731
        free, next_free = d.put(np.arange(n_pages, dtype=np.int32)), ints(1)
        out = {k: ints(max_tokens) for k in ("positions", "slots", "table_of", "seen")}
        new = np.zeros(n, np.uint32)
        new[n - 1] = 18  # in the row that begins anew: two pages, the two last ones that came back
        release = np.ones(n, np.uint32)
        args = ctx.kv_plan_args(
            n_requests=n, lens=d.put(np.full(n, pt * tp, np.uint32)), new=d.put(new), release=d.put(release), shared=None,
            next_lens=ints(n), tables=tables, table_pages=tp, table_stride=tp, page_tokens=pt, n_pages=n_pages, free=free,
            free_count=d.put(np.array([count], np.uint32)), next_free_count=next_free, max_tokens=max_tokens, firsts=ints(n + 1),
            granted=ints(n), last=None, workspace=d.new(ctx.kv_plan_workspace(n)), **out)
        ctx.kv_plan_dev(args)
        with pytest.raises(mm.MmhipError):  # the pages' numbers are wrong too
            ctx.synchronize()
        ctx.synchronize()
        assert free.to_numpy(np.int32, n_pages).tolist() == [0, 1, 2, 3] + list(range(100, 116))
        assert next_free.to_numpy(np.uint32, 1)[0] == n_pages - 2
        slots = out["slots"].to_numpy(np.int32, max_tokens)
        assert (slots == -1).all()  # pages 115 and 114 are not of the pool


def test_large_plan_in_place(ctx):
    """Lengths and the count of free pages in place, several launches and several sweeps over the requests."""
    rng = np.random.default_rng(4)
    n, max_tokens = 3000, 9000
    lens, tables, free, n_pages, table_pages = random_plan(rng, n, 16, 60, 9000)
    count = 9000
    with Buffers(ctx) as d:
        p = Planner(ctx, d, n=n, table_pages=table_pages, pt=16, n_pages=n_pages, max_tokens=max_tokens, aliased=True)
        p.set(lens=lens, tables=tables, free=free, count=count, shared=np.zeros(n))
        for _ in range(4):
            release = rng.random(n) < 0.2
            new = np.where(rng.random(n) < 0.5, 1, np.where(release, rng.integers(0, 30, n), 0))
            new = np.minimum(new, table_pages * 16 - np.where(release, 0, lens))
            new = np.where(np.cumsum(new) <= max_tokens, new, 0)
            p.set(new=new, release=release)
            ctx.kv_plan_dev(p.args)
            ctx.synchronize()
            want = ref.plan(lens, new, tables, free, count, page_tokens=16, n_pages=n_pages, max_tokens=max_tokens,
                            release=release, shared=np.zeros(n))
            p.check(want)
            lens, tables, free, count = want["next_lens"], want["tables"], want["free"], want["next_free"][0]


# ---- sampling -------------------------------------------------------------

def run_sample(ctx, x, u, t=None, k=None, p=None, least=None, pad=0, off=0, rows=None, n_logits=None, times=1):
    """(tokens, probs, kept) of every output row."""
    n, vocab = len(u), x.shape[1]
    with Buffers(ctx) as d:
        buf = np.full((x.shape[0], vocab + pad), np.inf, np.float32)  # behind a row stands what would be taken
        buf[:, :vocab] = x
        logits = At(d.put(np.concatenate([np.zeros(off, np.float32), buf.ravel()])), 4 * off)
        opt = lambda v, kind: None if v is None else d.put(np.broadcast_to(np.asarray(v, kind), n).copy())  # noqa: E731
        out = [d.put(np.full(n + 3, 7, kind)) for kind in (np.uint32, np.float32, np.uint32)]
        args = ctx.sample_args(logits=logits, n_rows=n, vocab=vocab, stride=vocab + pad, uniform=d.put(np.asarray(u, np.float32)),
                               tokens=out[0], probs=out[1], kept=out[2], temperature=opt(t, np.float32), top_k=opt(k, np.uint32),
                               top_p=opt(p, np.float32), min_p=opt(least, np.float32), rows=opt(rows, np.uint32),
                               n_logits=n_logits or 0, workspace=d.new(max(16, ctx.sample_workspace(n, vocab))))
        for _ in range(times):
            ctx.sample_dev(args)
        try:
            ctx.synchronize()
        finally:
            got = [b.to_numpy(kind, n + 3) for b, kind in zip(out, (np.uint32, np.float32, np.uint32))]
            assert all((g[n:] == 7).all() for g in got)
            run_sample.got = [g[:n] for g in got]  # for calls that end in a report
    return run_sample.got


def check_sample(got, x, u, t=1.0, k=0, p=1.0, least=0.0, rows=None):
    n = len(u)
    full = lambda v, kind: np.broadcast_to(np.asarray(v, kind), n)  # noqa: E731
    t, k, p, least, u = full(t, np.float32), full(k, np.uint32), full(p, np.float32), full(least, np.float32), full(u, np.float32)
    for r in range(n):
        want = ref.sample(x[r if rows is None else rows[r]], float(t[r]), int(k[r]), float(p[r]), float(least[r]), float(u[r]))
        assert (got[0][r], got[2][r]) == (want[0], want[2]), (r, [g[r] for g in got], want)
        assert abs(got[1][r] - want[1]) <= (U + 2.0 ** -26) * want[1] + 1e-45


def logits_like(rng, n, vocab, spread=2.0):
    """Few likely tokens above a broad rest."""
    x = (spread * rng.standard_normal((n, vocab))).astype(np.float32)
    for r in range(n):
        at = rng.integers(0, vocab, min(vocab, 12))
        x[r, at] = rng.uniform(4, 16) + 1.5 * rng.standard_normal(len(at))
    return x


SETTINGS = [dict(), dict(t=0.7), dict(t=0.0), dict(t=1.5, k=1), dict(k=2), dict(k=40), dict(t=0.8, k=300), dict(p=0.0), dict(p=0.5),
            dict(t=0.9, p=0.95), dict(t=1.7, p=0.999), dict(least=0.05), dict(least=1.0), dict(t=2.0, least=1e-6),
            dict(t=0.9, k=50, p=0.9), dict(t=1.2, k=1000, p=0.98, least=0.01), dict(k=0xFFFFFFFF, p=2.0)]


@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 65, 1000, 4096, 4097, 16384, 40000, 154880])
@pytest.mark.parametrize("settings", SETTINGS, ids=str)
def test_sampled_tokens(ctx, vocab, settings):
    rng = np.random.default_rng(vocab)
    n = 3 if vocab > 50000 else 5
    x, u = logits_like(rng, n, vocab), rng.random(n).astype(np.float32)
    u[0] = 0.0
    u[1] = np.float32(1 - 2.0 ** -24)
    check_sample(run_sample(ctx, x, u, **settings), x, u, **settings)


@pytest.mark.parametrize("vocab", [777, 33001])
def test_sampling_settings_by_row_with_strides(ctx, vocab):
    rng = np.random.default_rng(vocab)
    n = 70
    x, u = logits_like(rng, n, vocab), rng.random(n).astype(np.float32)
    x[:, rng.random(vocab) < 0.5] = -np.inf
    x[:, 3] = 1.0
    kw = dict(t=rng.choice([0, 0.3, 1, 1.4], n).astype(np.float32), k=rng.choice([0, 1, 7, 90], n), p=rng.choice([1, 0.3, 0.9], n).astype(np.float32),
              least=rng.choice([0, 0.02, 0.5], n).astype(np.float32))
    a = run_sample(ctx, x, u, pad=5, off=1, **kw)
    check_sample(a, x, u, **kw)
    for g, h in zip(a, run_sample(ctx, x, u, times=3, **kw)):  # other alignment, called again: the same bits
        assert np.array_equal(g.view(np.uint32), h.view(np.uint32))


@pytest.mark.parametrize("vocab", [5, 3000, 70000])
@pytest.mark.parametrize("settings", [dict(), dict(k=3), dict(p=0.5), dict(k=1000, p=0.25), dict(least=1.0)], ids=str)
def test_equal_logits(ctx, vocab, settings):
    """Ties go to the lower id, at a cut that falls among them too; equal to -0."""
    rng = np.random.default_rng(vocab)
    x = np.zeros((4, vocab), np.float32)
    x[1] = rng.choice([-0.0, 0.0], vocab)
    x[2] = rng.choice([1.0, 1.0, -3.0], vocab)
    x[3, vocab // 2:] = -np.inf
    u = np.array([0.3, 0.7, 0.49, 0.99], np.float32)
    check_sample(run_sample(ctx, x, u, **settings), x, u, **settings)


@pytest.mark.parametrize("vocab", [100, 20000])
@pytest.mark.parametrize("settings", [dict(), dict(t=0.5, k=30), dict(p=0.9), dict(t=1e-30), dict(t=3e38, p=0.9), dict(t=1e-3, k=50, p=0.99)], ids=str)
def test_extreme_logits_and_temperatures(ctx, vocab, settings):
    rng = np.random.default_rng(1)
    x = rng.standard_normal((6, vocab)).astype(np.float32)
    x[0] *= 1e30
    x[1] *= 1e-30
    x[2, ::3] = -3.4e38
    x[3, 5] = 3.4e38
    x[4, 1:] = -np.inf
    x[5, [3, 8, 50]] = np.inf
    u = rng.random(6).astype(np.float32)
    got = run_sample(ctx, x, u, **settings)
    check_sample(got, x, u, **settings)


@pytest.mark.parametrize("vocab", [50, 9000])
def test_nan_and_empty_rows(ctx, vocab):
    rng = np.random.default_rng(2)
    x = logits_like(rng, 4, vocab)
    x[0, ::2] = np.nan
    x[1] = np.nan
    x[2] = -np.inf
    x[3, 0] = np.nan
    u = np.full(4, 0.6, np.float32)
    for settings in (dict(), dict(k=5, p=0.8), dict(t=0.0)):
        with pytest.raises(mm.MmhipError, match="without a token"):
            run_sample(ctx, x, u, **settings)
        got = run_sample.got
        clean = np.where(np.isnan(x), -np.inf, x)
        check_sample([g[[0, 3]] for g in got], clean[[0, 3]], u[:2], **settings)
        assert (got[0][1:3] == NONE).all() and np.isnan(got[1][1:3]).all() and (got[2][1:3] == 0).all()


@pytest.mark.parametrize("vocab", [70, 20001])
@pytest.mark.parametrize("settings", [dict(), dict(t=0.0), dict(k=9), dict(t=1.3, p=0.9, least=0.001)], ids=str)
def test_every_kind_of_nan(ctx, vocab, settings):
    """Quiet and signalling ones of both signs, beside ordinary logits, infinities and zeros of both signs."""
    rng = np.random.default_rng(vocab)
    x = logits_like(rng, 6, vocab)
    x[3] = -np.abs(x[3])
    x[4] = np.abs(x[4]) + 1
    x[5] = np.where(rng.random(vocab) < 0.5, np.float32(-0.0), np.float32(0.0))
    bits = x.view(np.uint32)
    for i, nan in enumerate((0x7FC00000, 0xFFC00000, 0x7F800001, 0xFF800001, 0xFFFFFFFF, 0xFF800000)):
        bits[:, i * 9::64] = nan
    x[2, 33] = np.inf
    u = rng.random(6).astype(np.float32)
    got = run_sample(ctx, x, u, **settings)
    check_sample(got, np.where(np.isnan(x), np.float32(-np.inf), x), u, **settings)


@pytest.mark.parametrize("settings", [dict(t=0.8), dict(k=40), dict(t=0.9, k=300, p=0.95), dict(p=0.9, least=0.01)], ids=str)
def test_pieces_of_several_turns(ctx, settings):
    rng = np.random.default_rng(8)
    x, u = logits_like(rng, 600, 20000), rng.random(600).astype(np.float32)
    check_sample(run_sample(ctx, x, u, **settings), x, u, **settings)


@pytest.mark.parametrize("big,size", [(1e9, 1e-31), (3e38, 1e30), (-1e30, 1e-3), (1e30, 1.0), (65504.0, 0.01)])
@pytest.mark.parametrize("settings", [dict(), dict(k=6), dict(p=0.7), dict(k=30, p=0.9, least=1e-3)], ids=str)
def test_logits_far_from_zero(ctx, big, size, settings):
    """All logits about `big`, a temperature of `size`: nothing of them is lost in their differences from the largest."""
    rng = np.random.default_rng(11)
    x = np.full((3, 9000), np.float32(big))
    for _ in range(5):
        x = np.where(rng.random(x.shape) < 0.4, np.nextafter(x, np.float32(-np.inf)), x)
    u = rng.random(3).astype(np.float32)
    check_sample(run_sample(ctx, x, u, t=size, **settings), x, u, t=size, **settings)


def test_settings_out_of_range(ctx):
    x = np.zeros((1, 100), np.float32)
    ok = np.float32(0.5)
    for kw in (dict(t=-1.0), dict(t=np.nan), dict(t=np.inf), dict(p=-0.1), dict(p=np.nan), dict(least=-0.1), dict(least=1.1),
               dict(least=np.nan)):
        with pytest.raises(mm.MmhipError, match="out of range"):
            run_sample(ctx, x, [ok], **kw)
        assert run_sample.got[0][0] == NONE and np.isnan(run_sample.got[1][0]) and run_sample.got[2][0] == 0
    for u in (1.0, -0.5, np.nan, np.inf):
        with pytest.raises(mm.MmhipError, match="out of range"):
            run_sample(ctx, x, [u])


@pytest.mark.parametrize("vocab", [300, 30000])
def test_chosen_rows(ctx, vocab):
    """Rows by number, one twice, one left out, one that is not there."""
    rng = np.random.default_rng(3)
    x, u = logits_like(rng, 4, vocab), rng.random(5).astype(np.float32)
    rows = np.array([2, NONE, 2, 4, 0], np.uint32)
    with pytest.raises(mm.MmhipError, match="row that the logits"):
        run_sample(ctx, x, u, t=0.9, p=0.9, rows=rows, n_logits=4)
    got = run_sample.got
    assert got[0][1] == 7 and got[1][1] == 7 and got[2][1] == 7  # left as it was
    assert got[0][3] == NONE and np.isnan(got[1][3])
    keep = [0, 2, 4]
    check_sample([g[keep] for g in got], x, u[keep], t=0.9, p=0.9, rows=rows[keep])


@pytest.mark.parametrize("n,vocab", [(1, 3_000_000), (3, 1_100_000), (700, 2500)])
@pytest.mark.parametrize("settings", [dict(t=0.7), dict(t=0.8, k=100), dict(p=0.9), dict(t=0.2, k=40, p=0.99, least=1e-4)], ids=str)
def test_wide_and_many_rows(ctx, n, vocab, settings):
    """Several chunks to a thread of the last launch; pieces of one chunk and of many."""
    rng = np.random.default_rng(n)
    x, u = logits_like(rng, n, vocab), rng.random(n).astype(np.float32)
    check_sample(run_sample(ctx, x, u, **settings), x, u, **settings)


@pytest.mark.parametrize("spread", [0.0, 1e-6, 0.03, 30.0])
@pytest.mark.parametrize("settings", [dict(k=7), dict(k=20000), dict(p=0.5), dict(t=2.0, k=30000, p=0.7, least=0.4)], ids=str)
def test_cuts_among_many_tokens(ctx, spread, settings):
    """Logits so close or so far apart that a bin of the histogram holds more tokens than the list, or nearly none; with
    one at the type's lowest value, as masks leave it."""
    rng = np.random.default_rng(8)
    x = (spread * rng.standard_normal((3, 40000))).astype(np.float32)
    x[1, 77] = np.finfo(np.float32).min
    x[2, 500:] = np.round(x[2, 500:], 2)
    u = rng.random(3).astype(np.float32)
    check_sample(run_sample(ctx, x, u, **settings), x, u, **settings)


def test_frequencies_of_drawn_tokens(ctx):
    """Even steps of u over a row: each token is drawn as often as its probability says, to one draw."""
    rng = np.random.default_rng(4)
    x = np.repeat(rng.standard_normal((1, 40)).astype(np.float32) * 2, 4096, 0)
    u = (np.arange(4096) / 4096).astype(np.float32)
    got = run_sample(ctx, x, u, t=0.8, k=20)
    w = np.exp(x[0].astype(np.float64) / np.float64(np.float32(0.8)))
    w[np.argsort(-w, kind="stable")[20:]] = 0
    drawn = np.bincount(got[0], minlength=40)
    assert (np.abs(drawn - 4096 * w / w.sum()) <= 1.0).all()


def test_captured_sampling(ctx):
    rng = np.random.default_rng(5)
    n, vocab = 9, 20000
    with Buffers(ctx) as d:
        logits, u, t = d.new(n * vocab * 4), d.new(n * 4), d.new(n * 4)
        k, p = d.new(n * 4), d.new(n * 4)
        tok = d.new(n * 4)
        args = ctx.sample_args(logits=logits, n_rows=n, vocab=vocab, uniform=u, tokens=tok, temperature=t, top_k=k, top_p=p,
                               workspace=d.new(max(16, ctx.sample_workspace(n, vocab))))

        def fill():
            a = dict(x=logits_like(rng, n, vocab), u=rng.random(n).astype(np.float32),
                     t=rng.choice([0, 0.7, 1.1], n).astype(np.float32), k=rng.choice([0, 20, 500], n).astype(np.uint32),
                     p=rng.choice([1, 0.9], n).astype(np.float32))
            for b, v in zip((logits, u, t, k, p), a.values()):
                put_into(ctx, b, v)
            return a
        fill()
        ctx.sample_dev(args)  # the kernels are loaded outside the capture
        ctx.synchronize()
        g = Graph(ctx, lambda: ctx.sample_dev(args))
        try:
            for _ in range(4):
                a = fill()
                g.replay()
                ctx.synchronize()
                got = tok.to_numpy(np.uint32, n)
                for r in range(n):
                    assert got[r] == ref.sample(a["x"][r], float(a["t"][r]), int(a["k"][r]), float(a["p"][r]), 0.0, float(a["u"][r]))[0]
                ctx.sample_dev(args)  # the program's own call between replays
                ctx.synchronize()
                assert np.array_equal(tok.to_numpy(np.uint32, n), got)
        finally:
            g.free()


# ---- together -------------------------------------------------------------

class Loop:
    """A toy decoder of one layer whose steps need no host: embedding, plan, cache write, attention over the cache, a 4-bit
    output projection, sampling; the drawn tokens are the next step's."""

    def __init__(self, ctx, d, rng, lens, vocab=512, heads=4):
        self.ctx, self.n, self.vocab, self.heads = ctx, len(lens), vocab, heads
        n, pt, width, hid = self.n, 16, 576, heads * 512
        self.tp, self.n_pages = 12, 12 * n
        held = -(-np.array(lens) // pt)
        self.pool = Pool(rng, mm.F16, 512, 64, pt, self.n_pages)
        tables, ids, at = np.zeros((n, self.tp), np.int32), rng.permutation(self.n_pages), 0
        for r in range(n):
            tables[r, :held[r]] = ids[at:at + held[r]]
            at += held[r]
        free = np.zeros(self.n_pages, np.int32)
        free[:self.n_pages - at] = ids[at:]
        self.start = dict(lens=np.array(lens, np.uint32), tables=tables, free=free, count=np.array([self.n_pages - at], np.uint32),
                          tokens=rng.integers(0, vocab, n).astype(np.uint32), pool=self.pool.bytes)
        self.table_q = mm.make_weight(rng, mm.IQ4_NL, vocab, hid)
        self.table_kv = mm.make_weight(rng, mm.Q4_0, vocab, width)
        self.w_raw = mm.make_weight(rng, mm.Q4_0, vocab, hid)
        self.w = ctx.upload(self.w_raw, mm.Q4_0, vocab, hid)
        b = {k: d.put(v) for k, v in self.start.items()}
        for k, size in dict(new=n, positions=n, slots=n, table_of=n, seen=n, firsts=n + 1, granted=n, last=n, q=n * hid,
                            q_pe=n * heads * 64, kv=n * width, out=n * hid, logits=n * vocab, u=n, t=n, p=n).items():
            b[k] = d.new(4 * size)
        b["tq"], b["tkv"] = d.put(self.table_q), d.put(self.table_kv)
        self.b = b
        self.q_pe = rng.standard_normal((n, heads, 64)).astype(np.float32)
        put_into(ctx, b["new"], np.ones(n, np.uint32))
        put_into(ctx, b["q_pe"], self.q_pe)
        put_into(ctx, b["t"], np.full(n, 0.9, np.float32))
        put_into(ctx, b["p"], np.full(n, 0.95, np.float32))
        self.cache = mm.KvCache(b["pool"], mm.F16, rank=512, rope_dims=64, page_tokens=pt, n_pages=self.n_pages)
        self.plan = ctx.kv_plan_args(
            n_requests=n, lens=b["lens"], new=b["new"], next_lens=b["lens"], tables=b["tables"], table_pages=self.tp, page_tokens=pt,
            n_pages=self.n_pages, free=b["free"], free_count=b["count"], next_free_count=b["count"], max_tokens=n,
            positions=b["positions"], slots=b["slots"], table_of=b["table_of"], seen=b["seen"], firsts=b["firsts"],
            granted=b["granted"], last=b["last"], workspace=d.new(ctx.kv_plan_workspace(n)))
        self.attn = ctx.mla_attention_args(
            self.cache, q=b["q"], q_pe=b["q_pe"], out=b["out"], lens=b["seen"], tables=b["tables"], n_tables=n,
            table_pages=self.tp, table_of=b["table_of"], n_tokens=n, n_heads=heads, scale=0.05,
            workspace=d.new(ctx.mla_attention_workspace(n, heads, 512)))
        self.draw = ctx.sample_args(
            logits=b["logits"], n_rows=n, vocab=vocab, rows=b["last"], n_logits=n, uniform=b["u"], tokens=b["tokens"],
            temperature=b["t"], top_p=b["p"], workspace=d.new(max(16, ctx.sample_workspace(n, vocab))))

    def reset(self):
        for k, v in self.start.items():
            put_into(self.ctx, self.b[k], v)

    def run(self):
        c, b, n = self.ctx, self.b, self.n
        c.kv_plan_dev(self.plan)
        c.embed_dev(b["q"], b["tq"], mm.IQ4_NL, self.vocab, self.heads * 512, b["tokens"], n, scale=30.0)
        c.embed_dev(b["kv"], b["tkv"], mm.Q4_0, self.vocab, 576, b["tokens"], n, scale=30.0)
        c.kv_store_dev(self.cache, b["kv"], b["slots"], n)
        c.mla_attention_dev(self.attn)
        c.qmm_dev(self.w, 0, b["out"], b["logits"], n)
        c.sample_dev(self.draw)

    def steps(self, count, seed, call):
        rng, out = np.random.default_rng(seed), []
        self.reset()
        for _ in range(count):
            put_into(self.ctx, self.b["u"], rng.random(self.n).astype(np.float32))
            call()
            self.ctx.synchronize()
            out.append((self.b["tokens"].to_numpy(np.uint32, self.n), self.b["logits"].to_numpy(np.float32, self.n * self.vocab),
                        self.b["tables"].to_numpy(np.int32, self.n * self.tp), self.b["lens"].to_numpy(np.uint32, self.n)))
        return out


@pytest.mark.parametrize("n", [1, 3, 9])
def test_steps_without_the_host(ctx, n):
    """Twenty steps: called one by one, and captured and replayed. The same bits; and the first steps in 64 bits."""
    import step_reference as sref
    rng = np.random.default_rng(n)
    with Buffers(ctx) as d:
        loop = Loop(ctx, d, rng, rng.integers(1, 150, n))
        eager = loop.steps(20, 1, loop.run)
        loop.reset()
        g = Graph(ctx, loop.run)
        try:
            replayed = loop.steps(20, 1, g.replay)
        finally:
            g.free()
        for a, b in zip(eager, replayed):
            for v, w in zip(a, b):
                assert np.array_equal(v.view(np.uint32), w.view(np.uint32))
        # in 64 bits
        hid, s = loop.heads * 512, loop.start
        lens, tables, free, count = s["lens"].astype(np.int64), s["tables"], s["free"], int(s["count"][0])
        tokens, values = s["tokens"], loop.pool.values.copy()
        tq = ref.values_4bit(loop.table_q, mm.IQ4_NL).reshape(loop.vocab, hid)
        tkv = ref.values_4bit(loop.table_kv, mm.Q4_0).reshape(loop.vocab, 576)
        w = ref.values_4bit(loop.w_raw, mm.Q4_0).reshape(loop.vocab, hid)
        for step in range(4):
            p = ref.plan(lens, np.ones(n), tables, free, count, page_tokens=16, n_pages=loop.n_pages, max_tokens=n)
            lens, tables, free, count = np.array(p["next_lens"]), p["tables"], p["free"], p["next_free"][0]
            q = (tq[tokens] * 30).astype(np.float32).reshape(n, loop.heads, 512)
            for t, slot in enumerate(p["slots"]):
                values[slot // 16, slot % 16] = (tkv[tokens[t]] * 30).astype(np.float32).astype(np.float16)
            out, _ = sref.attention64(q, loop.q_pe, values, tables, np.array(p["table_of"]), np.array(p["seen"]), 16, 0.05, 512)
            logits = out.reshape(n, hid) @ w.T
            got = replayed[step]
            assert np.array_equal(got[2].reshape(n, -1), tables) and np.array_equal(got[3], lens)
            err = np.abs(got[1].reshape(n, -1) - logits).max() / np.abs(logits).max()
            assert err <= 1e-4  # the attention's 1e-5 of its output's norm, in sums of 2048 products
            tokens = got[0]
            u = np.random.default_rng(1)
            for _ in range(step + 1):
                drawn = u.random(n).astype(np.float32)
            for r in range(n):
                assert tokens[r] == ref.sample(got[1].reshape(n, -1)[r], float(np.float32(0.9)), 0, float(np.float32(0.95)), 0.0,
                                               float(drawn[r]))[0]
        loop.w.free()


def test_two_contexts_at_once(mm, ctx):
    """Two contexts' steps queued together: each as alone."""
    with mm.Context(0) as other, Buffers(ctx) as d, Buffers(other) as e:
        pair = [Loop(ctx, d, np.random.default_rng(5), [40, 100, 7, 150, 16]), Loop(other, e, np.random.default_rng(6), [3, 31, 120])]
        alone = []
        for s in pair:
            alone.append(s.steps(1, 9, s.run)[0])
        for s in pair:
            s.reset()
            put_into(s.ctx, s.b["u"], np.random.default_rng(9).random(s.n).astype(np.float32))
        for s in pair:
            s.run()
        for s, want in zip(pair, alone):
            s.ctx.synchronize()
            assert np.array_equal(s.b["tokens"].to_numpy(np.uint32, s.n), want[0])
            assert np.array_equal(s.b["logits"].to_numpy(np.float32, s.n * s.vocab), want[1])
            s.w.free()
