"""The operators of a decode step that stand between its matrix products, as
measurable cases: the root-mean-square norm with the residual's addition, rotary
positions, the paged latent key-value cache's writer, the attention of single
tokens over that cache, and log probabilities of the next token.

Each case runs in one of two forms: elementary torch operations, or (where `own`
is true) the calls a program makes of the Python binding. The shapes are those
of the benchmark and the tests: hidden 2048, latent projections of 768 and 512,
20 heads of 128 + 64 values, cached positions of 512 + 64 values in pages of 16
positions, a vocabulary of 154,880.
"""
import math
import os
import sys

import torch

own = False

EPS = 1e-5
BASE = 1e6
F16, Q8, F32 = "f16", "q8_0", "f32"
RANK, PE, HEADS, HEAD_DIM = 512, 64, 20, 192
SCALE = HEAD_DIM ** -0.5


def listed():
    return [
        # The norm before a layer's attention, one token being decoded: the
        # smallest call there is.
        dict(name="norm_decode", kind="norm", rows=1, cols=2048, residual=True, out=F32),
        # The same for a prompt, its result in blocks of 8 bits.
        dict(name="norm_prompt_q8", kind="norm", rows=4099, cols=2048, residual=True, out=Q8),
        # Rotary positions of the last 64 of each head's 192 values, for one
        # token, and for a prompt far into a context that is longer than the
        # one the model was trained on.
        dict(name="rope_decode", kind="rope", tokens=1, heads=HEADS, layout="interleaved", scaling="none", far=5000),
        dict(name="rope_prompt_yarn", kind="rope", tokens=4096, heads=HEADS, layout="half", scaling="yarn", far=120000),
        # What a layer caches: one position for each of 64 conversations, and a
        # prompt's positions.
        dict(name="store_decode_f16", kind="store", cache=F16, tokens=64, pages=4096, layout="interleaved"),
        dict(name="store_prompt_q8", kind="store", cache=Q8, tokens=4096, pages=512, layout="interleaved"),
        # Attention of one token of one short conversation, of one at the end
        # of a very long one, of a batch of conversations of all lengths, and
        # of a prompt's chunk over the context before it.
        dict(name="attn_short_q8", kind="attn", cache=Q8, tokens=1, heads=HEADS, longest=333, lens="same"),
        dict(name="attn_long_f16", kind="attn", cache=F16, tokens=1, heads=HEADS, longest=131072, lens="same"),
        dict(name="attn_batch_q8", kind="attn", cache=Q8, tokens=64, heads=HEADS, longest=16384, lens="ragged"),
        dict(name="attn_chunk_f16", kind="attn", cache=F16, tokens=256, heads=HEADS, longest=4096, lens="chunk"),
        # Log probabilities of a sampled token with its alternatives, and of a
        # prompt's tokens, some of the vocabulary masked.
        dict(name="logprobs_one", kind="logprobs", rows=1, vocab=154880, given=1, top=20, masked=False),
        dict(name="logprobs_prompt", kind="logprobs", rows=64, vocab=154880, given=1, top=5, masked=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "rope", "store", "attn", "attn", "attn", "logprobs", "logprobs"])
    if kind == "norm":
        return dict(kind=kind, rows=_log(rng, 1, 4099), cols=rng.choice([512, 768, 2048, rng.randint(33, 2048)]),
                    residual=rng.random() < 0.6, out=rng.choice([F32, F16, Q8]))
    if kind == "rope":
        return dict(kind=kind, tokens=_log(rng, 1, 4096), heads=rng.randint(1, HEADS),
                    layout=rng.choice(["interleaved", "half"]), scaling=rng.choice(["none", "linear", "yarn"]),
                    far=_log(rng, 10, 1000000))
    if kind == "store":
        tokens = _log(rng, 1, 4096)
        return dict(kind=kind, cache=rng.choice([F16, Q8]), tokens=tokens,
                    pages=(tokens + 15) // 16 + rng.randint(1, 256), layout=rng.choice(["interleaved", "half"]))
    if kind == "attn":
        lens = rng.choice(["same", "ragged", "ragged", "chunk"])
        longest = _log(rng, 1, 131072 if lens == "same" else 16384)
        most = max(1, min(256, (1 << 20) // longest))
        tokens = 1 if lens == "same" else _log(rng, 1, min(most, longest) if lens == "chunk" else most)
        return dict(kind=kind, cache=rng.choice([F16, Q8]), tokens=tokens,
                    heads=rng.choice([HEADS, HEADS, rng.randint(1, 40)]) if tokens < 16 else HEADS,
                    longest=longest, lens=lens)
    return dict(kind=kind, rows=_log(rng, 1, 64), vocab=rng.choice([154880, _log(rng, 1000, 154880)]),
                given=rng.randint(1, 4), top=rng.choice([0, 1, 5, rng.randint(2, 32)]), masked=rng.random() < 0.3)


# ---- inputs ---------------------------------------------------------------

class _State:
    """What a program has in hand before a call, and what it keeps between calls."""

    def __init__(self, case):
        self.case, self.args = dict(case), None


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _lens(c, g):
    n, longest = c["tokens"], c["longest"]
    if c["lens"] == "same":
        return torch.full((n,), longest, dtype=torch.int32, device="cuda")
    if c["lens"] == "chunk":  # the last n positions of one context
        return torch.arange(longest - n + 1, longest + 1, dtype=torch.int32, device="cuda")
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    u[0] = 1.0
    return torch.exp(u * math.log(longest)).round().clamp(1, longest).int()


def _pool(c, g, n_pages):
    """Pages of 16 positions as the cache holds them: rows of 512 + 64 values in
    16 bits, or per page 16 rows of codes and then 16 rows of block scales."""
    width = RANK + PE
    rows = _randn(g, n_pages * 16, width)
    if c["cache"] == F16:
        return rows.half().view(n_pages, 16 * width).view(torch.uint8)
    codes, scales = _quantised(rows)
    return torch.cat([codes.view(n_pages, 16 * width).view(torch.uint8),
                      scales.contiguous().view(n_pages, 16 * (width // 32)).view(torch.uint8)], 1).contiguous()


def _pages_seen(c):
    return (c["longest"] + 15) // 16


def prepare(case, seed):
    c, s, g, kind = case, _State(case), _gen(seed), case["kind"]
    if kind == "norm":
        n, d = c["rows"], c["cols"]
        s.x, s.weight = _randn(g, n, d), 1 + 0.2 * _randn(g, d)
        s.residual = 3 * _randn(g, n, d) if c["residual"] else None
        s.sum = torch.zeros(n, d, device="cuda") if c["residual"] else None
        if c["out"] == Q8:
            s.y = torch.zeros(n, (d + 31) // 32, 34, dtype=torch.uint8, device="cuda")
            s.outputs = [s.y[..., 2:].view(torch.int8), s.y[..., :2].view(torch.float16)[..., 0]]
        else:
            s.y = torch.zeros(n, d, device="cuda", dtype=torch.float16 if c["out"] == F16 else torch.float32)
            s.outputs = [s.y]
        s.outputs += [s.sum] if c["residual"] else []
    elif kind == "rope":
        n = c["tokens"]
        s.x = _randn(g, n, c["heads"], HEAD_DIM)
        start = int(torch.randint(0, c["far"], (1,), generator=g, device="cuda"))
        s.positions = torch.arange(start, start + n, dtype=torch.int32, device="cuda")
        s.y = torch.zeros_like(s.x)
    elif kind == "store":
        n = c["tokens"]
        s.kv, s.weight = 2 * _randn(g, n, RANK + PE), 1 + 0.2 * _randn(g, RANK)
        s.positions = torch.randint(0, 131072, (n,), generator=g, device="cuda", dtype=torch.int32)
        s.slots = torch.randperm(16 * c["pages"], generator=g, device="cuda")[:n].int()
        if n > 1:
            s.slots[n // 2] = -1  # a padded token of the batch
        s.pool = _pool(c, g, c["pages"])
        s.outputs = _pool_views(c, s.pool)
    elif kind == "attn":
        n, h, p = c["tokens"], c["heads"], _pages_seen(c)
        n_tables = 1 if c["lens"] == "chunk" else n
        s.lens = _lens(c, g)
        # Each table names the pages it needs, in no order; behind them it is 0.
        need = (s.lens.long() + 15) // 16 if n_tables == n else torch.full((1,), p, device="cuda")
        end = torch.cumsum(need, 0)
        n_pages = int(end[-1])
        at = (end - need)[:, None] + torch.arange(p, device="cuda")
        ids = torch.randperm(n_pages, generator=g, device="cuda").int()
        s.tables = torch.where(torch.arange(p, device="cuda") < need[:, None], ids[at.clamp(max=n_pages - 1)],
                               torch.zeros((), dtype=torch.int32, device="cuda")).contiguous()
        s.table_of = torch.zeros(n, dtype=torch.int32, device="cuda") if n_tables < n else None
        s.pool = _pool(c, g, n_pages)
        s.q, s.q_pe = _randn(g, n, h, RANK), _randn(g, n, h, PE)
        s.out, s.lse = torch.zeros(n, h, RANK, device="cuda"), torch.zeros(n, h, device="cuda")
    else:
        n, v = c["rows"], c["vocab"]
        s.logits = 2.5 * _randn(g, n, v)
        peak = torch.randint(0, v, (n, 8), generator=g, device="cuda")
        s.logits.scatter_add_(1, peak, 6 + 4 * torch.rand(n, 8, generator=g, device="cuda"))
        if c["masked"]:
            s.logits[:, torch.rand(v, generator=g, device="cuda") < 0.7] = -math.inf
            s.logits[:, 0] = 0.5
        pick = torch.randint(0, v, (n, c["given"]), generator=g, device="cuda")
        pick[:, 0] = s.logits.argmax(1)
        s.tokens = pick.int()
        s.logp, s.entropy = torch.zeros(n, c["given"], device="cuda"), torch.zeros(n, device="cuda")
        s.top_ids = torch.zeros(n, c["top"], dtype=torch.int32, device="cuda")
        s.top_logp = torch.zeros(n, c["top"], device="cuda")
    torch.cuda.synchronize()  # the library works on a stream of its own
    return s


# ---- the plain form -------------------------------------------------------

def _quantised(x):
    """Blocks of 32 along the last axis: codes, and scales in 16 bits. The block's
    codes are taken with the scale before it is rounded."""
    n, d = x.shape
    nb = (d + 31) // 32
    x = torch.nn.functional.pad(x, (0, nb * 32 - d)).view(n, nb, 32)
    peak = x.abs().amax(-1)
    scale = peak / torch.full_like(peak, 127.0)
    q = x / scale[..., None]
    q = torch.where(scale[..., None] > 0, torch.sign(q) * torch.floor(q.abs() + 0.5), torch.zeros_like(q))
    return q.clamp(-127, 127).to(torch.int8), scale.half()


def _rms(x, weight):
    """The mean and the root in 64 bits, the products in 32."""
    r = torch.rsqrt(x.double().square().mean(-1, keepdim=True) + EPS).float()
    return x * r * weight


def _frequencies(scaling):
    i = torch.arange(PE // 2, dtype=torch.float64, device="cuda")
    f = BASE ** (-2 * i / PE)
    if scaling == "linear":
        return f / 4, 1.0
    if scaling == "yarn":
        at = lambda turns: PE * math.log(8192 / (turns * 2 * math.pi)) / (2 * math.log(BASE))  # noqa: E731
        low, high = max(math.floor(at(32)), 0), min(math.ceil(at(1)), PE - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        return f * (1 - ramp) + f / 16 * ramp, 0.1 * math.log(16) + 1
    return f, 1.0


def _rotated(x, positions, layout, scaling, dtype=torch.float32):
    """The last axis of x [tokens, ..., PE] turned; cosines in 64 bits, rounded once."""
    f, magnitude = _frequencies(scaling)
    angle = positions.double().view(-1, *[1] * (x.dim() - 1)) * f
    c, s = (angle.cos() * magnitude).to(dtype), (angle.sin() * magnitude).to(dtype)
    half = PE // 2
    a, b = (x[..., 0::2], x[..., 1::2]) if layout == "interleaved" else (x[..., :half], x[..., half:])
    y = torch.empty_like(x)
    a, b = a * c - b * s, a * s + b * c
    if layout == "interleaved":
        y[..., 0::2], y[..., 1::2] = a, b
    else:
        y[..., :half], y[..., half:] = a, b
    return y


def _pool_views(c, pool):
    """The values that a pool of pages holds: [pages, 16, 576], or codes and scales."""
    width, n = RANK + PE, pool.shape[0]
    if c["cache"] == F16:
        return [pool.view(torch.float16).view(n, 16, width)]
    return [pool[:, :16 * width].view(torch.int8).view(n, 16, width),
            pool[:, 16 * width:].view(torch.float16).view(n, 16, width // 32)]


def _rows(c, pool, pages, dtype=torch.float32):
    """Cached rows of the named pages [..., p], as [..., 16 p, 576]."""
    v = _pool_views(c, pool)
    rows = v[0][pages.long()].to(dtype)
    if c["cache"] == Q8:
        rows = (rows.unflatten(-1, (-1, 32)) * v[1][pages.long()].to(dtype)[..., None]).flatten(-2)
    return rows.flatten(-3, -2)


def _plain(s):
    c, kind = s.case, s.case["kind"]
    if kind == "norm":
        x = s.x + s.residual if c["residual"] else s.x
        y = _rms(x, s.weight)
        more = [x] if c["residual"] else []
        if c["out"] == Q8:
            return [*_quantised(y), *more]
        return [y.half() if c["out"] == F16 else y, *more]
    if kind == "rope":
        y = s.x.clone()
        y[..., HEAD_DIM - PE:] = _rotated(s.x[..., HEAD_DIM - PE:], s.positions, c["layout"], c["scaling"])
        return y
    if kind == "store":
        row = torch.cat([_rms(s.kv[:, :RANK], s.weight),
                         _rotated(s.kv[:, RANK:], s.positions, c["layout"], "none")], 1)
        parts = [row.half()] if c["cache"] == F16 else _quantised(row)
        live = s.slots >= 0
        page, at = s.slots[live].long() // 16, s.slots[live].long() % 16
        for pool, part in zip(s.outputs, parts):
            pool[page, at] = part.reshape(c["tokens"], -1)[live]
        return s.outputs
    if kind == "attn":
        pages = s.tables if s.table_of is None else s.tables[s.table_of.long()]
        rows = _rows(c, s.pool, pages)
        scores = torch.matmul(torch.cat([s.q, s.q_pe], -1), rows.transpose(1, 2)) * SCALE
        scores.masked_fill_((torch.arange(rows.shape[1], device="cuda") >= s.lens[:, None])[:, None], -math.inf)
        top = scores.amax(-1, keepdim=True)
        e = torch.exp(scores - top)
        total = e.sum(-1, keepdim=True)
        return [torch.matmul(e, rows[..., :RANK]) / total, (top + torch.log(total))[..., 0]]
    x = s.logits
    shifted = x - x.amax(-1, keepdim=True)
    e = torch.exp(shifted)
    total = e.sum(-1, keepdim=True)
    logp = shifted - torch.log(total)
    entropy = torch.log(total[:, 0]) - torch.where(e > 0, e * shifted, torch.zeros_like(e)).sum(-1) / total[:, 0]
    bits = (x + 0.0).view(torch.int32)
    order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long()
    key = order * (1 << 32) + (0xFFFFFFFF - torch.arange(c["vocab"], device="cuda"))
    top = torch.topk(key, c["top"], dim=-1, sorted=True)[1]
    return [logp.gather(1, s.tokens.long()), entropy, top.int(), logp.gather(1, top)]


# ---- the framework's calls ------------------------------------------------

class _Ptr:
    """A device tensor as the binding takes device buffers (an address)."""

    def __init__(self, t):
        self.t, self.ptr, self.nbytes = t, t.data_ptr(), t.numel() * t.element_size()


_kept = {}


def _library():
    if not _kept:
        sys.path.insert(0, os.path.join(os.getcwd(), "mobile-moe.zig_amd", "python"))
        import mmhip
        torch.cuda.init()
        _kept.update(mm=mmhip, ctx=mmhip.Context(0), rope={})
    return _kept["mm"], _kept["ctx"]


def _rope(layout, scaling):
    """The rotary plans a program keeps: one for each of its models' settings."""
    mm, ctx = _library()
    if (layout, scaling) not in _kept["rope"]:
        more = {"none": {}, "linear": dict(factor=4.0),
                "yarn": dict(factor=16.0, original_context=8192, beta_fast=32.0, beta_slow=1.0)}[scaling]
        _kept["rope"][layout, scaling] = mm.Rope(ctx, dims=PE, base=BASE, layout=layout, scaling=scaling, **more)
    return _kept["rope"][layout, scaling]


def _cache(s):
    mm, _ = _library()
    return mm.KvCache(_Ptr(s.pool), mm.F16 if s.case["cache"] == F16 else mm.Q8_0, rank=RANK, rope_dims=PE,
                      page_tokens=16, n_pages=s.pool.shape[0])


def _arguments(s):
    """A call's buffers by their addresses: a program lays them out once for the steps it makes."""
    mm, ctx = _library()
    c, kind = s.case, s.case["kind"]
    if kind == "norm":
        kind_of = {F32: mm.F32, F16: mm.F16, Q8: mm.Q8_0}[c["out"]]
        more = dict(residual=_Ptr(s.residual), sum_out=_Ptr(s.sum)) if c["residual"] else {}
        return (_Ptr(s.y), _Ptr(s.x), _Ptr(s.weight), c["rows"], c["cols"]), dict(eps=EPS, y_type=kind_of, **more)
    if kind == "rope":
        return ((_rope(c["layout"], c["scaling"]), _Ptr(s.y), _Ptr(s.x), _Ptr(s.positions), c["tokens"], c["heads"],
                 HEAD_DIM), dict(first=HEAD_DIM - PE))
    if kind == "store":
        return ((_cache(s), _Ptr(s.kv), _Ptr(s.slots), c["tokens"]),
                dict(norm_weight=_Ptr(s.weight), eps=EPS, rope=_rope(c["layout"], "none"), positions=_Ptr(s.positions)))
    if kind == "attn":
        work = torch.empty(ctx.mla_attention_workspace(c["tokens"], c["heads"], RANK), dtype=torch.uint8, device="cuda")
        return ctx.mla_attention_args(
            _cache(s), q=_Ptr(s.q), q_pe=_Ptr(s.q_pe), out=_Ptr(s.out), lse=_Ptr(s.lse), tables=_Ptr(s.tables),
            n_tables=s.tables.shape[0], table_pages=s.tables.shape[1], lens=_Ptr(s.lens),
            table_of=None if s.table_of is None else _Ptr(s.table_of), n_tokens=c["tokens"], n_heads=c["heads"],
            scale=SCALE, workspace=_Ptr(work)), None
    work = torch.empty(ctx.logprobs_workspace(c["rows"], c["vocab"], c["top"]), dtype=torch.uint8, device="cuda")
    return ((_Ptr(s.logits), c["rows"], c["vocab"]),
            dict(tokens=_Ptr(s.tokens), n_given=c["given"], token_logprobs=_Ptr(s.logp), entropy=_Ptr(s.entropy),
                 top=c["top"], top_ids=_Ptr(s.top_ids), top_logprobs=_Ptr(s.top_logp), workspace=_Ptr(work)))


def _own(s):
    mm, ctx = _library()
    kind = s.case["kind"]
    if s.args is None:
        s.args = _arguments(s)
    args, more = s.args
    if kind == "norm":
        ctx.rms_norm_dev(*args, **more)
        return s.outputs
    if kind == "rope":
        ctx.rope_dev(*args, **more)
        return s.y
    if kind == "store":
        ctx.kv_store_dev(*args, **more)
        return s.outputs
    if kind == "attn":
        ctx.mla_attention_dev(args)
        return [s.out, s.lse]
    ctx.logprobs_dev(*args, **more)
    return [s.logp, s.entropy, s.top_ids, s.top_logp]


def run(s):
    return _own(s) if own else _plain(s)


# ---- what a pass cannot do without ----------------------------------------

def work(case):
    c, kind = case, case["kind"]
    if kind == "norm":
        n = c["rows"] * c["cols"]
        out = c["rows"] * ((c["cols"] + 31) // 32) * 34 if c["out"] == Q8 else n * (2 if c["out"] == F16 else 4)
        return dict(bytes=4 * n * (3 if c["residual"] else 1) + 4 * c["cols"] + out, flops=6 * n)
    if kind == "rope":
        n = c["tokens"] * c["heads"]
        return dict(bytes=8 * n * HEAD_DIM + 4 * c["tokens"], flops=3 * n * PE)
    row = (RANK + PE) * 2 if c.get("cache") == F16 else (RANK + PE) * 34 // 32
    if kind == "store":
        return dict(bytes=c["tokens"] * (4 * (RANK + PE) + row + 8) + 4 * RANK, flops=6 * c["tokens"] * (RANK + PE))
    if kind == "attn":
        n, longest = c["tokens"], c["longest"]
        if c["lens"] == "chunk":  # one context, read once
            seen, pairs = longest, n * (longest - (n - 1) / 2)
        elif c["lens"] == "ragged":  # lengths uniform in their logarithm
            seen = pairs = longest + (n - 1) * (longest - 1) / max(math.log(longest), 1e-9) if longest > 1 else n
        else:
            seen = pairs = n * longest
        return dict(bytes=seen * row + 4 * n * c["heads"] * (2 * RANK + PE + 1) + 4 * seen / 16,
                    flops=2 * c["heads"] * pairs * (2 * RANK + PE))
    n = c["rows"]
    return dict(bytes=4 * n * c["vocab"] + 8 * n * (c["given"] + c["top"]) + 4 * n, flops=6 * n * c["vocab"])


# ---- the same results in 64 bits ------------------------------------------

def _exact_rows(c, s, ids):
    width = RANK + PE
    raw = s.pool[ids.long()]
    if c["cache"] == F16:
        return raw.view(torch.float16).double().view(-1, width)
    codes = raw[:, :16 * width].contiguous().view(torch.int8).double().view(-1, width // 32, 32)
    scales = raw[:, 16 * width:].contiguous().view(torch.float16).double().view(-1, width // 32, 1)
    return (codes * scales).view(-1, width)


def _exact_turn(x, positions, layout, scaling):
    f, magnitude = _frequencies(scaling)
    z = torch.polar(torch.full((len(positions), PE // 2), float(magnitude), dtype=torch.float64, device="cuda"),
                    positions.double()[:, None] * f).view(-1, *[1] * (x.dim() - 2), PE // 2)
    pairs = x.double().unflatten(-1, (PE // 2, 2)) if layout == "interleaved" else \
        x.double().unflatten(-1, (2, PE // 2)).transpose(-1, -2)
    y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * z)
    return (y if layout == "interleaved" else y.transpose(-1, -2)).flatten(-2)


def exact(case, seed):
    c, s, kind = case, prepare(case, seed), case["kind"]
    if kind == "norm":
        x = s.x.double() + (s.residual.double() if c["residual"] else 0)
        y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * s.weight.double()
        if c["out"] == Q8:
            y = torch.nn.functional.pad(y, (0, -c["cols"] % 32)).unflatten(-1, (-1, 32)).abs().amax(-1) / 127
        return [*([None] if c["out"] == Q8 else []), y, *([x] if c["residual"] else [])]
    if kind == "rope":
        keep = HEAD_DIM - PE
        return torch.cat([s.x[..., :keep].double(),
                          _exact_turn(s.x[..., keep:], s.positions, c["layout"], c["scaling"])], -1)
    if kind == "store":
        x = s.kv[:, :RANK].double()
        row = torch.cat([x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * s.weight.double(),
                         _exact_turn(s.kv[:, RANK:], s.positions, c["layout"], "none")], 1)
        values = s.outputs[-1].double()
        for t, slot in enumerate(s.slots.tolist()):
            if slot >= 0:
                values[slot // 16, slot % 16] = row[t] if c["cache"] == F16 else row[t].view(-1, 32).abs().amax(-1) / 127
        return [values] if c["cache"] == F16 else [None, values]
    if kind == "attn":
        out, lse = [], []
        shared = _exact_rows(c, s, s.tables[0]) if s.table_of is not None else None
        for t, n in enumerate(s.lens.tolist()):
            rows = (shared if shared is not None else _exact_rows(c, s, s.tables[t, :(n + 15) // 16]))[:n]
            scores = torch.cat([s.q[t], s.q_pe[t]], -1).double() @ rows.t().contiguous() * SCALE
            out.append(torch.softmax(scores, -1) @ rows[:, :RANK])
            lse.append(torch.logsumexp(scores, -1))
        return [torch.stack(out), torch.stack(lse)]
    logp = torch.log_softmax(s.logits.double(), -1)
    p = logp.exp()
    top = torch.sort(s.logits, dim=-1, descending=True, stable=True)[1][:, :c["top"]]
    return [logp.gather(1, s.tokens.long()), -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(-1), None,
            logp.gather(1, top)]
