"""The two ends of a serving step and its 4-bit tensors, as measurable cases:
products with 4-bit weights that share a scale in groups of 32, the rows of a
quantised embedding table, the page tables, slots and positions of a step's
requests, and tokens drawn from the logits with temperature, top-k, top-p and
min-p.

Each case runs in one of two forms: elementary torch operations, or (where `own`
is true) the calls a program makes of the Python binding. The shapes are those
of the benchmark and the tests: hidden 2048, experts of width 1536, latent
projections of 768 and 3840, a dense width of 10240, pages of 16 positions, a
vocabulary of 154,880, prompts in chunks of up to 256 tokens.
"""
import math
import os
import re
import sys

import torch

own = False

Q4, IQ4, Q8, IQ2, F16, F32 = "q4_0", "iq4_nl", "q8_0", "iq2_xxs", "f16", "f32"
VOCAB, HIDDEN, PAGE = 154880, 2048, 16
NO_TOKEN = -1  # 0xFFFFFFFF
# The 16 values of an IQ4_NL code (the format's table).
IQ4_VALUES = [-127, -104, -83, -65, -49, -35, -22, -10, 1, 13, 25, 38, 53, 69, 89, 113]


def listed():
    return [
        # The first latent projection for one token: the smallest product.
        dict(name="q4_proj_decode", kind="product", fmt=Q4, mats=1, rows=768, cols=2048, tokens=1),
        # A layer's 64 experts' gate matrices times one token, in one launch.
        dict(name="q4_experts_step", kind="product", fmt=IQ4, mats=64, rows=1536, cols=2048, tokens=1),
        # The output projection for four conversations at once.
        dict(name="q4_logits", kind="product", fmt=Q4, mats=1, rows=VOCAB, cols=HIDDEN, tokens=4),
        # A ragged chunk of a prompt through the second latent projection, and
        # a whole chunk through the dense layer's wide one.
        dict(name="q4_chunk_ragged", kind="product", fmt=IQ4, mats=1, rows=3840, cols=768, tokens=77),
        dict(name="q4_prompt", kind="product", fmt=Q4, mats=1, rows=10240, cols=2048, tokens=256),
        # Embedding rows: one token, and the tokens of several prompts with
        # padding behind them.
        dict(name="embed_decode", kind="embed", fmt=Q8, rows=VOCAB, cols=HIDDEN, tokens=1, pad=0),
        dict(name="embed_prompt", kind="embed", fmt=IQ4, rows=VOCAB, cols=HIDDEN, tokens=4096, pad=77),
        # A step of 64 conversations that each add a token, and one in which
        # prompts of all lengths arrive beside conversations that go on.
        dict(name="plan_decode", kind="plan", requests=64, prompts=0, longest=16384, idle=3),
        dict(name="plan_prompts", kind="plan", requests=512, prompts=64, longest=16384, idle=40),
        # One token of one conversation with a nucleus; a batch with few
        # candidates each; a batch in which every request has settings of its
        # own, some of the vocabulary masked.
        dict(name="sample_one", kind="sample", rows=1, vocab=VOCAB, mode="nucleus", masked=False),
        dict(name="sample_topk", kind="sample", rows=16, vocab=VOCAB, mode="topk", masked=False),
        dict(name="sample_batch", kind="sample", rows=64, vocab=VOCAB, mode="mixed", masked=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["product", "product", "product", "embed", "plan", "sample", "sample"])
    if kind == "product":
        cols = 32 * rng.randint(8, 128)
        tokens = rng.choice([1, 1, rng.randint(2, 16), _log(rng, 2, 256)])
        mats = rng.choice([1, 1, rng.randint(2, 64)]) if tokens == 1 else 1
        most = min(200_000_000 // (cols * mats), 4_000_000_000 // (cols * tokens), VOCAB)
        return dict(kind=kind, fmt=rng.choice([Q4, IQ4]), mats=mats, rows=_log(rng, 200, max(201, most)), cols=cols,
                    tokens=tokens)
    if kind == "embed":
        fmt = rng.choice([Q4, IQ4, Q8, IQ2, F16, F32])
        cols = 256 * rng.randint(1, 8) if fmt == IQ2 else 32 * rng.randint(4, 64)
        tokens = _log(rng, 1, 4096)
        return dict(kind=kind, fmt=fmt, rows=_log(rng, 1000, VOCAB), cols=cols, tokens=tokens,
                    pad=rng.choice([0, rng.randint(0, tokens - 1)]))
    if kind == "plan":
        requests = _log(rng, 1, 512)
        return dict(kind=kind, requests=requests, prompts=rng.randint(0, max(1, requests // 8)),
                    longest=_log(rng, 16, 16384), idle=rng.randint(0, requests // 8))
    return dict(kind=kind, rows=_log(rng, 1, 64), vocab=rng.choice([VOCAB, _log(rng, 1000, VOCAB)]),
                mode=rng.choice(["nucleus", "topk", "mixed", "plain"]), masked=rng.random() < 0.3)


# ---- inputs ---------------------------------------------------------------

class _State:
    """What a program has in hand before a call, and what it keeps between calls."""

    def __init__(self, case):
        self.case, self.args, self.weight = dict(case), None, None

    def __del__(self):
        if self.weight is not None:
            self.weight.free()


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _blocks(g, fmt, n):
    """n blocks as a file holds them: a scale in 16 bits, then the codes."""
    size, scale = {Q4: (16, 0.005), IQ4: (16, 0.0006), Q8: (32, 0.0003), IQ2: (64, 0.0004)}[fmt]
    codes = torch.randint(0, 256, (n, size), generator=g, device="cuda", dtype=torch.uint8)
    d = scale * (0.5 + torch.rand(n, 1, generator=g, device="cuda"))
    return torch.cat([d.half().view(torch.uint8), codes], 1)


def _lengths(n, longest):
    """n lengths, uniform in their logarithm."""
    return [max(1, round(math.exp((i + 0.5) / n * math.log(longest)))) for i in range(n)]


def _pages(positions):
    return -(-positions // PAGE)


def prepare(case, seed):
    c, s, g, kind = case, _State(case), _gen(seed), case["kind"]
    if kind == "product":
        n, r, k = c["mats"], c["rows"], c["cols"]
        s.raw = _blocks(g, c["fmt"], n * r * k // 32)
        s.x = _randn(g, c["tokens"], k)
        s.y = torch.zeros(max(n, c["tokens"]), r, device="cuda")
    elif kind == "embed":
        n, v, k = c["tokens"], c["rows"], c["cols"]
        if c["fmt"] in (F16, F32):
            s.table = (0.02 * _randn(g, v, k)).to(torch.float16 if c["fmt"] == F16 else torch.float32)
        else:
            s.table = _blocks(g, c["fmt"], v * k // (256 if c["fmt"] == IQ2 else 32)).view(v, -1)
        s.tokens = torch.randint(0, v, (n,), generator=g, device="cuda", dtype=torch.int32)
        s.tokens[n - c["pad"]:] = NO_TOKEN
        s.y = torch.zeros(n, k, device="cuda")
    elif kind == "plan":
        n, new_ones, longest = c["requests"], c["prompts"], c["longest"]
        who = torch.randperm(n, generator=g, device="cuda")
        lens, prompts = _lengths(n - new_ones, longest), _lengths(new_ones, longest)
        s.lens, s.new = (torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(2))
        s.new[who[:new_ones]] = torch.tensor(prompts, dtype=torch.int32, device="cuda")  # nothing is cached yet
        s.lens[who[new_ones:]], s.new[who[new_ones:]] = torch.tensor(lens, dtype=torch.int32, device="cuda"), 1
        # Idle rows; those that ended give their pages back.
        s.release = torch.zeros(n, dtype=torch.int32, device="cuda")
        idle = who[n - torch.randperm(n - new_ones, generator=g, device="cuda")[:c["idle"]] - 1]
        s.new[idle], s.release[idle] = 0, 1
        s.table_pages = (longest + PAGE) // PAGE + 1
        held = (s.lens.long() + PAGE - 1) // PAGE
        total = sum(_pages(v) for v in lens)
        s.n_pages = total + sum(_pages(v) for v in prompts) + n + 64
        ids = torch.randperm(s.n_pages, generator=g, device="cuda").int()
        s.tables = torch.zeros(n, s.table_pages, dtype=torch.int32, device="cuda")
        s.tables[torch.arange(s.table_pages, device="cuda") < held[:, None]] = ids[:total]
        s.free = torch.zeros(s.n_pages, dtype=torch.int32, device="cuda")
        s.free[:s.n_pages - total] = ids[total:]
        s.free_count = torch.full((1,), s.n_pages - total, dtype=torch.int32, device="cuda")
        s.max_tokens = sum(prompts) + n - new_ones - c["idle"] + 13
        ints = lambda m: torch.zeros(m, dtype=torch.int32, device="cuda")  # noqa: E731
        s.positions, s.slots, s.table_of, s.seen = (ints(s.max_tokens) for _ in range(4))
        s.firsts, s.granted, s.last, s.next_lens, s.next_free = ints(n + 1), ints(n), ints(n), ints(n), ints(1)
        s.outputs = [s.positions, s.slots, s.table_of, s.seen, s.firsts, s.granted, s.last, s.next_lens, s.tables,
                     s.free, s.next_free]
    else:
        n, v, mode = c["rows"], c["vocab"], c["mode"]
        # Few likely tokens above a broad rest; how far above differs by row.
        s.logits = 2.0 * _randn(g, n, v)
        peak = torch.randint(0, v, (n, 24), generator=g, device="cuda")
        sure = 6 + 12 * torch.rand(n, 1, generator=g, device="cuda")
        s.logits.scatter_(1, peak, sure + 1.5 * _randn(g, n, 24))
        if c["masked"]:
            s.logits[:, torch.rand(v, generator=g, device="cuda") < 0.6] = -math.inf
            s.logits[:, 0] = 0.5
        pick = lambda *of: torch.tensor(of, device="cuda")[  # noqa: E731
            torch.randint(0, len(of), (n,), generator=g, device="cuda")]
        if mode == "mixed":
            s.temperature = pick(0.0, 0.6, 0.8, 1.0, 1.3).float()
            s.top_k, s.top_p, s.min_p = pick(0, 0, 40, 200).int(), pick(1.0, 0.9, 0.95).float(), pick(0.0, 0.0, 0.05).float()
        else:
            s.temperature = torch.full((n,), 0.8, device="cuda")
            s.top_k = torch.full((n,), 40 if mode == "topk" else 0, dtype=torch.int32, device="cuda")
            s.top_p = torch.full((n,), 0.95 if mode == "nucleus" else 1.0, device="cuda")
            s.min_p = torch.zeros(n, device="cuda")
        s.uniform = torch.rand(n, generator=g, device="cuda")
        s.tokens, s.kept = (torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(2))
        s.probs = torch.zeros(n, device="cuda")
    torch.cuda.synchronize()  # the library works on a stream of its own
    return s


# ---- the plain form -------------------------------------------------------

def _iq2_signs_and_grid():
    """The 256 groups of eight magnitudes of the 2-bit format, from the data file of its table."""
    if "grid" not in _kept:
        path = os.path.join(os.getcwd(), "mobile-moe.zig_amd", "csrc", "iq2xxs_grid.inc")
        text = "".join(line for line in open(path) if not line.lstrip().startswith("//"))
        words = [int(w, 16) for w in re.findall(r"0x[0-9a-fA-F]{16}", text)]
        _kept["grid"] = torch.tensor([[w >> (8 * i) & 255 for i in range(8)] for w in words], device="cuda")
        signs = [[-1 if (i | (bin(i).count("1") & 1) << 7) >> j & 1 else 1 for j in range(8)] for i in range(128)]
        _kept["signs"] = torch.tensor(signs, device="cuda")
    return _kept["grid"], _kept["signs"]


def _values(fmt, raw, dtype):
    """Blocks [..., bytes] -> their weights [..., 32 or 256]."""
    d = raw[..., :2].contiguous().view(torch.float16).to(dtype)
    codes = raw[..., 2:]
    if fmt == Q8:
        return codes.contiguous().view(torch.int8).to(dtype) * d
    if fmt == IQ2:  # eight groups of 32: four grid numbers, then four sign codes and a 4-bit scale
        grid, signs = _iq2_signs_and_grid()
        q = codes.contiguous().view(*codes.shape[:-1], 8, 8)
        word = q[..., 4:].contiguous().view(torch.int32)[..., 0].long() & 0xFFFFFFFF
        v = grid[q[..., :4].int()].to(dtype) * signs[torch.stack([word >> (7 * i) & 127 for i in range(4)], -1)].to(dtype)
        return ((0.5 + (word >> 28).to(dtype)) * 0.25)[..., None].mul(d[..., None] * v.flatten(-2)).flatten(-2)
    nibbles = torch.cat([codes & 15, codes >> 4], -1)
    if fmt == Q4:
        return (nibbles.to(dtype) - 8) * d
    return torch.tensor(IQ4_VALUES, dtype=dtype, device="cuda")[nibbles.int()] * d


def _plan_plain(s):
    dev = "cuda"
    L, new, P = s.lens.long(), s.new.long(), PAGE
    L0 = torch.where(s.release > 0, 0, L)
    count = s.free_count.long()
    # Pages that come back, request by request.
    back = torch.where(s.release > 0, (L + P - 1) // P, 0)
    used = torch.arange(s.table_pages, device=dev) < back[:, None]
    given = s.tables[used]
    s.free[count + torch.arange(len(given), device=dev)] = given
    count = count + len(given)
    # Whose tokens and pages there is room for.
    fits = (new > 0) & (L0 + new <= s.table_pages * P)
    asked = torch.where(fits, new, 0)
    fits &= torch.cumsum(asked, 0) <= s.max_tokens
    need = torch.where(fits, (L0 + new + P - 1) // P - (L0 + P - 1) // P, 0)
    ok = fits & ((need == 0) | (torch.cumsum(need, 0) <= count))
    need, new = torch.where(ok, need, 0), torch.where(ok, new, 0)
    # New pages from the top of the free ones.
    end = torch.cumsum(need, 0)
    r = torch.repeat_interleave(torch.arange(len(L), device=dev), need)
    i = torch.arange(len(r), device=dev)
    s.tables[r, (L0[r] + P - 1) // P + i - (end - need)[r]] = s.free[count - 1 - i]
    # The step's tokens.
    last = torch.cumsum(new, 0)
    t = torch.repeat_interleave(torch.arange(len(L), device=dev), new)
    j = torch.arange(len(t), device=dev)
    pos = L0[t] + j - (last - new)[t]
    for out, value, pad in ((s.positions, pos, 0), (s.table_of, t, 0), (s.seen, pos + 1, 0),
                            (s.slots, s.tables[t, pos // P].long() * P + pos % P, -1)):
        out.fill_(pad)
        out[:len(t)] = value.int()
    s.firsts[0], s.firsts[1:] = 0, last.int()
    s.granted.copy_(ok)
    s.last.copy_(torch.where(new > 0, last - 1, NO_TOKEN))
    s.next_lens.copy_(L0 + new)
    s.next_free.copy_(count - need.sum())
    return s.outputs


def _sample_plain(s):
    x, order = torch.sort(s.logits, dim=-1, descending=True, stable=True)  # equal logits by the lower id
    x, rank = x.double(), torch.arange(s.case["vocab"], device="cuda")
    t = s.temperature.double()[:, None]
    z = (x - x[:, :1]) / torch.where(t > 0, t, torch.ones_like(t))
    k = s.top_k.long()[:, None]
    k = torch.where(t > 0, torch.where(k > 0, k, s.case["vocab"]), torch.ones_like(k))
    w = torch.where(rank < k, torch.exp(z), torch.zeros_like(z))
    before = torch.cumsum(w, -1) - w
    p = s.top_p.double()[:, None]
    keep = (rank < k) & (x > -math.inf) & (z >= torch.log(s.min_p.double())[:, None])
    keep &= (p >= 1) | (before < p * w.sum(-1, keepdim=True)) | (rank == 0)
    w = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, torch.zeros_like(w)))
    running = torch.cumsum(w, -1)
    total = running[:, -1:]
    token = (running <= s.uniform.double()[:, None] * total).sum(-1, keepdim=True)
    return [token[:, 0].int(), (w.gather(1, token) / total)[:, 0].float(), keep.sum(-1).int()]


def _plain(s):
    c, kind = s.case, s.case["kind"]
    if kind == "product":
        w = _values(c["fmt"], s.raw, torch.float32).view(c["mats"] * c["rows"], c["cols"])
        return torch.matmul(s.x, w.t()).view(-1, c["rows"])
    if kind == "embed":
        live = s.tokens != NO_TOKEN
        rows = s.table[s.tokens[live].long()]
        if c["fmt"] in (F16, F32):
            rows = rows.float()
        else:
            rows = _values(c["fmt"], rows.view(len(rows), -1, 66 if c["fmt"] == IQ2 else 34 if c["fmt"] == Q8 else 18),
                           torch.float32).flatten(1)
        s.y[live] = rows * math.sqrt(c["cols"])
        return s.y
    if kind == "plan":
        return _plan_plain(s)
    return _sample_plain(s)


# ---- the framework's calls ------------------------------------------------

class _Ptr:
    """A device tensor as the binding takes device buffers (an address)."""

    def __init__(self, t):
        self.t, self.ptr, self.nbytes = t, t.data_ptr(), t.numel() * t.element_size()


_kept = {}


def _library():
    if "mm" not in _kept:
        sys.path.insert(0, os.path.join(os.getcwd(), "mobile-moe.zig_amd", "python"))
        import mmhip
        torch.cuda.init()
        _kept.update(mm=mmhip, ctx=mmhip.Context(0))
    return _kept["mm"], _kept["ctx"]


def _type(fmt):
    mm, _ = _library()
    return {Q4: mm.Q4_0, IQ4: mm.IQ4_NL, Q8: mm.Q8_0, IQ2: mm.IQ2_XXS, F16: mm.F16, F32: mm.F32}[fmt]


def _arguments(s):
    """A call's buffers by their addresses: a program lays them out once for the steps it makes."""
    mm, ctx = _library()
    c, kind = s.case, s.case["kind"]
    if kind == "product":
        s.weight = ctx.weight_from_device(_Ptr(s.raw), _type(c["fmt"]), c["rows"], c["cols"], c["mats"])
        return _Ptr(s.x), _Ptr(s.y)
    if kind == "embed":
        return _Ptr(s.y), _Ptr(s.table), _type(c["fmt"]), c["rows"], c["cols"], _Ptr(s.tokens), c["tokens"]
    if kind == "plan":
        work = torch.empty(ctx.kv_plan_workspace(c["requests"]), dtype=torch.uint8, device="cuda")
        return ctx.kv_plan_args(
            n_requests=c["requests"], lens=_Ptr(s.lens), new=_Ptr(s.new), release=_Ptr(s.release),
            next_lens=_Ptr(s.next_lens), tables=_Ptr(s.tables), table_pages=s.table_pages, page_tokens=PAGE,
            n_pages=s.n_pages, free=_Ptr(s.free), free_count=_Ptr(s.free_count), next_free_count=_Ptr(s.next_free),
            max_tokens=s.max_tokens, positions=_Ptr(s.positions), slots=_Ptr(s.slots), table_of=_Ptr(s.table_of),
            seen=_Ptr(s.seen), firsts=_Ptr(s.firsts), granted=_Ptr(s.granted), last=_Ptr(s.last), workspace=_Ptr(work))
    work = torch.empty(ctx.sample_workspace(c["rows"], c["vocab"]), dtype=torch.uint8, device="cuda")
    return ctx.sample_args(
        logits=_Ptr(s.logits), n_rows=c["rows"], vocab=c["vocab"], temperature=_Ptr(s.temperature), top_k=_Ptr(s.top_k),
        top_p=_Ptr(s.top_p), min_p=_Ptr(s.min_p), uniform=_Ptr(s.uniform), tokens=_Ptr(s.tokens), probs=_Ptr(s.probs),
        kept=_Ptr(s.kept), workspace=_Ptr(work))


def _own(s):
    _, ctx = _library()
    c, kind = s.case, s.case["kind"]
    if s.args is None:
        s.args = _arguments(s)
    if kind == "product":
        x, y = s.args
        if c["tokens"] == 1:
            ctx.gemv_batched_dev(s.weight, 0, c["mats"], x, 0, y, c["rows"])
        else:
            ctx.qmm_dev(s.weight, 0, x, y, c["tokens"])
        return s.y
    if kind == "embed":
        ctx.embed_dev(*s.args, scale=math.sqrt(c["cols"]))
        return s.y
    if kind == "plan":
        ctx.kv_plan_dev(s.args)
        return s.outputs
    ctx.sample_dev(s.args)
    return [s.tokens, s.probs, s.kept]


def run(s):
    return _own(s) if own else _plain(s)


# ---- what a pass cannot do without ----------------------------------------

def work(case):
    c, kind = case, case["kind"]
    if kind == "product":
        n = c["mats"] * c["rows"]
        return dict(bytes=n * c["cols"] // 32 * 18 + 4 * c["tokens"] * c["cols"] + 4 * n * c["tokens"],
                    flops=2 * n * c["cols"] * c["tokens"])
    if kind == "embed":
        row = c["cols"] * {F32: 4, F16: 2, Q8: 34 / 32, IQ2: 66 / 256}.get(c["fmt"], 18 / 32)
        n = c["tokens"] - c["pad"]
        return dict(bytes=int(n * (row + 4 * c["cols"]) + 4 * c["tokens"]), flops=2 * n * c["cols"])
    if kind == "plan":
        # Per request six numbers in and out, per token four out; the pages that
        # are taken are read and written, those of the idle ones too.
        prompts, lens = _lengths(c["prompts"], c["longest"]), _lengths(c["requests"] - c["prompts"], c["longest"])
        tokens = sum(prompts) + len(lens) - c["idle"]
        moved = sum(_pages(v) for v in prompts) + (len(lens) - c["idle"]) / PAGE
        back = c["idle"] * sum(_pages(v) for v in lens) / max(1, len(lens))
        return dict(bytes=int(4 * (6 * c["requests"] + 4 * tokens + 2 * moved + 2 * back)),
                    flops=int(4 * tokens + 8 * c["requests"]))
    n = c["rows"]
    return dict(bytes=4 * n * c["vocab"] + 32 * n, flops=10 * n * c["vocab"])


# ---- the same results in 64 bits ------------------------------------------

def _exact_weights(fmt, raw):
    d = raw[:, :2].contiguous().view(torch.float16).double()
    if fmt == Q8:
        return raw[:, 2:].contiguous().view(torch.int8).double() * d
    table = torch.arange(-8, 8, device="cuda") if fmt == Q4 else torch.tensor(IQ4_VALUES, device="cuda")
    out = torch.empty(len(raw), 32, dtype=torch.float64, device="cuda")
    out[:, :16] = table[(raw[:, 2:] % 16).int()].double()
    out[:, 16:] = table[torch.div(raw[:, 2:], 16, rounding_mode="floor").int()].double()
    return out.mul_(d)


def _exact_plan(s):
    """Request by request, as a program on the host would go about it."""
    lens, new, rel = s.lens.tolist(), s.new.tolist(), s.release.tolist()
    tables, free = s.tables.tolist(), s.free.tolist()
    top = int(s.free_count)
    n, P = len(lens), PAGE
    for r in range(n):
        if rel[r]:
            for i in range(-(-lens[r] // P)):
                free[top] = tables[r][i]
                top += 1
            lens[r] = 0
    stack, asked, wanted = top, 0, 0
    firsts, granted, last, pos, slots, of = [0], [], [], [], [], []
    for r in range(n):
        ok = 0 < new[r] <= s.table_pages * P - lens[r]
        if ok:
            asked += new[r]
            ok = asked <= s.max_tokens
        if ok:
            held, all_ = -(-lens[r] // P), -(-(lens[r] + new[r]) // P)
            wanted += all_ - held
            ok = all_ == held or wanted <= stack
        if ok:
            for i in range(held, all_):
                top -= 1
                tables[r][i] = free[top]
            for q in range(lens[r], lens[r] + new[r]):
                pos.append(q)
                slots.append(tables[r][q // P] * P + q % P)
                of.append(r)
            lens[r] += new[r]
        granted.append(int(ok))
        last.append(len(pos) - 1 if ok else NO_TOKEN)
        firsts.append(len(pos))
    pad = s.max_tokens - len(pos)
    return [torch.tensor(v, device="cuda") for v in (
        pos + [0] * pad, slots + [-1] * pad, of + [0] * pad, [q + 1 for q in pos] + [0] * pad, firsts, granted, last, lens,
        tables, free, [top])]


def _exact_sample(s):
    tokens, probs, kept = [], [], []
    for r in range(s.case["rows"]):
        x = s.logits[r].double()
        t, k, p, least = float(s.temperature[r]), int(s.top_k[r]), float(s.top_p[r]), float(s.min_p[r])
        ids = torch.nonzero(x > -math.inf)[:, 0]
        ids = ids[torch.sort(-x[ids], stable=True)[1]]
        if t == 0:
            tokens.append(int(ids[0])), probs.append(1.0), kept.append(1)
            continue
        ids = ids[:k] if k else ids
        w = torch.softmax(x[ids] / t, 0)
        n = len(ids) if p >= 1 else max(1, int((w.cumsum(0) - w < p).sum()))
        n = min(n, int((w >= least * w[0]).sum()))
        ids, back = torch.sort(ids[:n])
        w = w[:n][back] / w[:n].sum()
        at = min(int(torch.searchsorted(w.cumsum(0), s.uniform[r].double(), right=True)), n - 1)
        tokens.append(int(ids[at])), probs.append(float(w[at])), kept.append(n)
    dev = dict(device="cuda")
    return [torch.tensor(tokens, **dev), torch.tensor(probs, dtype=torch.float64, **dev), torch.tensor(kept, **dev)]


def exact(case, seed):
    c, s, kind = case, prepare(case, seed), case["kind"]
    if kind == "product":
        w = _exact_weights(c["fmt"], s.raw).view(c["mats"], c["rows"], c["cols"])
        if c["tokens"] > 1:
            return s.x.double() @ w[0].t().contiguous()
        return torch.stack([m @ s.x[0].double() for m in w])
    if kind == "embed":
        if c["fmt"] == IQ2:
            rows = _values(IQ2, s.table.view(c["rows"], -1, 66), torch.float64).flatten(1)
        elif c["fmt"] in (F16, F32):
            rows = s.table.double()
        else:
            rows = _exact_weights(c["fmt"], s.table.view(-1, s.table.shape[1] * 32 // c["cols"])).view(c["rows"], -1)
        y = s.y.double()
        for t, token in enumerate(s.tokens.tolist()):
            if token != NO_TOKEN:
                y[t] = rows[token] * math.sqrt(c["cols"])
        return y
    return _exact_plan(s) if kind == "plan" else _exact_sample(s)
