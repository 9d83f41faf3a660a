"""Plain 64-bit forms of the operators between a decode step's products, and
what their tests share: a paged pool's bytes, and buffers on the device."""
import ctypes
import math

import numpy as np

import mmhip as mm

U = 2.0 ** -24  # half a step of f32, relative


def rms_norm64(s, w, eps):
    s = s.astype(np.float64)
    return s / np.sqrt((s * s).mean(-1, keepdims=True) + eps) * w.astype(np.float64)


def frequencies64(dims, base, scaling="none", factor=1.0, original_context=0, beta_fast=32.0, beta_slow=1.0, **_):
    f = [base ** (-2.0 * i / dims) for i in range(dims // 2)]
    if scaling == "linear":
        return [x / factor for x in f]
    if scaling == "yarn":
        def pair_of(turns):  # the pair that makes so many turns over the original context
            return dims * math.log(original_context / (turns * 2 * math.pi)) / (2 * math.log(base))
        low = min(max(math.floor(pair_of(beta_fast)), 0), dims - 1)
        high = min(max(math.ceil(pair_of(beta_slow)), 0), dims - 1)
        out = []
        for i, x in enumerate(f):
            r = min(max((i - low) / max(high - low, 0.001), 0.0), 1.0)
            out.append(x * (1 - r) + x / factor * r)
        return out
    return f


def rope64(x, positions, layout, freqs, magnitude=1.0):
    """x [tokens, heads, dims] turned."""
    x = x.astype(np.float64)
    n = x.shape[-1] // 2
    ia = np.arange(n) * 2 if layout == "interleaved" else np.arange(n)
    ib = ia + (1 if layout == "interleaved" else n)
    ang = positions.astype(np.float64)[:, None, None] * np.asarray(freqs)
    c, s = np.cos(ang) * magnitude, np.sin(ang) * magnitude
    y = x.copy()
    y[..., ia] = x[..., ia] * c - x[..., ib] * s
    y[..., ib] = x[..., ia] * s + x[..., ib] * c
    return y


def q8_blocks(rows):
    """Codes and scales of blocks of 32 (rows [..., 32 k], f32), as the codec's format has them: d = max / 127, code =
    x / d rounded half away from zero, d stored in f16."""
    b = rows.astype(np.float32).reshape(*rows.shape[:-1], -1, 32)
    d = (np.abs(b).max(-1) / np.float32(127)).astype(np.float32)
    with np.errstate(divide="ignore", invalid="ignore"):
        z = (b / d[..., None]).astype(np.float32)
    q = np.where(d[..., None] > 0, np.sign(z) * np.floor(np.abs(z).astype(np.float64) + 0.5), 0)
    return np.clip(q, -127, 127).astype(np.int8).reshape(rows.shape), d.astype(np.float16)


class Pool:
    """Pages of a cache on the host: raw bytes, and the values that they stand for."""

    def __init__(self, rng, ggml_type, rank, rope, page_tokens, n_pages, sigma=1.0):
        self.type, self.rank, self.rope, self.page_tokens, self.n_pages = ggml_type, rank, rope, page_tokens, n_pages
        self.width = rank + rope
        rows = (rng.standard_normal((n_pages, page_tokens, self.width)) * sigma).astype(np.float32)
        if ggml_type == mm.F16:
            h = rows.astype(np.float16)
            self.values = h.astype(np.float64)
            self.bytes = h.view(np.uint8).reshape(n_pages, -1).copy()
        else:
            q, d = q8_blocks(rows)
            self.values = (q.reshape(n_pages, page_tokens, -1, 32).astype(np.float64)
                           * d.astype(np.float64)[..., None]).reshape(rows.shape)
            self.bytes = np.concatenate([q.view(np.uint8).reshape(n_pages, -1),
                                         d.view(np.uint8).reshape(n_pages, -1)], 1).copy()

    def spoil(self, page, at):
        """NaN in the row's every value (codes at their largest with NaN scales)."""
        w = self.width
        if self.type == mm.F16:
            self.bytes[page].view(np.float16).reshape(self.page_tokens, w)[at] = np.nan
        else:
            self.bytes[page, at * w:(at + 1) * w] = 127
            s = self.bytes[page, self.page_tokens * w:].view(np.float16).reshape(self.page_tokens, w // 32)
            s[at] = np.nan


def attention64(q, q_pe, values, tables, rows, lens, page_tokens, scale, rank):
    """out, lse, and per row the largest |score| and sum of the scores' terms, in 64 bits. values [pages, page_tokens,
    width]; page numbers outside the pool are left out."""
    n, h, _ = q.shape
    out, lse = np.zeros((n, h, rank)), np.full((n, h), -np.inf)
    qq = np.concatenate([q, q_pe], -1).astype(np.float64) if q_pe is not None else q.astype(np.float64)
    for t in range(n):
        if rows[t] >= len(tables):
            continue
        length = min(int(lens[t]), tables.shape[1] * page_tokens)
        pos = np.arange(length)
        page = tables[rows[t]][pos // page_tokens]
        live = (page >= 0) & (page < len(values))
        if not live.any():
            continue
        k = values[page[live], (pos % page_tokens)[live]]
        s = qq[t] @ k.T * scale
        m = s.max(-1, keepdims=True)
        e = np.exp(s - m)
        z = e.sum(-1, keepdims=True)
        out[t] = e @ k[:, :rank] / z
        lse[t] = (m + np.log(z))[:, 0]
    return out, lse


def logprobs64(x):
    with np.errstate(invalid="ignore", over="ignore"):
        x = x.astype(np.float64)
        m = x.max(-1, keepdims=True)
        e = np.exp(x - m)
        z = e.sum(-1, keepdims=True)
        lp = (x - m) - np.log(z)
        p = e / z
        return lp, -np.where(p > 0, p * np.where(p > 0, lp, 0), np.where(np.isnan(p), np.nan, 0)).sum(-1)


def top_ids(x, k):
    """The k largest of each row, equal ones by the lower id, NaN after every number."""
    key = np.where(np.isnan(x), -np.inf, x.astype(np.float64) + 0.0)
    out = []
    for r in range(len(x)):
        out.append(np.lexsort((np.arange(x.shape[1]), -key[r], np.isnan(x[r])))[:k])
    return np.array(out, np.uint32).reshape(len(x), k)


class Buffers:
    """Device buffers of a test, freed with it."""

    def __init__(self, ctx):
        self.ctx, self.held = ctx, []

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        for b in self.held:
            b.free()

    def put(self, arr):
        b = mm.DeviceArray.from_numpy(self.ctx, np.ascontiguousarray(arr))
        self.held.append(b)
        return b

    def new(self, nbytes, fill=0xFF):
        """A buffer of bytes `fill` (0xFF: NaN in every float type here)."""
        return self.put(np.full(max(1, int(nbytes)), fill, np.uint8))


class At:
    """A place inside a device buffer."""

    def __init__(self, buf, offset, nbytes=None):
        self.buf, self.ptr = buf, buf.ptr + offset
        self.nbytes = buf.nbytes - offset if nbytes is None else nbytes


class Graph:
    """A captured sequence of calls on the context's stream (HIP runtime)."""

    def __init__(self, ctx, calls):
        self.hip = ctypes.CDLL("libamdhip64.so")
        self.stream, self.exec, graph = ctypes.c_void_p(ctx.stream), ctypes.c_void_p(), ctypes.c_void_p()
        self._ok(self.hip.hipStreamBeginCapture(self.stream, 2))  # hipStreamCaptureModeRelaxed
        try:
            calls()
        finally:
            rc = self.hip.hipStreamEndCapture(self.stream, ctypes.byref(graph))
        self._ok(rc)
        self._ok(self.hip.hipGraphInstantiate(ctypes.byref(self.exec), graph, None, None, 0))
        self._ok(self.hip.hipGraphDestroy(graph))

    def _ok(self, rc):
        assert rc == 0, f"HIP error {rc}"

    def replay(self):
        self._ok(self.hip.hipGraphLaunch(self.exec, self.stream))

    def free(self):
        self._ok(self.hip.hipGraphExecDestroy(self.exec))
