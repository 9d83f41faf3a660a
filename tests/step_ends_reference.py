"""Plain 64-bit forms of what stands at a decode step's two ends, for the tests:
4-bit blocks, page plans made request by request, and sampling by sorting."""
import numpy as np

import mmhip as mm

IQ4_VALUES = np.array([-127, -104, -83, -65, -49, -35, -22, -10, 1, 13, 25, 38, 53, 69, 89, 113], np.float64)


def values_4bit(raw, ggml_type):
    """Raw blocks -> their weights [blocks, 32] in 64 bits (exact: f16 times a small integer)."""
    b = np.asarray(raw, np.uint8).reshape(-1, 18)
    with np.errstate(invalid="ignore"):
        d = b[:, :2].copy().view(np.float16).astype(np.float64)
        codes = np.concatenate([b[:, 2:] & 15, b[:, 2:] >> 4], 1)
        return (codes.astype(np.float64) - 8 if ggml_type == mm.Q4_0 else IQ4_VALUES[codes]) * d


def plan(lens, new, tables, free, free_count, *, page_tokens, n_pages, max_tokens, release=None, shared=None):
    """The formula's results, one request after the other, as the header words it. Valid inputs only."""
    lens, tables, free, P = [int(v) for v in lens], tables.copy(), free.copy(), page_tokens
    n, top, capacity = len(lens), int(free_count), tables.shape[1] * page_tokens
    for r in range(n):
        if release is not None and release[r]:
            held = -(-lens[r] // P)
            for i in range(min(int(shared[r]), held) if shared is not None else 0, held):
                free[top] = tables[r, i]
                top += 1
            lens[r] = 0
    stack, asked, wanted = top, 0, 0
    firsts, granted, last, pos, slots, of = [0], [], [], [], [], []
    for r in range(n):
        add = int(new[r])
        ok = add > 0 and lens[r] + add <= capacity
        if ok:
            asked += add
            ok = asked <= max_tokens
        if ok:
            held, need = -(-lens[r] // P), -(-(lens[r] + add) // P) - -(-lens[r] // P)
            wanted += need
            ok = need == 0 or wanted <= stack
        if ok:
            for i in range(held, held + need):
                top -= 1
                tables[r, i] = free[top]
            for p in range(lens[r], lens[r] + add):
                pos.append(p)
                slots.append(tables[r, p // P] * P + p % P)
                of.append(r)
            lens[r] += add
        granted.append(int(ok))
        last.append(len(pos) - 1 if ok else mm.NO_TOKEN)
        firsts.append(len(pos))
    pad = max_tokens - len(pos)
    return dict(positions=pos + [0] * pad, slots=slots + [-1] * pad, table_of=of + [0] * pad,
                seen=[p + 1 for p in pos] + [0] * pad, firsts=firsts, granted=granted, last=last, next_lens=lens,
                tables=tables, free=free, next_free=[top])


def sample(x, t, k, p, least, u):
    """(token, probability, kept) of one row of logits."""
    x = np.asarray(x, np.float32).astype(np.float64)
    ids = np.flatnonzero(x > -np.inf)
    if len(ids) == 0:
        return mm.NO_TOKEN, np.nan, 0
    ids = ids[np.argsort(-x[ids], kind="stable")]
    if t == 0:
        return ids[0], 1.0, 1
    z = np.where(x[ids] == x[ids[0]], 0.0, (x[ids] - (0.0 if np.isinf(x[ids[0]]) else x[ids[0]])) / t)
    if np.isinf(x[ids[0]]):
        z[x[ids] < np.inf] = -np.inf
    w = np.exp(z)
    n = min(int(k), len(ids)) if k else len(ids)
    if p < 1:
        before = np.cumsum(w[:n]) - w[:n]
        n = max(1, int((before < p * w[:n].sum()).sum()))
    n = min(n, int((w >= least).sum()))
    ids, order = np.sort(ids[:n]), np.argsort(ids[:n], kind="stable")
    w = w[:n][order]
    at = int((np.cumsum(w) <= u * np.cumsum(w)[-1]).sum())
    return ids[at], w[at] / w.sum(), n
