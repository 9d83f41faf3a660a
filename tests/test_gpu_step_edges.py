"""The operators between a decode step's products where their numbers or their
dispatch can go wrong: infinite cached values, block scales of all sizes, the
precision of the operands, large finite queries, every kernel the attention can
take. Against the plain 64-bit forms of tests/step_reference.py; u = 2^-24, half a
step of f32."""
import numpy as np
import pytest

import mmhip as mm
import step_reference as ref
from step_reference import Buffers, Pool, U
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
