"""Page plans that meet a wrong length in a row that is over: what is reported, and what happens."""
import numpy as np
import pytest

import mmhip as mm
from step_reference import Buffers
from test_gpu_step_ends import Planner

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,max_tokens", [(6, 60), (1500, 9000)])
def test_a_released_length_beyond_its_table(ctx, n, max_tokens):
    """Its table's four pages come back, its row's new tokens are granted, and the report says that the length was cut."""
    pt, tp, n_pages = 16, 4, 20
    lens, new, release = (np.zeros(n, np.uint32) for _ in range(3))
    lens[:2], new[:2], release[0] = (500, 500), (20, 1), 1
    tables = np.zeros((n, tp), np.int32)
    tables[0] = [10, 11, 12, 13]
    with Buffers(ctx) as d:
        p = Planner(ctx, d, n=n, table_pages=tp, pt=pt, n_pages=n_pages, max_tokens=max_tokens)
        p.set(lens, new, release, np.zeros(n), tables, np.arange(n_pages), 3)
        ctx.kv_plan_dev(p.args)
        with pytest.raises(mm.MmhipError, match="a released one cut there, otherwise its request got nothing"):
            ctx.synchronize()
        ctx.synchronize()
        g = p.get()
    assert g["granted"][:2].tolist() == [1, 0] and g["next_lens"][:2].tolist() == [20, 500] and g["next_free"].tolist() == [5]
    assert g["slots"][:20].tolist() == [13 * 16 + i for i in range(16)] + [12 * 16 + i for i in range(4)]
    assert (g["slots"][20:] == -1).all()
