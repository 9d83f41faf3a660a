"""The binding's optional arguments: a buffer or rotary plan that was freed is
refused, not taken as left out (which would store unrotated rows, norm without the
residual, or read other page tables). No device: a call that is passed on ends
at the null context."""
import pytest

import mmhip as mm


class Buf:
    def __init__(self, ptr=0x10000):
        self.ptr, self.nbytes = ptr, 1 << 20


@pytest.fixture
def ctx():
    c = mm.Context.__new__(mm.Context)
    c.lib, c.handle = mm.load_library(), None
    return c


def plan(handle):
    r = mm.Rope.__new__(mm.Rope)
    r.handle = handle
    return r


GONE = Buf(None)


def refused(call, word):
    with pytest.raises(mm.MmhipError, match=word) as e:
        call()
    assert e.value.code == mm.ERR_INVALID


def test_freed_arguments(ctx):
    b, c = Buf(), Buf(0x40000)
    refused(lambda: ctx.rms_norm_dev(b, c, c, 1, 64), "null context")
    refused(lambda: ctx.rms_norm_dev(b, c, c, 1, 64, residual=GONE), "freed")
    refused(lambda: ctx.rms_norm_dev(b, c, c, 1, 64, sum_out=GONE), "freed")
    cache = mm.KvCache(b, mm.F16, rank=512, rope_dims=64, page_tokens=16, n_pages=4)
    refused(lambda: ctx.kv_store_dev(cache, c, c, 1), "null context")
    for kw in (dict(norm_weight=GONE), dict(positions=GONE), dict(rope=plan(None), positions=c)):
        refused(lambda: ctx.kv_store_dev(cache, c, c, 1, **kw), "freed")
    refused(lambda: ctx.logprobs_dev(b, 1, 100, entropy=c, workspace=c), "null context")
    for k in ("tokens", "token_logprobs", "entropy", "top_ids", "top_logprobs", "workspace"):
        refused(lambda: ctx.logprobs_dev(b, 1, 100, **{k: GONE}), "freed")
    kw = dict(q=b, q_pe=b, out=c, lens=c, tables=c, n_tables=1, table_pages=1, n_tokens=1, n_heads=1, scale=1.0, workspace=c)
    refused(lambda: ctx.mla_attention_dev(ctx.mla_attention_args(cache, **kw)), "null context")
    for k in ("q_pe", "lse", "table_of"):
        refused(lambda: ctx.mla_attention_args(cache, **dict(kw, **{k: GONE})), "freed")


def test_freed_pool(ctx):
    b, c = Buf(), Buf(0x40000)
    cache = mm.KvCache(b, mm.F16, rank=512, rope_dims=64, page_tokens=16, n_pages=4)
    b.ptr = None
    refused(lambda: ctx.kv_store_dev(cache, c, c, 1), "freed")
    refused(lambda: ctx.mla_attention_args(cache, q=c, q_pe=c, out=c, lens=c, tables=c, n_tables=1, table_pages=1, n_tokens=1,
                                           n_heads=1, scale=1.0, workspace=c), "freed")
