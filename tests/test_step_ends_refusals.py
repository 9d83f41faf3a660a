"""What the operators at a decode step's two ends refuse, without a device:
arguments are checked before the context, so every refusal is met with a null
context and pointers that are never followed; a call that passes all the checks
ends at the null context. The binding refuses freed optional buffers, and the Zig
wrappers pass every argument on."""
import ctypes
import math
import os
import re

import pytest

import mmhip as mm
from test_zig_step_ops import ZIG, arguments, calls

P = 0x1000  # an address that passes for a buffer; nothing reads it


def refused(rc, code, *words):
    msg = mm.load_library().mmhip_last_error().decode()
    assert rc == code, (rc, msg)
    for w in words:
        assert w in msg, (w, msg)


def embed(**kw):
    a = dict(y=P, ys=64, table=P, type=mm.Q8_0, rows=10, cols=64, tokens=P, n=3, scale=1.0)
    a.update(kw)
    return mm.load_library().mmhip_embed_dev(None, a["y"], a["ys"], a["table"], a["type"], a["rows"], a["cols"], a["tokens"],
                                             a["n"], a["scale"])


def test_embed():
    for ok in (dict(), dict(n=0), dict(type=mm.F16, cols=63), dict(type=mm.Q8_0, cols=33), dict(n=1, ys=0), dict(table=P + 2),
               dict(scale=math.inf), dict(rows=0xFFFFFFFF)):
        refused(embed(**ok), mm.ERR_INVALID, "embed: null context")
    for t in (3, 12, 99):
        refused(embed(type=t), mm.ERR_UNSUPPORTED, "type")
    for bad in (dict(y=None), dict(table=None), dict(tokens=None), dict(ys=63), dict(cols=0), dict(cols=2 ** 31), dict(rows=0),
                dict(rows=2 ** 32), dict(n=2 ** 24), dict(n=2 ** 23, cols=4096, ys=4096), dict(type=mm.Q4_0, cols=48),
                dict(type=mm.IQ4_NL, cols=33), dict(type=mm.IQ2_XXS, cols=128), dict(y=P + 2), dict(tokens=P + 1), dict(table=P + 1),
                dict(type=mm.F32, table=P + 2)):
        refused(embed(**bad), mm.ERR_INVALID, "embed")
        assert "null context" not in mm.load_library().mmhip_last_error().decode(), bad


def plan(**kw):
    a = mm.KvPlan()
    for k in ("lens", "new", "next_lens", "tables", "free", "free_count", "next_free_count", "positions", "slots", "table_of", "seen",
              "firsts", "granted", "workspace"):
        setattr(a, k + "_dev", P)
    a.n_requests, a.page_tokens, a.n_pages, a.table_pages, a.table_stride, a.max_tokens, a.workspace_bytes = 4, 16, 100, 8, 8, 10, 1 << 20
    for k, v in kw.items():
        setattr(a, k, v)
    return mm.load_library().mmhip_kv_plan_dev(None, ctypes.byref(a))


def test_plan():
    for ok in (dict(), dict(n_requests=0, lens_dev=None, tables_dev=None), dict(max_tokens=0, slots_dev=None, seen_dev=None),
               dict(release_dev=P, shared_dev=P, last_dev=P), dict(n_requests=1, table_stride=0), dict(page_tokens=1024),
               dict(next_lens_dev=P, lens_dev=P)):
        refused(plan(**ok), mm.ERR_INVALID, "kv_plan: null context")
    for bad in (dict(page_tokens=8), dict(page_tokens=17), dict(page_tokens=2048), dict(page_tokens=0), dict(n_pages=0),
                dict(n_pages=2 ** 27), dict(n_requests=2 ** 24), dict(table_pages=0), dict(table_stride=7), dict(table_pages=2 ** 28, table_stride=2 ** 28),
                dict(max_tokens=2 ** 31), dict(shared_dev=P), dict(firsts_dev=None), dict(free_dev=None), dict(free_count_dev=None),
                dict(next_free_count_dev=None), dict(lens_dev=None), dict(new_dev=None), dict(next_lens_dev=None), dict(tables_dev=None),
                dict(granted_dev=None), dict(positions_dev=None), dict(slots_dev=None), dict(table_of_dev=None), dict(seen_dev=None),
                dict(lens_dev=P + 1), dict(tables_dev=P + 2), dict(last_dev=P + 3), dict(release_dev=P + 2)):
        refused(plan(**bad), mm.ERR_INVALID, "kv_plan")
        assert "null context" not in mm.load_library().mmhip_last_error().decode(), bad
    refused(mm.load_library().mmhip_kv_plan_dev(None, None), mm.ERR_INVALID, "null arguments")


def sample(**kw):
    a = mm.Sample()
    a.logits_dev, a.uniform_dev, a.tokens_dev, a.workspace_dev, a.workspace_bytes = P, P, P, P, 1 << 30
    a.stride, a.n_rows, a.vocab = 100, 2, 100
    for k, v in kw.items():
        setattr(a, k, v)
    return mm.load_library().mmhip_sample_dev(None, ctypes.byref(a))


def test_sample():
    for ok in (dict(), dict(n_rows=0), dict(n_rows=1, stride=0), dict(rows_dev=P, n_logits=1, stride=0), dict(vocab=1 << 24, stride=1 << 24),
               dict(temperature_dev=P, top_k_dev=P, top_p_dev=P, min_p_dev=P, probs_dev=P, kept_dev=P)):
        refused(sample(**ok), mm.ERR_INVALID, "sample: null context")
    for bad in (dict(vocab=0), dict(vocab=(1 << 24) + 1, stride=1 << 25), dict(n_rows=2 ** 22), dict(stride=99), dict(logits_dev=None), dict(uniform_dev=None),
                dict(tokens_dev=None), dict(rows_dev=P), dict(rows_dev=P, n_logits=2, stride=99), dict(rows_dev=P, n_logits=0xFFFFFFFF),
                dict(logits_dev=P + 2), dict(tokens_dev=P + 1), dict(probs_dev=P + 3), dict(top_k_dev=P + 2)):
        refused(sample(**bad), mm.ERR_INVALID, "sample")
        assert "null context" not in mm.load_library().mmhip_last_error().decode(), bad
    refused(mm.load_library().mmhip_sample_dev(None, None), mm.ERR_INVALID, "null arguments")


def test_workspaces_without_a_context():
    lib = mm.load_library()
    assert lib.mmhip_kv_plan_workspace(None, 5) == 0 and lib.mmhip_sample_workspace(None, 5, 100) == 0


class Buf:
    def __init__(self, ptr=P):
        self.ptr, self.nbytes = ptr, 1 << 20


def test_freed_optional_buffers():
    c = mm.Context.__new__(mm.Context)
    c.lib, c.handle = mm.load_library(), None
    b, gone = Buf(), Buf(None)
    kw = dict(logits=b, n_rows=1, vocab=9, uniform=b, tokens=b)
    with pytest.raises(mm.MmhipError, match="null context"):
        c.sample_dev(c.sample_args(**kw))
    for k in ("workspace", "rows", "temperature", "top_k", "top_p", "min_p", "probs", "kept"):
        with pytest.raises(mm.MmhipError, match="freed"):
            c.sample_args(**dict(kw, **{k: gone}))
    kw = {k: b for k in ("lens", "new", "next_lens", "tables", "free", "free_count", "next_free_count", "positions", "slots",
                         "table_of", "seen", "firsts", "granted", "workspace")}
    kw.update(n_requests=1, table_pages=1, page_tokens=16, n_pages=1, max_tokens=1)
    with pytest.raises(mm.MmhipError, match="null context"):
        c.kv_plan_dev(c.kv_plan_args(**kw))
    for k in ("release", "shared", "last"):
        with pytest.raises(mm.MmhipError, match="freed"):
            c.kv_plan_args(**dict(kw, **{k: gone}))


@pytest.mark.parametrize("name", ["embed_dev", "kv_plan_workspace", "kv_plan_dev", "sample_workspace", "sample_dev"])
def test_every_argument_can_be_given_in_zig(name):
    m = re.search(r"^extern fn mmhip_" + name + r"\((.*?)\)", ZIG, flags=re.M)
    n, found = len(arguments(m.group(1))), False
    for params, args in calls("mmhip_" + name):
        assert len(args) == n
        own = [a for a in args if a != "self.ctx"]
        found |= all(a in params for a in own) and len(set(own)) == len(own)
    assert found


def test_files_with_4bit_tensors(tmp_path):
    """Their bytes are found and bounded."""
    import gguf_writer as gw
    import numpy as np
    path = os.path.join(tmp_path, "f.gguf")
    raw = mm.make_weight(np.random.default_rng(1), mm.Q4_0, 3, 64)
    gw.write(path, [], [("a", [64, 3], mm.Q4_0, raw), ("b", [32, 1], mm.IQ4_NL, raw[:18]), ("c", [64, 4], mm.IQ4_NL, raw)])
    with mm.Gguf(path) as g:
        assert g.tensor("a")["n_bytes"] == 108 and g.tensor("b")["n_bytes"] == 18
        assert g.tensor("a")["data"] and g.tensor("b")["data"] and not g.tensor("c")["data"]  # c's bytes leave the file
