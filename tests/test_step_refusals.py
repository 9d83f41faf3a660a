"""What the operators between a decode step's products refuse, without a
device: arguments are checked before the context, so every refusal is met with
a null context and pointers that are never followed; a call that passes all the
checks ends at the null context. And the indexes that the kernels form from
device data (page tables, slots, lengths), from the same header in a host
program: none leaves the pool."""
import ctypes
import math
import os
import shutil
import subprocess

import numpy as np
import pytest

import mmhip as mm
import step_reference as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 0x1000  # an address that passes for a buffer; nothing reads it
P2, P3, P4 = 0x20000, 0x30000, 0x40000


def refused(rc, code, *words):
    msg = mm.load_library().mmhip_last_error().decode()
    assert rc == code, (rc, msg)
    for w in words:
        assert w in msg, (w, msg)


def norm(**kw):
    a = dict(y=P, y_type=mm.F32, ys=64, sum=None, ss=64, x=P2, xs=64, res=None, rs=64, w=P3, n=2, cols=64, eps=1e-5)
    a.update(kw)
    return mm.load_library().mmhip_rms_norm_dev(None, a["y"], a["y_type"], a["ys"], a["sum"], a["ss"], a["x"], a["xs"],
                                                a["res"], a["rs"], a["w"], a["n"], a["cols"], a["eps"])


def test_norm():
    refused(norm(), mm.ERR_INVALID, "null context")
    refused(norm(n=0), mm.ERR_INVALID, "null context")
    refused(norm(y_type=16), mm.ERR_UNSUPPORTED, "y_type")
    for bad in (dict(cols=0), dict(cols=2 ** 31), dict(eps=-1.0), dict(eps=math.nan), dict(n=2 ** 31), dict(y=None),
                dict(x=None), dict(w=None), dict(xs=63), dict(ys=63), dict(y_type=mm.F16, ys=63),
                dict(res=P4, rs=63), dict(sum=P4, ss=63), dict(y=P + 2), dict(y=P + 1, y_type=mm.Q8_0), dict(x=P2 + 2),
                dict(w=P3 + 1), dict(sum=P4 + 2), dict(res=P4 + 3)):
        refused(norm(**bad), mm.ERR_INVALID, "rms_norm")
        assert "null context" not in mm.load_library().mmhip_last_error().decode(), bad
    # outputs on inputs: the same values at the same places only
    refused(norm(y=P2), mm.ERR_INVALID, "null context")
    refused(norm(y=P2, ys=96), mm.ERR_INVALID, "its stride")
    refused(norm(y=P2, y_type=mm.F16), mm.ERR_INVALID, "f32")
    refused(norm(y=P4, res=P4, y_type=mm.Q8_0), mm.ERR_INVALID, "f32")
    refused(norm(sum=P4, res=P4), mm.ERR_INVALID, "null context")
    refused(norm(sum=P4, res=P4, ss=96), mm.ERR_INVALID, "its stride")
    refused(norm(sum=P), mm.ERR_INVALID, "same buffer")
    refused(norm(y_type=mm.Q8_0, ys=0), mm.ERR_INVALID, "null context")  # blocks have no stride


def rope(**kw):
    p = mm.rope_params(64, base=1e4)
    for k, v in kw.items():
        setattr(p, k, v)
    h = ctypes.c_void_p()
    return mm.load_library().mmhip_rope_create(None, ctypes.byref(p), ctypes.byref(h))


def test_rope_create():
    refused(rope(), mm.ERR_INVALID, "null context")
    yarn = dict(scaling=2, factor=16.0, original_context=4096)
    refused(rope(**yarn), mm.ERR_INVALID, "null context")
    for bad in (dict(dims=0), dict(dims=63), dict(dims=258), dict(layout=2), dict(scaling=3), dict(base=1.0),
                dict(base=math.inf), dict(base=math.nan), dict(magnitude=math.inf), dict(scaling=1, factor=0.0),
                dict(scaling=1, factor=math.nan), dict(yarn, original_context=0), dict(yarn, beta_fast=0.0),
                dict(yarn, beta_slow=-1.0), dict(yarn, factor=math.inf)):
        refused(rope(**bad), mm.ERR_INVALID, "rope_create")
        assert "null context" not in mm.load_library().mmhip_last_error().decode(), bad
    lib = mm.load_library()
    assert lib.mmhip_rope_create(None, None, None) == mm.ERR_INVALID
    refused(lib.mmhip_rope_dev(None, None, P, 64, 64, P2, 64, 64, P3, 1, 1, 64, 0), mm.ERR_INVALID, "null rope")


@pytest.mark.parametrize("kw", [dict(dims=64, base=1e6), dict(dims=2, base=1e4), dict(dims=256, base=500000.0),
                                dict(dims=64, base=1e4, scaling="linear", factor=4.0),
                                dict(dims=64, base=1e6, scaling="yarn", factor=16.0, original_context=8192),
                                dict(dims=128, base=1e4, scaling="yarn", factor=2.5, original_context=100),
                                dict(dims=64, base=1e4, scaling="yarn", factor=8.0, original_context=4096,
                                     beta_fast=1.0, beta_slow=1.0)])
def test_rope_frequencies(kw):
    """Against the formulas in 64 bits; a ramp of no width (low = high) is a step."""
    p = mm.rope_params(**kw)
    f, m = mm.rope_frequencies(p)
    kw = dict(kw, base=float(np.float32(kw["base"])), factor=float(np.float32(kw.get("factor", 1.0))))
    np.testing.assert_allclose(f, ref.frequencies64(**kw), rtol=1e-14)
    assert m == (0.1 * math.log(kw["factor"]) + 1 if kw.get("scaling") == "yarn" else 1.0)
    p.magnitude = 0.5
    assert mm.rope_frequencies(p)[1] == 0.5


def cache(**kw):
    a = dict(pool=P, type=mm.F16, rank=512, rope=64, pt=16, n=4)
    a.update(kw)
    return mm.KvCacheDesc(a["pool"], a["type"], a["rank"], a["rope"], a["pt"], a["n"])


BAD_CACHES = [dict(rank=0), dict(rank=500), dict(rank=544), dict(rope=16), dict(rope=96), dict(pt=8), dict(pt=24),
              dict(pt=2048), dict(pt=0), dict(n=0), dict(n=2 ** 27)]


def test_cache_sizes():
    lib = mm.load_library()
    for t, row in ((mm.F16, 1152), (mm.Q8_0, 612)):
        assert mm.KvCache.page_bytes(t, 512, 64, 16) == 16 * row
        assert mm.KvCache.page_bytes(t, 512, 64, 1024) == 1024 * row
    assert mm.KvCache.page_bytes(mm.Q8_0, 32, 0, 16) == 16 * 34
    assert mm.KvCache.page_bytes(mm.F32, 512, 64, 16) == 0
    for bad in BAD_CACHES:
        assert lib.mmhip_kv_page_bytes(ctypes.byref(cache(**bad))) == 0, bad
    assert lib.mmhip_kv_page_bytes(None) == 0


def store(c=None, kv=P2, stride=576, w=P3, eps=1e-5, rope=None, pos=None, slots=P4, n=3):
    c = cache() if c is None else c
    return mm.load_library().mmhip_kv_store_dev(None, ctypes.byref(c), kv, stride, w, eps, rope, pos, slots, n)


def test_store():
    refused(store(), mm.ERR_INVALID, "null context")
    refused(store(n=1, stride=0), mm.ERR_INVALID, "null context")  # one row has no stride
    refused(store(w=None, eps=-1.0), mm.ERR_INVALID, "null context")  # eps belongs to the norm
    refused(store(c=cache(type=mm.F32)), mm.ERR_UNSUPPORTED, "F16 or Q8_0")
    for bad in [dict(c=cache(**b)) for b in BAD_CACHES] + [
            dict(c=cache(pool=None)), dict(c=cache(pool=P + 8)), dict(kv=None), dict(slots=None), dict(stride=575),
            dict(eps=-1.0), dict(n=2 ** 31), dict(kv=P2 + 1), dict(slots=P4 + 2), dict(w=P3 + 2)]:
        refused(store(**bad), mm.ERR_INVALID, "kv_store")
        assert "null context" not in mm.load_library().mmhip_last_error().decode(), bad


def attention(c=None, **kw):
    a = mm.MlaAttention()
    a.cache = cache() if c is None else c
    f = dict(q_dev=P, q_pe_dev=P, out_dev=P2, lse_dev=None, q_token_stride=20 * 512, q_head_stride=512,
             q_pe_token_stride=20 * 64, q_pe_head_stride=64, out_token_stride=20 * 512, out_head_stride=512,
             tables_dev=P3, table_stride=4, n_tables=2, table_pages=4, table_of_dev=None, lens_dev=P4, n_tokens=2,
             n_heads=20, scale=0.07, workspace_dev=P, workspace_bytes=0)
    f.update(kw)
    for k, v in f.items():
        setattr(a, k, v)
    return mm.load_library().mmhip_mla_attention_dev(None, ctypes.byref(a))


def test_attention():
    refused(attention(), mm.ERR_INVALID, "null context")
    refused(attention(n_tokens=0), mm.ERR_INVALID, "null context")
    refused(attention(c=cache(rope=0), q_pe_dev=None, q_pe_head_stride=0), mm.ERR_INVALID, "null context")
    refused(attention(n_tokens=1, n_heads=1, q_token_stride=0, q_head_stride=0, out_token_stride=0, out_head_stride=0),
            mm.ERR_INVALID, "null context")
    refused(attention(c=cache(type=mm.IQ2_XXS)), mm.ERR_UNSUPPORTED, "F16 or Q8_0")
    assert mm.load_library().mmhip_mla_attention_dev(None, None) == mm.ERR_INVALID
    for bad in [dict(c=cache(**b)) for b in BAD_CACHES] + [
            dict(c=cache(pool=P + 4)), dict(q_dev=None), dict(q_pe_dev=None), dict(out_dev=None), dict(tables_dev=None),
            dict(lens_dev=None), dict(n_heads=0), dict(n_tables=0), dict(table_pages=0), dict(table_stride=3),
            dict(scale=math.nan), dict(scale=math.inf), dict(q_head_stride=511), dict(q_pe_head_stride=63),
            dict(out_head_stride=511), dict(q_token_stride=100), dict(q_pe_token_stride=10), dict(out_token_stride=20 * 512 - 1),
            dict(n_tokens=2 ** 31 - 1), dict(table_pages=2 ** 28, table_stride=2 ** 28), dict(q_dev=P + 2),
            dict(out_dev=P + 1), dict(tables_dev=P + 2), dict(lens_dev=P + 1), dict(lse_dev=P + 2),
            dict(table_of_dev=P + 3)]:
        refused(attention(**bad), mm.ERR_INVALID, "attention")
        assert "null context" not in mm.load_library().mmhip_last_error().decode(), bad


def logprobs(logits=P, stride=100, n=2, vocab=100, tokens=P2, given=1, out=P3, entropy=None, top=3, ids=P4, tlp=None,
             ws=None, wb=0):
    return mm.load_library().mmhip_logprobs_dev(None, logits, stride, n, vocab, tokens, given, out, entropy, top, ids,
                                                tlp, ws, wb)


def test_logprobs():
    refused(logprobs(), mm.ERR_INVALID, "null context")
    refused(logprobs(given=0, tokens=None, out=None, top=0, ids=None), mm.ERR_INVALID, "null context")
    refused(logprobs(n=1, stride=0), mm.ERR_INVALID, "null context")
    for bad in (dict(logits=None), dict(tokens=None), dict(out=None), dict(ids=None), dict(vocab=0, stride=0),
                dict(vocab=2 ** 31, stride=2 ** 31), dict(top=33), dict(vocab=2), dict(stride=99), dict(n=2 ** 31),
                dict(given=2 ** 31), dict(logits=P + 2), dict(tokens=P + 1), dict(entropy=P + 2), dict(tlp=P + 3)):
        refused(logprobs(**bad), mm.ERR_INVALID, "logprobs")
        assert "null context" not in mm.load_library().mmhip_last_error().decode(), bad


def test_most_rows():
    """Calls of 2^24 rows or tokens are refused, of one less not."""
    for call in (norm, store, logprobs):
        refused(call(n=1 << 24), mm.ERR_INVALID, "2^24")
        refused(call(n=(1 << 24) - 1), mm.ERR_INVALID, "null context")


def test_workspaces_without_a_context():
    lib = mm.load_library()
    assert lib.mmhip_mla_attention_workspace(None, 1, 1, 512) == 0
    assert lib.mmhip_logprobs_workspace(None, 1, 100, 5) == 0


_HARNESS = r"""
#include "paged.hpp"
#include <cstdio>
#include <cstdlib>
#include <initializer_list>
using namespace mmhip;
#define CHECK(x) do { if (!(x)) { printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)
int main() {
    for (uint32_t q8 = 0; q8 < 2; ++q8)
        for (uint32_t shift = 4; shift <= 10; ++shift)
            for (uint32_t width : {32u, 96u, 576u})
                for (uint32_t n_pages : {1u, 3u, 77u, (1u << (31 - shift)) - 1}) {
                    PagedGeom g{width, width - (width > 32 ? 32 : 0), shift, n_pages, q8, 0};
                    g.page_bytes = paged_page_bytes(q8, width, 1u << shift);
                    const uint64_t pool = g.page_bytes * n_pages;
                    const int64_t rows = (int64_t)n_pages << shift;
                    CHECK(g.page_bytes % 16 == 0);
                    const int64_t slots[] = {0, 1, rows - 1, rows / 2, rows, rows + 1, -1, -2147483647 - 1, 2147483647};
                    for (int64_t s : slots) {
                        uint32_t page, at;
                        const bool ok = paged_slot(g, (int32_t)s, page, at);
                        CHECK(ok == (s >= 0 && s < rows));
                        if (!ok) continue;
                        CHECK(paged_row(g, page, at) + (q8 ? width : 2 * width) <= (q8 ? paged_scales(g, page, 0) : pool));
                        CHECK(paged_row(g, page, at) % (q8 ? 32 : 64) == page * g.page_bytes % (q8 ? 32 : 64));
                        if (q8) CHECK(paged_scales(g, page, at) + width / 32 * 2 <= (page + 1) * g.page_bytes);
                        if (q8) CHECK(paged_scales(g, page, at) >= page * g.page_bytes + ((uint64_t)width << shift));
                    }
                    const int32_t ids[] = {0, (int32_t)n_pages - 1, (int32_t)n_pages, -1, -2147483647 - 1, 2147483647};
                    for (int32_t id : ids) CHECK(paged_has(g, id) == (id >= 0 && (uint32_t)id < n_pages));
                    uint32_t bad;
                    for (uint32_t table_pages : {1u, 5u, 0xFFFFFFFFu >> shift}) {
                        const uint64_t most = (uint64_t)table_pages << shift;
                        for (uint32_t len : {0u, 1u, 16u, 80u, 0x7FFFFFFFu, 0xFFFFFFFFu}) {
                            const uint32_t seen = paged_seen(g, len, 1, 2, table_pages, bad);
                            CHECK(seen == (len > most ? most : len) && bad == (len > most ? 2u : 0u));
                            CHECK(seen == 0 || ((uint64_t)(seen - 1) >> shift) < table_pages);
                        }
                        CHECK(paged_seen(g, 7, 2, 2, table_pages, bad) == 0 && bad == 1);
                        CHECK(paged_seen(g, 7, 0xFFFFFFFFu, 2, table_pages, bad) == 0 && bad == 1);
                    }
                }
    return 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not available")
def test_no_index_leaves_the_pool(tmp_path):
    src, exe = tmp_path / "paged.cpp", tmp_path / "paged"
    src.write_text(_HARNESS)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover", "-I",
                    os.path.join(ROOT, "mobile-moe.zig_amd", "csrc", "kernels"), str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
