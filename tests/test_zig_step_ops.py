"""The Zig wrappers of the operators between a decode step's products: each C
function can be called through HipBackend with every argument of its own (the
externs themselves are not public), and the struct fields that the integration
guide's snippets name exist. Read from the sources: the image has no Zig
compiler."""
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ZIG = open(os.path.join(ROOT, "mobile-moe.zig_amd", "zig", "hip_backend.zig")).read()
GUIDE = open(os.path.join(ROOT, "INTEGRATION.md")).read()

FUNCTIONS = ["rms_norm_dev", "rope_create", "rope_destroy", "rope_frequencies", "rope_dev", "kv_page_bytes", "kv_store_dev",
             "mla_attention_workspace", "mla_attention_dev", "logprobs_workspace", "logprobs_dev"]


def arguments(text):
    out, depth, cur = [], 0, ""
    for ch in text:
        depth += ch in "([{"
        depth -= ch in ")]}"
        if ch == "," and depth == 0:
            out.append(cur.strip())
            cur = ""
        else:
            cur += ch
    return out + ([cur.strip()] if cur.strip() else [])


def calls(name):
    """(the public function's own parameters, the arguments passed on) of every call in one."""
    for m in re.finditer(r"pub fn (\w+)\((.*?)\) [^{]*\{(.*?)\n    \}", ZIG, flags=re.S):
        params = [p.split(":")[0].strip() for p in arguments(m.group(2))]
        for c in re.finditer(r"\b" + name + r"\((.*?)\)\)?;", m.group(3), flags=re.S):
            yield params, arguments(c.group(1))


@pytest.mark.parametrize("name", FUNCTIONS)
def test_every_argument_can_be_given(name):
    m = re.search(r"^extern fn mmhip_" + name + r"\((.*?)\)", ZIG, flags=re.M)
    n = len(arguments(m.group(1)))
    found = False
    for params, args in calls("mmhip_" + name):
        assert len(args) == n
        own = [re.sub(r"^&", "", a) for a in args if a not in ("self.ctx", "&h")]  # &h: the wrapper's result
        found |= all(a in params for a in own) and len(set(own)) == len(own)
    assert found, f"no wrapper passes every argument of mmhip_{name} on"


def test_snippets_name_fields_that_exist():
    alias = dict(re.findall(r"^pub const (\w+) = (mmhip_\w+);", ZIG, flags=re.M))
    seen = 0
    for name, body in re.findall(r"\b(\w+)\{([^{}]*)\}", GUIDE, flags=re.S):
        if name not in alias and not name.startswith("mmhip_"):
            continue
        struct = re.search(r"pub const " + alias.get(name, name) + r" = extern struct \{(.*?)\};", ZIG, flags=re.S)
        fields = set(re.findall(r"^\s*(\w+):", struct.group(1), flags=re.M))
        for f in re.findall(r"\.(\w+)\s*=", body):
            assert f in fields, (name, f)
            seen += 1
    assert seen
