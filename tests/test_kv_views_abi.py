"""CPU checks of the entry points for windows, drafts and rules on logits that need no
device: the rules' layout, a null context."""
import ctypes as C
import os
import re

import pytest


@pytest.fixture(scope="module")
def L():
    from goneuron_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        from goneuron_amd import build
        build.build()
    return _lib.lib()


def test_rules_are_laid_out_as_declared():
    from goneuron_amd._lib import LogitRules
    header = open(os.path.join(os.path.dirname(__file__), "..", "include", "goneuron_hip.h")).read()
    body = re.search(r"typedef struct gn_logit_rules \{(.*?)\} gn_logit_rules;", header, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    declared = []
    for line in body.split(";"):
        m = re.match(r"\s*(const \w+|\w+)\s+(.*)", line, re.S)
        if m:
            for name in m.group(2).split(","):
                name = name.strip()
                kind = C.c_void_p if name.startswith("*") else {"int64_t": C.c_int64, "int32_t": C.c_int32}[m.group(1)]
                declared.append((name.lstrip("*"), kind))
    assert declared == LogitRules._fields_ and C.sizeof(LogitRules) == 120


def test_null_context(L):
    assert L.gn_kv_attention_window(None, None, None, None, 0, 0, None, None, 1, 1, 1, 1, 1, 1.0, 0, 1, 0, None, None) == -1
    assert L.gn_kv_attention_tree(None, None, None, None, 0, 0, None, 0, None, None, 1, 1, 1, 1, 1, 1.0, 0, None, None) == -1
    assert L.gn_kv_append_at(None, None, *[None] * 4, 0, 0, 0, 0, None, None, 0, None, None, None, 1, 1, 1, 1, 0, None) == -1
    assert L.gn_kv_keep(None, None, None, None, None, None, 1, 1, 1, None) == -1
    assert L.gn_logits_adjust(None, None, 0, None, 0, 0, None, 1, 1) == -1
