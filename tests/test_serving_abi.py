"""The structs of the serving calls: the Python mirror against the header, field by field, and the packed form against the
ctypes form.  No GPU."""
import ctypes as C
import os
import re

import pytest

import moeflux_b200 as M
from moeflux_b200 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = {"mfc_shared_prefix_attn": _lib.SharedPrefixAttn, "mfc_attn_weights": _lib.AttnWeights, "mfc_kv_evict": _lib.KvEvict,
           "mfc_verify_drafts": _lib.VerifyDrafts}
TYPES = {"int32_t": C.c_int32, "int64_t": C.c_int64, "float": C.c_float}


def header_fields(name):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "moeflux_cuda.h")).read(), flags=re.S)
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, flags=re.S).group(1)
    fields = []
    for decl in filter(None, (d.strip() for d in body.split(";"))):
        kind, names = re.match(r"(?:const\s+)?(\w+)\s+(.*)", decl, flags=re.S).groups()
        for n in (x.strip() for x in names.split(",")):
            fields.append((n.lstrip("* "), C.c_void_p if n.startswith("*") else TYPES[kind]))
    return fields


@pytest.mark.parametrize("name", STRUCTS)
def test_structs_follow_the_header(name):
    assert list(STRUCTS[name]._fields_) == header_fields(name)


@pytest.mark.parametrize("name", STRUCTS)
def test_packed_form_is_the_struct(name):
    s = STRUCTS[name]
    pack = _lib.packer(s)
    values = {f: 2.5 if t is C.c_float else (1 << 40) + i if t is not C.c_int32 else -i for i, (f, t) in enumerate(s._fields_)}
    assert pack(**values) == bytes(s(**values))
    assert pack() == bytes(s())
    assert pack(**{f: None for f, t in s._fields_ if t is C.c_void_p}) == bytes(s())
    with pytest.raises(TypeError):
        pack(no_such_field=1)


def test_null_context_and_null_struct():
    L = M.lib()
    for fn in (L.mfc_shared_prefix_attn_dev, L.mfc_attn_weights_accumulate_dev, L.mfc_kv_evict_dev, L.mfc_verify_drafts_dev):
        assert fn(None, None) == -1
    assert L.mfc_kv_cache_view(None, 3, 0, None, None, None, None, None) == -1
