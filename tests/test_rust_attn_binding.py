"""The Rust module of the attention operators (nebula_amd/rust/attn.rs) against the header it binds
(include/hq_attn.h): the same functions with the same types, the same struct fields in the same order, the
sizes and constants of the ABI. No Rust toolchain exists in this image, so this keeps the two in step."""
import ctypes
import re
from pathlib import Path

import pytest

from nebula_amd import attn

ROOT = Path(__file__).resolve().parent.parent
HEADER = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "hq_attn.h").read_text(), flags=re.S)
RUST = (ROOT / "nebula_amd" / "rust" / "attn.rs").read_text()

C_TO_RUST = {
    "uint32_t": "u32", "int64_t": "i64", "size_t": "usize", "size_t*": "*mut usize", "int": "c_int", "float": "f32", "float*": "*mut f32",
    "char*": "*mut c_char", "const void*": "*const c_void", "void*": "*mut c_void", "int32_t*": "*mut i32", "const int32_t*": "*const i32",
    "uint32_t*": "*mut u32", "hq_status": "Status", "hq_dtype": "Dtype", "hq_stream": "Stream", "hq_attn_kind": "AttnKind",
    "const hq_attn_io*": "*const AttnIo", "const hq_kv_cache*": "*const KvCache",
}


def test_every_function_is_bound_with_the_same_signature():
    c = {}
    for m in re.finditer(r"(\w+) (hq_\w+)\(([^)]*)\);", HEADER):
        types = [" ".join(p.split()).rsplit(" ", 1)[0] for p in m[3].split(",")]
        c[m[2]] = (C_TO_RUST[m[1]], [C_TO_RUST[t] for t in types])
    block = RUST[RUST.index('extern "C" {'):]
    r = {}
    for m in re.finditer(r"pub fn (hq_\w+)\(([^)]*)\) -> (\w+);", block[:block.index("\n}\n")]):
        r[m[1]] = (m[3], [p.split(":", 1)[1].strip() for p in m[2].split(",")])
    assert c == r and set(c) == set(attn.EXPORTS)


@pytest.mark.parametrize("cname,rname,binding", [("hq_attn_io", "AttnIo", attn.AttnIO), ("hq_kv_cache", "KvCache", attn.KVCacheDesc)])
def test_structs_mirror_the_header(cname, rname, binding):
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (cname, cname), HEADER, flags=re.S)[1]
    fields = []
    for line in filter(None, (" ".join(x.split()) for x in body.split(";"))):
        t, names = re.match(r"((?:const )?\w+\*?) (.*)", line).groups()
        fields += [(n.strip().lower(), C_TO_RUST[t]) for n in names.split(",")]
    got = re.findall(r"pub (\w+): ([^,]+),", re.search(r"pub struct %s \{(.*?)\n\}" % rname, RUST, flags=re.S)[1])
    assert got == fields and [n.lower() for n, _ in binding._fields_] == [n for n, _ in fields]
    assert int(re.search(r"size_of::<%s>\(\) == (\d+)" % rname, RUST)[1]) == ctypes.sizeof(binding)


def test_constants():
    for name, value in (("BAD_ROW", attn.BAD_ROW), ("NO_PAGES", attn.NO_PAGES), ("ROW_FULL", attn.ROW_FULL), ("BAD_PAGE", attn.BAD_PAGE),
                        ("MAX_BATCH", attn.MAX_BATCH)):
        assert f"pub const CACHE_{name}: u32 = {value};" in RUST and f"#define HQ_CACHE_{name} {value}u" in HEADER
    for name, value in (("Prompt", attn.KIND_PROMPT), ("Paged", attn.KIND_PAGED), ("Shared", attn.KIND_SHARED)):
        assert f"{name} = {value}," in RUST and f"HQ_ATTN_{name.upper()} = {value}" in HEADER
