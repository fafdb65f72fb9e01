"""The Rust modules of the rotary and state space operators (nebula_amd/rust/rotary.rs, ssm.rs) against the headers they
bind: the same functions with the same types, the same struct fields in the same order, the sizes and constants of the ABI."""
import ctypes
import re
from pathlib import Path

import pytest

from nebula_amd import rotary, ssm

ROOT = Path(__file__).resolve().parent.parent
C_TO_RUST = {
    "uint32_t": "u32", "int64_t": "i64", "size_t": "usize", "size_t*": "*mut usize", "int": "c_int", "float": "f32", "float*": "*mut f32",
    "const float*": "*const f32", "const double*": "*const f64", "char*": "*mut c_char", "const void*": "*const c_void", "void*": "*mut c_void",
    "const int32_t*": "*const i32", "uint32_t*": "*mut u32", "hq_status": "Status", "hq_dtype": "Dtype", "hq_stream": "Stream",
    "hq_rotary_layout": "RotaryLayout", "const hq_rotary*": "*const Rotary", "const hq_rotary_heads*": "*const RotaryHeads",
    "const hq_kv_cache*": "*const KvCache", "const hq_state_cache*": "*const StateCache", "const hq_ssm_io*": "*const SsmIo",
}


def both(name):
    return (re.sub(r"/\*.*?\*/", "", (ROOT / "include" / f"hq_{name}.h").read_text(), flags=re.S),
            (ROOT / "nebula_amd" / "rust" / f"{name}.rs").read_text())


@pytest.mark.parametrize("name,module", [("rotary", rotary), ("ssm", ssm)])
def test_every_function_is_bound_with_the_same_signature(name, module):
    header, rust = both(name)
    c = {}
    for m in re.finditer(r"(\w+) (hq_\w+)\(([^)]*)\);", header):
        types = [" ".join(p.split()).rsplit(" ", 1)[0] for p in m[3].split(",")]
        c[m[2]] = (C_TO_RUST[m[1]], [C_TO_RUST[t] for t in types])
    block = rust[rust.index('extern "C" {'):]
    r = {}
    for m in re.finditer(r"pub fn (hq_\w+)\(([^)]*)\) -> (\w+);", block[:block.index("\n}\n")]):
        r[m[1]] = (m[3], [p.split(":", 1)[1].strip() for p in m[2].split(",")])
    assert c == r and set(c) == set(module.EXPORTS)


@pytest.mark.parametrize("name,cname,rname,binding", [("rotary", "hq_rotary", "Rotary", rotary.RotaryDesc), ("rotary", "hq_rotary_heads", "RotaryHeads", rotary.RotaryHeads),
                                                      ("ssm", "hq_state_cache", "StateCache", ssm.StateCacheDesc), ("ssm", "hq_ssm_io", "SsmIo", ssm.ScanIO)])
def test_structs_mirror_the_header(name, cname, rname, binding):
    header, rust = both(name)
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (cname, cname), header, flags=re.S)[1]
    fields = []
    for line in filter(None, (" ".join(x.split()) for x in body.split(";"))):
        t, names = re.match(r"((?:const )?\w+\*?) (.*)", line).groups()
        fields += [(n.strip().lower(), C_TO_RUST[t]) for n in names.split(",")]
    got = re.findall(r"pub (?:r#)?(\w+): ([^,]+),", re.search(r"pub struct %s \{(.*?)\n\}" % rname, rust, flags=re.S)[1])
    assert got == fields and [n.lower() for n, _ in binding._fields_] == [n for n, _ in fields]
    assert int(re.search(r"size_of::<%s>\(\) == (\d+)" % rname, rust)[1]) == ctypes.sizeof(binding)


def test_constants():
    header, rust = both("ssm")
    assert f"pub const SSM_MAX_BATCH: u32 = {ssm.MAX_BATCH};" in rust and f"#define HQ_SSM_MAX_BATCH {ssm.MAX_BATCH}u" in header
    header, rust = both("rotary")
    for name, value in (("Half", rotary.LAYOUTS["half"]), ("Interleaved", rotary.LAYOUTS["interleaved"])):
        assert f"{name} = {value}," in rust and f"HQ_ROTARY_{name.upper()} = {value}" in header
