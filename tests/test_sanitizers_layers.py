"""The validators of the attention, cache, rotary and state space entry points under AddressSanitizer and
UndefinedBehaviorSanitizer (CPU only), as tests/test_sanitizers.py runs those of the products and the parsers: strides,
spans and layouts at their ends, null and misaligned pointers, packed descriptors, workspace queries over lengths.
"""
import os
import subprocess
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent
SUITES = ["attn_abi", "attn_grids", "attn_output_overlap", "attn_workspace_range", "cache_refused_abi", "rotary_abi", "rotary_aliases", "ssm_abi",
          "ssm_conv_grid", "ssm_workspace_range"]


def test_validators_under_asan_and_ubsan():
    sys.path.insert(0, str(ROOT))
    from nebula_amd import build_sanitize as BS

    assert {"hq_attn_api.cpp", "hq_ssm_api.cpp"} <= set(BS.SAN_SOURCES)
    lib, olib = BS.build_sanitized()
    env = dict(os.environ, HQ_LIB=str(lib), HQO_LIB=str(olib), LD_PRELOAD=str(BS.asan_runtime()),
               ASAN_OPTIONS="detect_leaks=0:halt_on_error=1", UBSAN_OPTIONS="halt_on_error=1:print_stacktrace=1")
    suites = [f"tests/test_{name}.py" for name in SUITES]
    proc = subprocess.run([sys.executable, "-m", "pytest", "-q", "-x", "-p", "no:cacheprovider", *suites, "-m", "not gpu"], cwd=str(ROOT), env=env,
                          capture_output=True, text=True, timeout=900)
    out = proc.stdout + proc.stderr
    assert "AddressSanitizer" not in out and "runtime error:" not in out, out[-4000:]
    assert proc.returncode == 0 and " passed" in proc.stdout, out[-4000:]
