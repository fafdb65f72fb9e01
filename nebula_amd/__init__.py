"""nebula_amd — MI355X (gfx950) weight-only quantized GEMM for hydrogen's qGEMM path, and the attention between its projections.

The compute lives in libnebula_hq.so (HIP, built by nebula_amd.build); this package
holds its ctypes bindings (nebula_amd.hq, nebula_amd.attn) and the build recipe.
"""
from . import attn, hq  # noqa: F401

__all__ = ["attn", "hq"]
