"""The compiled binding is a shorter way to the library and no condition for it: without one that
loads, the library's own route (ctypes) serves the 4-bit operators and everything else as before."""

from __future__ import annotations

import importlib.util
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
PKG = ROOT / "bdh-gpu-fast_amd"

CHECK = """
import sys, types, warnings
sys.path.insert(0, {pkg!r})
{how}
with warnings.catch_warnings(record=True) as told:
    warnings.simplefilter("always")
    import bdh_hip_ext as ext
    import kernels
assert kernels.has_hip_ext() and ext._bind is None
assert any("bdh_bind" in str(w.message) for w in told)
import torch
x = torch.zeros(1, 1, 2, 64)
m = kernels.mx4_quantize(x, impl="eager")
cos, sin = kernels.rope_cos_sin(2, 0, kernels.get_freqs(64))
assert ext.mx4_quantize_fast(x, m) is None and ext.mx4_dequantize_fast(m, x) is None
assert ext.mx4_rope_fast(x, cos, sin, m, None) is None and ext.mx4_decode_fast(x, m, x) is None
assert ext.mx4_gemm_fast(x[0, 0].bfloat16(), m[0][0], False, None, None, True) is None
assert ext.launch_count() == 0
"""


@pytest.mark.parametrize("how", [
    "sys.modules['bdh_bind'] = None",  # not built
    "sys.modules['bdh_bind'] = types.ModuleType('bdh_bind')",  # of another version
])
def test_library_without_the_binding(how):
    r = subprocess.run([sys.executable, "-c", CHECK.format(pkg=str(PKG), how=how)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


def test_library_is_built_where_the_binding_is_not(tmp_path, monkeypatch):
    """A failed build of the binding is an error, the library is there all the same, and no binding of
    an earlier build is left beside it."""
    spec = importlib.util.spec_from_file_location("bdh_build_again", PKG / "build.py")
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    monkeypatch.setattr(b, "BUILD", tmp_path / "obj")
    monkeypatch.setattr(b, "LIB", tmp_path / "libbdh_hip.so")
    monkeypatch.setattr(b, "BIND", tmp_path / "bdh_bind.so")
    monkeypatch.setattr(b, "SOURCES", ["api.hip"])
    monkeypatch.setattr(b, "bind_cmd", lambda out: ["false"])
    (tmp_path / "bdh_bind.so").write_bytes(b"an earlier one")
    with pytest.raises(RuntimeError):
        b.build()
    assert (tmp_path / "libbdh_hip.so").stat().st_size > 0 and not (tmp_path / "bdh_bind.so").exists()
