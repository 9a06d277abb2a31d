"""Build the gfx950 C-ABI library ``libbdh_hip.so`` with hipcc.

Usage:  python bdh-gpu-fast_amd/build.py [--jobs N] [--verbose]

Each ``csrc/*.hip`` file is compiled to an object under ``_build/`` (in
parallel), then linked into ``libbdh_hip.so`` next to this file.  hipcc
cross-compiles for gfx950 without a GPU present.  ``csrc/bind.cpp`` (host code,
against torch's headers) becomes the Python module ``bdh_bind`` beside it.
"""

from __future__ import annotations

import argparse
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

HERE = Path(__file__).resolve().parent
ROOT = HERE.parent
CSRC = HERE / "csrc"
BUILD = HERE / "_build"
LIB = HERE / "libbdh_hip.so"
BIND = HERE / "bdh_bind.so"
SOURCES = ["api.hip", "fwd.hip", "syrk.hip", "bwd.hip", "f32.hip", "decode.hip", "decode_step.hip", "rope.hip", "model.hip", "gated_dec.hip", "gated_bwd.hip", "few.hip", "enc.hip", "mx4.hip", "mx4_gemm.hip"]
ARCH = os.environ.get("BDH_OFFLOAD_ARCH", "gfx950")


def hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", "hipcc"):
        if cand and (os.path.sep not in cand or Path(cand).exists()):
            return cand
    raise RuntimeError("hipcc not found")


def common_flags() -> list[str]:
    return [
        f"--offload-arch={ARCH}",
        "-O3",
        "-std=c++17",
        "-fPIC",
        # packed fp32 VALU ops are disabled for every HIP translation unit
        "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
        "-Wno-unused-command-line-argument",
        f"-I{ROOT / 'include'}",
        f"-I{CSRC}",
    ]


def bind_cmd(out: Path) -> list[str]:
    """Compile and link ``bdh_bind`` (a CPython extension; torch's libraries are loaded by then)."""
    import sysconfig

    import torch
    from torch.utils.cpp_extension import include_paths

    lib = Path(torch.__file__).resolve().parent / "lib"
    return [
        "g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-w",
        f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
        *(f"-isystem{p}" for p in (*include_paths(), sysconfig.get_paths()["include"])),
        f"-I{ROOT / 'include'}", str(CSRC / "bind.cpp"), "-o", str(out),
        f"-L{lib}", "-ltorch_python", "-ltorch_cpu", "-lc10",
    ]


def _run(cmd: list[str], verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError(f"command failed ({res.returncode}): {' '.join(cmd)}")
    noise = "is not a recognized feature for this target"
    err = "\n".join(l for l in res.stderr.splitlines() if noise not in l and l.strip())
    if err and verbose:
        sys.stderr.write(err + "\n")


def build(jobs: int | None = None, verbose: bool = False) -> Path:
    BUILD.mkdir(exist_ok=True)
    cc = hipcc()
    flags = common_flags()
    objs = []
    cmds = []
    for src in SOURCES:
        obj = BUILD / (Path(src).stem + ".o")
        objs.append(obj)
        cmds.append([cc, *flags, "-c", str(CSRC / src), "-o", str(obj)])
    bind = BIND.with_suffix(".so.tmp")
    jobs = jobs or min(len(cmds) + 1, os.cpu_count() or 4, 8)
    with ThreadPoolExecutor(max_workers=jobs) as ex:
        binding = ex.submit(lambda: _run(bind_cmd(bind), verbose))
        list(ex.map(lambda c: _run(c, verbose), cmds))
    tmp = LIB.with_suffix(".so.tmp")
    _run([cc, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", str(tmp), *map(str, objs)], verbose)
    # the library needs no binding: a failure there comes after it, and leaves none of an earlier build
    os.replace(tmp, LIB)
    BIND.unlink(missing_ok=True)
    binding.result()
    os.replace(bind, BIND)
    return LIB


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--jobs", type=int, default=None)
    ap.add_argument("--verbose", action="store_true")
    args = ap.parse_args()
    print(build(args.jobs, args.verbose))


if __name__ == "__main__":
    main()
