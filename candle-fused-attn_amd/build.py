"""Build recipe of libfattn.so: hand-written HIP for gfx950 only.

It plays the part of the reference's build.rs (build.rs:5-30), which compiles
kernels/fused_attn.cu to PTX with nvcc: here hipcc compiles the kernels and the C-ABI layer
into one shared library holding a gfx950 code object (no PTX, no JIT, no other target).

Usage: ``python candle-fused-attn_amd/build.py`` (or ``build()`` from Python).
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
import tempfile
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
REPO = PKG_DIR.parent
CSRC = PKG_DIR / "csrc"
LIB_DIR = PKG_DIR / "lib"
LIB = LIB_DIR / "libfattn.so"
SOURCES = [CSRC / "fattn_pair.hip", CSRC / "fattn_cross.hip", CSRC / "fattn_scored.hip",
           CSRC / "fattn_paged.hip", CSRC / "fattn_rotary.hip",
           CSRC / "fattn_kernels.hip", CSRC / "fattn_api.cpp", CSRC / "fattn_operators.cpp"]
HEADERS = [REPO / "include" / "fattn.h", CSRC / "fattn_internal.h", CSRC / "fattn_device.h",
           CSRC / "fattn_pair_kernels.h"]
# The C++ op layer over the C ABI (the reference's src/lib.rs ops for C++ callers), linked
# against libfattn.so, and its test program (links the CPU oracle; test infrastructure).
HOST = PKG_DIR / "host"
HOST_LIB = LIB_DIR / "libcandle_fused_attn.so"
HOST_TEST_SRC = REPO / "tests" / "cpp" / "parity_host.cpp"
HOST_TEST = REPO / "tests" / "cpp" / "parity_host"
ORACLE_DIR = REPO / "oracle"

# gfx950 only. Packed fp32 ALU instructions are disabled (-packed-fp32-ops); the host pass warns
# that it does not know that target feature, which is harmless.
HIPCC_FLAGS = [
    "--offload-arch=gfx950",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-shared",
    "-mcode-object-version=5",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall",
]


def hipcc() -> str:
    path = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not Path(path).exists():
        raise RuntimeError("hipcc not found: the ROCm toolchain is required to build libfattn.so")
    return path


def compile_command(src: Path, out: Path) -> list[str]:
    flags = [f for f in HIPCC_FLAGS if f != "-shared"]
    return [hipcc(), *flags, f"-I{REPO / 'include'}", f"-I{CSRC}", "-x", "hip", "-c", str(src),
            "-o", str(out)]


def link_command(objects: list[Path], out: Path = LIB) -> list[str]:
    return [hipcc(), "--offload-arch=gfx950", "-fPIC", "-shared", *[str(o) for o in objects], "-o",
            str(out)]


def _run(cmd: list[str], tmp: Path, out: Path, verbose: bool, cwd: Path | None = None) -> Path:
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True, cwd=cwd)
    if res.returncode != 0:
        raise RuntimeError(f"hipcc failed ({res.returncode}):\n{res.stdout}\n{res.stderr}")
    if tmp != out:
        os.replace(tmp, out)
    return out


def compile_objects(sources: list[Path], folder: Path, verbose: bool = False) -> list[Path]:
    """One object file in `folder` per source, compiled at once. The commands name them without the
    folder: hipcc puts a hash of its command into the object, and a library of the same sources has to
    be the same file wherever it was built (bench.py knows by its hash which one was measured)."""
    outs = [Path(s.name + ".o") for s in sources]
    with ThreadPoolExecutor(len(sources)) as pool:
        # (list() waits for every source and raises what a compilation raised.)
        list(pool.map(lambda so: _run(compile_command(*so), so[1], so[1], verbose, folder),
                      zip(sources, outs)))
    return [folder / o for o in outs]


def build(verbose: bool = False) -> Path:
    """Compile libfattn.so in-tree (always; the caller decides when to rebuild)."""
    LIB_DIR.mkdir(parents=True, exist_ok=True)
    tmp = LIB.with_suffix(".so.tmp")
    with tempfile.TemporaryDirectory() as d:
        return _run(link_command(compile_objects(SOURCES, Path(d), verbose), tmp), tmp, LIB, verbose)


def host_command(out: Path = HOST_LIB) -> list[str]:
    return [hipcc(), "-x", "hip", *HIPCC_FLAGS, f"-I{REPO / 'include'}", f"-I{HOST}",
            str(HOST / "candle_fused_attn.cpp"), f"-L{LIB_DIR}", "-lfattn",
            "-Wl,-rpath,$ORIGIN", "-o", str(out)]


def build_host(verbose: bool = False) -> Path:
    """Compile libcandle_fused_attn.so (the C++ op layer; needs libfattn.so built first)."""
    tmp = HOST_LIB.with_suffix(".so.tmp")
    return _run(host_command(tmp), tmp, HOST_LIB, verbose)


# The operators around self-attention for Python (torch's C++ API over libfattn.so).
OPERATORS_SRC = HOST / "torch_operators.cpp"
OPERATORS = LIB_DIR / "torch_operators.so"


def operators_command(out: Path = OPERATORS) -> list[str]:
    import torch

    root = Path(torch.__file__).resolve().parent
    abi = int(torch.compiled_with_cxx11_abi())
    return [hipcc(), "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-fvisibility=hidden",
            "-DUSE_ROCM", f"-D_GLIBCXX_USE_CXX11_ABI={abi}", f"-I{REPO / 'include'}",
            f"-I{root / 'include'}", f"-I{root / 'include/torch/csrc/api/include'}",
            f"-I{sysconfig.get_paths()['include']}", str(OPERATORS_SRC), f"-L{LIB_DIR}", "-lfattn",
            f"-L{root / 'lib'}", "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch_python",
            "-Wl,-rpath,$ORIGIN", "-o", str(out)]


def build_operators(verbose: bool = False) -> Path:
    """Compile lib/torch_operators.so (needs libfattn.so built first)."""
    tmp = OPERATORS.with_suffix(".so.tmp")
    return _run(operators_command(tmp), tmp, OPERATORS, verbose)


STEP_BENCH_SRC = HOST / "step_bench.cpp"
STEP_BENCH = LIB_DIR / "cfa_step_bench"


def step_bench_command(out: Path = STEP_BENCH) -> list[str]:
    return [hipcc(), "-O2", "-std=c++17", "-Wall", f"-I{HOST}", str(STEP_BENCH_SRC),
            f"-L{LIB_DIR}", "-lcandle_fused_attn", "-lfattn", "-Wl,-rpath,$ORIGIN",
            "-o", str(out)]


def build_step_bench(verbose: bool = False) -> Path:
    """Compile lib/cfa_step_bench (times steps through the C++ op layer; needs
    libcandle_fused_attn.so built first)."""
    tmp = STEP_BENCH.with_name(STEP_BENCH.name + ".tmp")
    return _run(step_bench_command(tmp), tmp, STEP_BENCH, verbose)


def host_test_command(out: Path = HOST_TEST) -> list[str]:
    rpath = "$ORIGIN/../../candle-fused-attn_amd/lib:$ORIGIN/../../oracle"
    return [hipcc(), "-O2", "-std=c++17", "-Wall", f"-I{HOST}", str(HOST_TEST_SRC),
            f"-L{LIB_DIR}", "-lcandle_fused_attn", "-lfattn", f"-L{ORACLE_DIR}", "-loracle",
            f"-Wl,-rpath,{rpath}", "-o", str(out)]


def build_host_test(verbose: bool = False) -> Path:
    """Compile tests/cpp/parity_host (needs libcandle_fused_attn.so and oracle/liboracle.so)."""
    tmp = HOST_TEST.with_name(HOST_TEST.name + ".tmp")
    return _run(host_test_command(tmp), tmp, HOST_TEST, verbose)


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
    print(build_operators(verbose="-v" in sys.argv))
    print(build_host(verbose="-v" in sys.argv))
    print(build_step_bench(verbose="-v" in sys.argv))
