"""In-tree build of libsimilaripy_hip.so (hipcc, gfx950 only).

The shared object is written next to the sources (``similaripy_amd/lib/``): it is
git-ignored, and it is the library that the Python process loads.
"""
from __future__ import annotations

import os
import shutil
import subprocess
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
REPO_DIR = PKG_DIR.parent
CSRC_DIR = PKG_DIR / "csrc"
LIB_DIR = PKG_DIR / "lib"
LIB_PATH = LIB_DIR / "libsimilaripy_hip.so"

INCLUDE_DIR = REPO_DIR / "include"
# the kernels of the dense operators and what they include
DENSE_HEADERS = [CSRC_DIR / n for n in ("sp_dense_common.hpp", "sp_embed_kernels.hpp", "sp_adjust_kernel.hpp", "sp_distill_kernels.hpp")]
# every translation unit with the files it reads: each is compiled to an object of its own, all at once, and linked into the one library
UNITS = {
    CSRC_DIR / "sp_knn.hip": [INCLUDE_DIR / "sp_knn.h", INCLUDE_DIR / "sp_prep.h",
                              *sorted(p for p in CSRC_DIR.glob("*.hpp") if p not in DENSE_HEADERS), *sorted(CSRC_DIR.glob("*.inc"))],
    CSRC_DIR / "sp_dense.hip": [INCLUDE_DIR / "sp_knn.h", INCLUDE_DIR / "sp_dense.h", *DENSE_HEADERS],
}
SOURCES = list(UNITS)
HEADERS = sorted({h for hs in UNITS.values() for h in hs})

HIPCC_FLAGS = [
    "--offload-arch=gfx950",
    "-O3",
    "-std=c++17",
    "-munsafe-fp-atomics",  # LDS float adds must lower to ds_add_f32, never a CAS loop
    # one lane's returning atomic on the row queue must stay PENDING until its value is used a row later: the atomic optimizer
    # rewrites it into a wave-aggregated form whose lanes need the result at once (s_waitcnt vmcnt(0) right behind the atomic)
    "-mllvm", "-amdgpu-atomic-optimizer-strategy=None",
    # no packed float32 instructions (v_pk_add / mul / fma_f32): some of their forms have given wrong results on this hardware
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-fPIC",
    "-Wno-unused-function",
]


def find_hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found (looked at $HIPCC, /opt/rocm/bin/hipcc, PATH)")


def _flags() -> list:
    return [*HIPCC_FLAGS, *os.environ.get("SIMILARIPY_AMD_HIPCC_EXTRA", "").split()]      # (profiling builds only, e.g. -DSP_ABLATION=1)


def _stamp(made: Path) -> Path:
    """Where the command that made a file is kept."""
    return made.with_name(made.name + ".cmd")


def _made_by(made: Path) -> str | None:
    try:
        return _stamp(made).read_text()
    except FileNotFoundError:
        return None


def _put(tmp: Path, made: Path, command: str) -> None:
    """Moves a finished file into place; at no time does another command stand beside it."""
    _stamp(made).unlink(missing_ok=True)
    os.replace(tmp, made)
    _stamp(made).write_text(command)


def is_stale() -> bool:
    """The library is missing, older than its sources or made with other flags (a library without its command counts by time alone)."""
    if not LIB_PATH.exists() or _made_by(LIB_PATH) not in (None, " ".join(_flags())):
        return True
    t = LIB_PATH.stat().st_mtime
    return any(p.exists() and p.stat().st_mtime > t for p in SOURCES + HEADERS)


def _object(src: Path) -> Path:
    return LIB_DIR / (src.stem + ".o")


def _command(src: Path) -> list:
    return [find_hipcc(), *_flags(), "-I", str(INCLUDE_DIR), "-c", str(src)]


def _compile(src: Path, verbose: bool) -> None:
    """One translation unit -> its object next to the library (written aside, then moved into place)."""
    obj = _object(src)
    tmp = obj.with_suffix(".o.tmp%d" % os.getpid())
    made_by = " ".join(_command(src))
    cmd = [*_command(src), "-o", str(tmp)]
    if verbose:
        print(" ".join(cmd))
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0 and "-mllvm" in cmd and ("amdgpu-atomic-optimizer-strategy" in proc.stderr or "Unknown command line argument" in proc.stderr):
        # the -mllvm option is an LLVM internal, not a stable hipcc interface: a toolchain that no longer knows it still builds the
        # library (a performance detail of the row queue's prefetch is lost, nothing else)
        cmd = [c for i, c in enumerate(cmd) if c != "-mllvm" and (i == 0 or cmd[i - 1] != "-mllvm")]
        proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError("hipcc failed:\n" + proc.stdout + proc.stderr)
    _put(tmp, obj, made_by)


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile the HIP library if missing, older than its sources or made with other flags (the units of which that is so; all of them with
    `force`). Returns its path."""
    if not force and not is_stale():
        return LIB_PATH
    LIB_DIR.mkdir(parents=True, exist_ok=True)

    def stale(src):
        obj = _object(src)
        return force or not obj.exists() or _made_by(obj) != " ".join(_command(src)) or any(p.exists() and p.stat().st_mtime > obj.stat().st_mtime for p in [src, *UNITS[src]])
    todo = [s for s in SOURCES if stale(s)]
    with ThreadPoolExecutor(max_workers=max(1, len(todo))) as pool:
        for done in [pool.submit(_compile, s, verbose) for s in todo]:
            done.result()
    tmp = LIB_PATH.with_suffix(".so.tmp%d" % os.getpid())
    cmd = [find_hipcc(), "--offload-arch=gfx950", "-shared", "-fPIC", "-o", str(tmp), *(str(_object(s)) for s in SOURCES)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError("hipcc failed to link:\n" + proc.stdout + proc.stderr)
    _put(tmp, LIB_PATH, " ".join(_flags()))
    return LIB_PATH


if __name__ == "__main__":
    print(build(force=True, verbose=True))
