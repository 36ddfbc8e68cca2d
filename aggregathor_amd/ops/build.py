"""In-tree build of the ``_gar_hip`` torch extension for gfx950.

(The reference's auto-compiling native-op infrastructure equivalent,
/root/reference/native/__init__.py:208-304: mtime-incremental compilation of
the native op library at import/build time; here one hipcc invocation a source, run side
by side, and one that links them into one in-tree .so.)

Direct hipcc invocations (no hipify, no CUDA compatibility machinery): the
kernels are native HIP/CDNA4 and the glue uses the c10::hip API directly.
The resulting ``_gar_hip.so`` is written next to this file, so that a copy of the
tree has it (git ignores it).

Usage: ``python -m aggregathor_amd.ops.build`` (re-builds only when sources
are newer than the .so; ``--force`` to rebuild).
"""

import os
import pathlib
import subprocess
import sys
import sysconfig

OPS_DIR = pathlib.Path(__file__).resolve().parent
CSRC = OPS_DIR / "csrc"
OUT = OPS_DIR / "_gar_hip.so"
OBJ = OPS_DIR / "_obj"

SOURCES = [CSRC / "gar_ops.cpp", CSRC / "gar_kernels.hip",
           CSRC / "bn_kernels.hip", CSRC / "adamw_ops.cpp",
           CSRC / "adamw_kernels.hip"]
FLAGS = pathlib.Path(__file__).resolve()  # how they are compiled
HEADERS = [CSRC / "gar_kernels.h", CSRC / "adamw_kernels.h"]

ARCH = os.environ.get("PYTORCH_ROCM_ARCH", "gfx950")


def _torch_paths():
    import torch.utils.cpp_extension as ce
    return ce.include_paths("cuda"), ce.library_paths("cuda")


def needs_build():
    if not OUT.exists():
        return True
    out_mtime = OUT.stat().st_mtime
    return any(p.stat().st_mtime > out_mtime
               for p in SOURCES + HEADERS + [FLAGS])


def _compile_flags():
    import torch
    includes, _ = _torch_paths()
    abi = int(torch._C._GLIBCXX_USE_CXX11_ABI)
    return [
        f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC",
        # NaN ordering is load-bearing in every GAR: never fast-math.
        "-fno-fast-math",
        # No packed fp32 instructions: some of their forms have given wrong
        # results on this hardware now and then, without an error, and the GAR
        # kernels are as fast without them (profiles/gar_kernels.md). (The host
        # pass does not know the feature and says so; that is harmless.)
        "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
        f"-D_GLIBCXX_USE_CXX11_ABI={abi}",
        "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
        "-DTORCH_EXTENSION_NAME=_gar_hip",
        "-DTORCH_API_INCLUDE_EXTENSION_H",
    ] + [f"-I{inc}" for inc in includes + [sysconfig.get_paths()["include"]]]


def build(force=False, verbose=True):
    if not force and not needs_build():
        if verbose:
            print(f"[ops.build] {OUT.name} up to date")
        return OUT
    import concurrent.futures
    flags = _compile_flags()
    OBJ.mkdir(exist_ok=True)
    newest_header = max(h.stat().st_mtime for h in HEADERS)

    def compile_one(src):
        obj = OBJ / (src.name + ".o")
        if (not force and obj.exists() and obj.stat().st_mtime
                > max(src.stat().st_mtime, newest_header,
                      pathlib.Path(__file__).stat().st_mtime)):
            return obj
        cmd = ["hipcc", "-c", str(src), "-o", str(obj)] + flags
        if verbose:
            print("[ops.build]", " ".join(cmd))
        subprocess.run(cmd, check=True)
        return obj

    with concurrent.futures.ThreadPoolExecutor(len(SOURCES)) as pool:
        objs = list(pool.map(compile_one, SOURCES))
    _, libdirs = _torch_paths()
    cmd = ["hipcc", f"--offload-arch={ARCH}", "-fPIC", "-shared"]
    cmd += [str(o) for o in objs]
    for lib in libdirs:
        cmd.append(f"-L{lib}")
        cmd.append(f"-Wl,-rpath,{lib}")
    cmd += ["-ltorch", "-ltorch_hip", "-lc10", "-lc10_hip", "-ltorch_python",
            "-lamdhip64", "-o", str(OUT)]
    if verbose:
        print("[ops.build]", " ".join(cmd))
    subprocess.run(cmd, check=True)
    if verbose:
        print(f"[ops.build] built {OUT}")
    return OUT


if __name__ == "__main__":
    build(force="--force" in sys.argv)
