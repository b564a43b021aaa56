"""Build ``purin_b200/_lib/libpurin_cp.so`` for sm_100a with nvcc, and its torch binding.

Usage: ``python -m purin_b200.csrc.build [--verbose]``.  The library is built in
tree so it travels with the repository snapshot to the GPU host.  Every projection
kernel is compiled with ``-fmad=false`` so that products and sums round separately,
matching the reference's elementwise arithmetic one operation at a time.
``_ops_torch.so`` (host code only, g++) holds the training-step operators' autograd nodes.
"""

from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
from pathlib import Path

HERE = Path(__file__).resolve().parent
PACKAGE = HERE.parent
ROOT = PACKAGE.parent
LIB_DIR = PACKAGE / "_lib"
LIB = LIB_DIR / "libpurin_cp.so"
SOURCES = ["capi.cu", "cp_forward.cu", "cp_adjoint.cu", "cp_gmres_cluster.cu", "cp_post.cu",
           "sell_order.cu", "admm_forward.cu"]
# The training-step operators (include/purin_ops.h).  They have no reference arithmetic to
# match one operation at a time, so their products and sums may contract (no -fmad=false).
OPS_SOURCES = ["ops_sort.cu", "ops_embedding.cu", "ops_routing.cu", "ops_loss.cu",
               "ops_gradients.cu"]
TORCH_SOURCE = "ops_torch.cpp"
TORCH_LIB = LIB_DIR / "_ops_torch.so"
TORCH_STAMP = LIB_DIR / "_ops_torch.built_for"  # the torch and CPython that it was compiled against
# cp_forward.cu is also compiled once per (dtype, shared values, QP) combination
# of its kernels, so that the heavy template instantiations build in parallel.
FORWARD_PARTS = [(t, sh, qp) for t in ("double", "float") for sh in ("true", "false")
                 for qp in ("true", "false")]
HEADERS = ["common.cuh", "plan.cuh", "cp_kernels.cuh", "sell.cuh", "sell_order.h",
           "adjoint_common.cuh", "ops_common.cuh", "ops_sort.cuh", "ops_umma.cuh"]

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
OPS_FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-Xcompiler", "-O3"]
FLAGS = OPS_FLAGS + ["-fmad=false"]


def nvcc() -> str:
    found = shutil.which("nvcc")
    if found:
        return found
    candidate = Path(os.environ.get("CUDA_HOME", "/usr/local/cuda")) / "bin" / "nvcc"
    if candidate.exists():
        return str(candidate)
    raise RuntimeError("nvcc not found; set CUDA_HOME")


def _inputs():
    files = [HERE / s for s in SOURCES + OPS_SOURCES] + [HERE / h for h in HEADERS]
    files += [ROOT / "include" / "purin_cp.h", ROOT / "include" / "purin_ops.h",
              HERE / TORCH_SOURCE]
    return files


def built_for() -> str:
    """What the binding depends on besides its sources: torch's and CPython's binary interfaces."""
    import sysconfig

    import torch

    return f"torch {torch.__version__}, {sysconfig.get_config_var('SOABI')}\n"


def up_to_date() -> bool:
    if not LIB.exists() or not TORCH_LIB.exists() or not TORCH_STAMP.exists():
        return False
    if TORCH_STAMP.read_text() != built_for():
        return False
    stamp = min(LIB.stat().st_mtime, TORCH_LIB.stat().st_mtime)
    return all(f.stat().st_mtime <= stamp for f in _inputs())


def _torch_paths():
    """Include directories and library directory of torch, CUDA and CPython."""
    import sysconfig

    import torch

    root = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc()).resolve().parents[1]
    include = [root / "include", root / "include" / "torch" / "csrc" / "api" / "include",
               cuda / "include", Path(sysconfig.get_paths()["include"])]
    return include, root / "lib", cuda / "lib64", int(torch._C._GLIBCXX_USE_CXX11_ABI)


def _compile_torch(obj: str):
    include, _, _, abi = _torch_paths()
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-DTORCH_EXTENSION_NAME=_ops_torch",
           f"-D_GLIBCXX_USE_CXX11_ABI={abi}", *[f"-isystem{p}" for p in include], "-c", "-o", obj,
           str(HERE / TORCH_SOURCE)]
    return obj, subprocess.run(cmd, cwd=str(HERE), capture_output=True, text=True)


def _link_torch(obj: str):
    """The binding finds the projection library beside itself, and torch's libraries loaded."""
    _, torch_lib, cuda_lib, _ = _torch_paths()
    tmp = TORCH_LIB.with_suffix(".so.tmp")
    cmd = ["g++", "-shared", "-o", str(tmp), obj, f"-L{LIB_DIR}", "-l:libpurin_cp.so",
           f"-L{torch_lib}", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python",
           f"-L{cuda_lib}", "-lcudart", "-Wl,-rpath,$ORIGIN"]
    proc = subprocess.run(cmd, cwd=str(HERE), capture_output=True, text=True)
    if proc.returncode != 0:
        sys.stderr.write(proc.stdout + proc.stderr)
        raise RuntimeError("g++ failed linking _ops_torch.so")
    os.replace(tmp, TORCH_LIB)
    TORCH_STAMP.write_text(built_for())


def build(verbose: bool = False, force: bool = False) -> Path:
    """Compile every source to an object in parallel (one nvcc per file), then link."""
    from concurrent.futures import ThreadPoolExecutor
    import tempfile

    if not force and up_to_date():
        return LIB
    LIB_DIR.mkdir(parents=True, exist_ok=True)
    tmp = LIB.with_suffix(".so.tmp")
    with tempfile.TemporaryDirectory(prefix="purin_build_") as objdir:
        def compile_one(job):
            src, defines, stem = job
            flags = OPS_FLAGS if src in OPS_SOURCES else FLAGS
            obj = str(Path(objdir) / (stem + ".o"))
            cmd = [nvcc(), *ARCH, *flags, *defines, "-c", "-o", obj, str(HERE / src)]
            if verbose:
                cmd.insert(1, "-Xptxas=-v")
            return obj, subprocess.run(cmd, cwd=str(HERE), capture_output=True, text=True)

        jobs = [(src, [], Path(src).stem) for src in SOURCES + OPS_SOURCES]
        jobs += [("cp_forward.cu", [f"-DPURIN_FWD_PART_T={t}", f"-DPURIN_FWD_PART_SHARED={sh}",
                                    f"-DPURIN_FWD_PART_QP={qp}"], f"cp_forward_{t}_{sh}_{qp}")
                 for t, sh, qp in FORWARD_PARTS]
        workers = min(len(jobs), max(os.cpu_count() or 1, 1)) + 1
        with ThreadPoolExecutor(max_workers=workers) as pool:
            binding = pool.submit(_compile_torch, str(Path(objdir) / "ops_torch.o"))
            results = list(pool.map(compile_one, jobs))
            torch_obj, torch_proc = binding.result()
        for _, proc in results + [(torch_obj, torch_proc)]:
            if proc.returncode != 0:
                sys.stderr.write(proc.stdout + proc.stderr)
                raise RuntimeError("the compiler failed building libpurin_cp.so or its binding")
            if verbose:
                sys.stderr.write(proc.stdout + proc.stderr)
        link = [nvcc(), *ARCH, "-shared", "-o", str(tmp), *[obj for obj, _ in results]]
        proc = subprocess.run(link, cwd=str(HERE), capture_output=True, text=True)
        if proc.returncode != 0:
            sys.stderr.write(proc.stdout + proc.stderr)
            raise RuntimeError("nvcc failed linking libpurin_cp.so")
        os.replace(tmp, LIB)
        _link_torch(torch_obj)
    return LIB


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__)
    parser.add_argument("--verbose", action="store_true")
    parser.add_argument("--force", action="store_true")
    args = parser.parse_args()
    print(build(verbose=args.verbose, force=args.force))


if __name__ == "__main__":
    main()
