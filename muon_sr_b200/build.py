"""Build the engine's C-ABI shared library, ``muon_sr_b200/libmuon_sr_b200.so``, with nvcc, and
the Python binding of the gradient norm, ``muon_sr_b200/_native.so``, against the installed torch.

    python -m muon_sr_b200.build [--verbose-ptxas] [--force]

builds what is older than its sources, and the binding again under another torch or interpreter.
Every CUDA source under ``csrc/`` is compiled for sm_100a only
(``-gencode arch=compute_100a,code=sm_100a``) and linked with the static CUDA runtime into
one in-tree shared object that the Python layer loads with ctypes. The elementwise and
8-bit sources are compiled with ``--fmad=false`` so no multiply-add is contracted (their
results are bit-compared with the reference). nvcc cross-compiles without a GPU.
"""
import argparse
import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
import sysconfig

from ._lib import built_for

PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG, "csrc")
BUILD = os.path.join(PKG, "_build")
LIB = os.path.join(PKG, "libmuon_sr_b200.so")
BINDING = os.path.join(PKG, "_native.so")
BINDING_OBJ = os.path.join(BUILD, "binding.o")
BINDING_FOR = os.path.join(BUILD, "binding.for")  # what the binding was built against
INCLUDE = os.path.join(os.path.dirname(PKG), "include")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
COMMON = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC,-O2", "--expt-relaxed-constexpr", "-I", INCLUDE]
NO_FMA = {"elementwise.cu", "adamw8bit.cu"}


def nvcc():
    path = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(path):
        raise RuntimeError("nvcc not found; the CUDA 12.9 toolkit is required to build muon_sr_b200")
    return path


def sources():
    return sorted(f for f in os.listdir(CSRC) if f.endswith(".cu"))


def _deps_mtime():
    files = [os.path.join(CSRC, f) for f in os.listdir(CSRC)] + [os.path.join(INCLUDE, f) for f in os.listdir(INCLUDE)]
    return max(os.path.getmtime(f) for f in files)


def _current(path):
    return os.path.exists(path) and os.path.getmtime(path) >= _deps_mtime()


def _binding_current():
    """Whether the binding is newer than its sources and built against this torch: it holds
    torch's inline accessors and the interpreter's ABI, which file times say nothing of."""
    if not _current(BINDING) or not os.path.exists(BINDING_FOR):
        return False
    with open(BINDING_FOR) as f:
        return f.read() == built_for()


def build(force: bool = False, verbose_ptxas: bool = False) -> str:
    library = force or not _current(LIB)
    if not library and _binding_current():
        return LIB
    os.makedirs(BUILD, exist_ok=True)
    if not library:
        _build_binding()
        return LIB
    cc = nvcc()

    def compile_one(src):
        obj = os.path.join(BUILD, src.replace(".cu", ".o"))
        cmd = [cc, *ARCH, *COMMON, "-c", os.path.join(CSRC, src), "-o", obj]
        if src in NO_FMA:
            cmd.insert(1, "--fmad=false")
        if verbose_ptxas:
            cmd.insert(1, "-Xptxas=-v")
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src}:\n{r.stdout}\n{r.stderr}")
        return obj, r.stderr

    with cf.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        binding = ex.submit(_compile_binding)
        results = list(ex.map(compile_one, sources()))
    if verbose_ptxas:
        for obj, err in results:
            sys.stderr.write(f"== {os.path.basename(obj)}\n{err}")
    tmp = LIB + ".tmp"
    cmd = [cc, *ARCH, "-shared", "-cudart", "static", "-o", tmp, *[o for o, _ in results]]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, LIB)
    binding.result()  # after the library, which does not need it
    _link_binding()
    return LIB


def _run(cmd, what):
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{what} failed:\n{r.stdout}\n{r.stderr}")


def _build_binding():
    _compile_binding()
    _link_binding()


def _compile_binding():
    import torch
    root = os.path.join(os.path.dirname(torch.__file__), "include")
    cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(nvcc()))), "include")
    dirs = [root, os.path.join(root, "torch", "csrc", "api", "include"), cuda, sysconfig.get_paths()["include"]]
    _run(["g++", "-O2", "-std=c++17", "-fPIC", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
          f'-DMSR_BUILT_FOR="{built_for()}"', *[f"-isystem{d}" for d in dirs], "-c", os.path.join(CSRC, "binding.cpp"),
          "-o", BINDING_OBJ], "g++ on binding.cpp")


def _link_binding():
    import torch
    libs = os.path.join(os.path.dirname(torch.__file__), "lib")
    tmp = BINDING + ".tmp"
    _run(["g++", "-shared", "-o", tmp, BINDING_OBJ, f"-L{PKG}", "-lmuon_sr_b200", f"-L{libs}", "-ltorch_python", "-ltorch_cpu",
          "-lc10", "-lc10_cuda", "-Wl,-rpath,$ORIGIN"], "linking the binding")
    os.replace(tmp, BINDING)
    with open(BINDING_FOR, "w") as f:
        f.write(built_for())


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose-ptxas", action="store_true")
    args = ap.parse_args()
    print(build(force=args.force, verbose_ptxas=args.verbose_ptxas))


if __name__ == "__main__":
    main()
