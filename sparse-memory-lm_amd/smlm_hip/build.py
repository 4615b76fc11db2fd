"""Build the gfx950 C-ABI library libsmlm_pkm.so from csrc/*.hip with hipcc.

    python -m smlm_hip.build            (from sparse-memory-lm_amd/)

Every .hip file is compiled to an object in sparse-memory-lm_amd/_build/ (in parallel), then linked into
smlm_hip/libsmlm_pkm.so next to this file, where smlm_hip._lib loads it.  The autograd nodes of the training operators
and the wrappers of the ragged-serving operators (csrc/torch/*.cpp, host code against torch's headers) become the Python
modules smlm_hip/_train_ops.so and _serve_ops.so.  The memory-ceiling
kernels of bench.py (csrc/bench/*.hip: sequential read / write / copy and random-row reads) go into a separate
smlm_hip/libsmlm_bench.so, so the lookup library holds only the product.
"""
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG_DIR)                       # sparse-memory-lm_amd/
REPO = os.path.dirname(ROOT)
CSRC = os.path.join(ROOT, "csrc")
INCLUDE = os.path.join(REPO, "include")
BUILD_DIR = os.path.join(ROOT, "_build")
LIB_NAME = "libsmlm_pkm.so"
LIB_PATH = os.path.join(PKG_DIR, LIB_NAME)
BENCH_LIB_PATH = os.path.join(PKG_DIR, "libsmlm_bench.so")
TORCH_MODULES = ("train_ops", "serve_ops")            # csrc/torch/<name>.cpp -> smlm_hip/_<name>.so
ARCH = "gfx950"

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
CXX = os.environ.get("CXX", "g++")
CFLAGS = [
    f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC", "-Wall",
    # no packed-fp32 (v_pk_*_f32) instructions anywhere in the device code
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    # MFMA accumulators in ordinary VGPRs: otherwise the compiler keeps them in AGPRs and copies them back and
    # forth around every epilogue / softmax (v_accvgpr_read / write; ~23k of them across the decode linears)
    "-mllvm", "-amdgpu-mfma-vgpr-form",
    f"-I{INCLUDE}",
]


def sources(folder=CSRC):
    return sorted(os.path.join(folder, f) for f in os.listdir(folder) if f.endswith(".hip"))


def _compile(src):
    sub = os.path.relpath(os.path.dirname(src), CSRC).replace(os.sep, "_").strip("._")
    obj = os.path.join(BUILD_DIR, (sub + "_" if sub else "") + os.path.basename(src)[:-4] + ".o")
    cmd = [HIPCC, *CFLAGS, "-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    # hipcc's host pass does not know the packed-fp32 feature and says so; that warning is harmless
    err = "\n".join(line for line in r.stderr.splitlines() if "packed-fp32-ops" not in line)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{' '.join(cmd)}\n{err}")
    if err.strip():
        print(err, file=sys.stderr)
    return obj


def _link(objs, path):
    tmp = path + ".tmp"
    cmd = [HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", *objs, "-o", tmp]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{' '.join(cmd)}\n{r.stderr}")
    os.replace(tmp, path)


def _compile_torch(name):
    """The object of csrc/torch/<name>.cpp: plain C++ with torch's headers and the HIP runtime's."""
    import sysconfig

    import torch
    from torch.utils import cpp_extension
    obj = os.path.join(BUILD_DIR, f"torch_{name}.o")
    rocm = os.path.dirname(os.path.dirname(HIPCC))
    cmd = [CXX, "-O2", "-std=c++17", "-fPIC", "-Wall", "-Wno-attributes", "-fvisibility=hidden", "-D__HIP_PLATFORM_AMD__=1",
           "-DUSE_ROCM=1", f"-DTORCH_EXTENSION_NAME=_{name}", "-DTORCH_API_INCLUDE_EXTENSION_H",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-I{INCLUDE}",
           *(f"-isystem{p}" for p in (*cpp_extension.include_paths(), sysconfig.get_paths()["include"],
                                      os.path.join(rocm, "include"))),
           "-c", os.path.join(CSRC, "torch", f"{name}.cpp"), "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{CXX} failed for {name}.cpp:\n{' '.join(cmd)}\n{r.stderr}")
    if r.stderr.strip():
        print(r.stderr, file=sys.stderr)
    return obj


def _link_torch(name, obj):
    from torch.utils import cpp_extension
    libs = cpp_extension.library_paths()
    path = os.path.join(PKG_DIR, f"_{name}.so")
    tmp = path + ".tmp"
    cmd = [CXX, "-shared", obj, f"-L{PKG_DIR}", "-lsmlm_pkm", "-Wl,-rpath,$ORIGIN", *(f"-L{p}" for p in libs), "-lc10",
           "-lc10_hip", "-ltorch_cpu", "-ltorch", "-ltorch_python", "-o", tmp]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{' '.join(cmd)}\n{r.stderr}")
    os.replace(tmp, path)


def build(verbose=True):
    """Compile every csrc/*.hip for gfx950 and link libsmlm_pkm.so, csrc/torch into _train_ops.so and _serve_ops.so and csrc/bench/*.hip into
    libsmlm_bench.so.  Always rebuilds."""
    os.makedirs(BUILD_DIR, exist_ok=True)
    srcs, bench_srcs = sources(), sources(os.path.join(CSRC, "bench"))
    with ThreadPoolExecutor(max_workers=min(8, len(srcs) + len(bench_srcs))) as ex:
        torch_objs = [(name, ex.submit(_compile_torch, name)) for name in TORCH_MODULES]          # the longest first
        objs = list(ex.map(_compile, srcs + bench_srcs))
    _link(objs[:len(srcs)], LIB_PATH)
    for name, obj in torch_objs:
        _link_torch(name, obj.result())
    _link(objs[len(srcs):], BENCH_LIB_PATH)
    if verbose:
        print(f"built {LIB_PATH} from {len(srcs)} sources and {BENCH_LIB_PATH} from {len(bench_srcs)}", flush=True)
    return LIB_PATH


if __name__ == "__main__":
    build()
