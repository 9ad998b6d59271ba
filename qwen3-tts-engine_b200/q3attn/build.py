"""Build libq3attn.so in-tree for sm_100a (B200) with nvcc.

    python -m q3attn.build            (from qwen3-tts-engine_b200/)   or   q3attn.build.build()

Every .cu under qwen3-tts-engine_b200/csrc is compiled separately (in parallel) and linked into
qwen3-tts-engine_b200/q3attn/libq3attn.so next to this file, where q3attn._lib loads it; csrc/torch_ops.cpp (PyTorch
bindings written in C++) becomes libq3torch.so beside it, linked against libq3attn.so and torch's own libraries. Objects go
to qwen3-tts-engine_b200/_build/. The library is rebuilt unless the SHA-256 of every source, header and this script (and
the nvcc flags and torch's version) equals the digest stamped beside it when it was last built, so a copied tree never runs a library that
was built from other sources, whatever the files' modification times say.
"""
import concurrent.futures as cf
import glob
import hashlib
import os
import re
import shutil
import subprocess
import sys

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG_DIR)                       # qwen3-tts-engine_b200/
REPO = os.path.dirname(ROOT)
CSRC = os.path.join(ROOT, "csrc")
INCLUDE = os.path.join(REPO, "include")
BUILD_DIR = os.path.join(ROOT, "_build")
LIB = os.path.join(PKG_DIR, "libq3attn.so")
TORCH_LIB = os.path.join(PKG_DIR, "libq3torch.so")
TORCH_SRC = os.path.join(CSRC, "torch_ops.cpp")
STAMP = LIB + ".sha256"
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
              "-I", CSRC, "-I", INCLUDE] + ARCH


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: the q3attn CUDA library cannot be built")


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _deps():
    return sources() + [TORCH_SRC] + glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(CSRC, "*.h")) + \
        glob.glob(os.path.join(INCLUDE, "*.h")) + [os.path.abspath(__file__)]


def source_digest() -> str:
    """SHA-256 over the build inputs: each dependency's name and bytes, in name order, plus the nvcc flags and the torch
    that the bindings are compiled against (its C++ interface differs from version to version)."""
    import torch
    h = hashlib.sha256(" ".join(NVCC_FLAGS + [torch.__version__, str(torch._C._GLIBCXX_USE_CXX11_ABI)]).encode())
    for d in sorted(set(_deps())):
        h.update(os.path.basename(d).encode() + b"\0")
        with open(d, "rb") as f:
            h.update(f.read())
    return h.hexdigest()


def up_to_date() -> bool:
    if not (os.path.exists(LIB) and os.path.exists(TORCH_LIB) and os.path.exists(STAMP)):
        return False
    with open(STAMP) as f:
        return f.read().strip() == source_digest()


def torch_flags():
    """Compile and link flags of the PyTorch bindings, from the torch that imports here."""
    import torch
    root = os.path.dirname(os.path.abspath(torch.__file__))
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(nvcc())))
    inc = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
           os.path.join(cuda, "include"), INCLUDE]
    compile_ = ["-O2", "-std=c++17", "-fPIC", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"] + \
        [f for i in inc for f in ("-isystem" if i != INCLUDE else "-I", i)]
    link = ["-L" + os.path.join(root, "lib"), "-ltorch_cpu", "-lc10", "-lc10_cuda", "-L" + PKG_DIR, "-lq3attn",
            "-Wl,-rpath,$ORIGIN", "-Wl,--no-as-needed"]
    return compile_, link


def check_registers(ptxas_log: str) -> None:
    """paged_tree.cu moves registers between its warps, from the count that a kernel is launched with: built at another
    count its launches are refused (they could wait for ever). Raises when the compiler settled on one, so that the build
    says it and not the first call."""
    with open(os.path.join(CSRC, "paged_tree.cu")) as f:
        two_streams, eight_tokens = map(int, re.search(r"kLaunchRegs = kConsumers == 16 \? (\d+) : (\d+)", f.read()).groups())
    found = re.findall(r"Compiling entry function '\S*paged_tree_kernelILb\dELb\dELi(\d)ELi(\d)ELi\dE\S*'.*?Used (\d+) registers",
                       ptxas_log, re.S)
    if not found:
        raise RuntimeError("paged_tree.cu: the compiler's output names no kernel's registers")
    for streams, nt, used in found:
        want = two_streams if streams == "2" else eight_tokens if nt == "2" else int(used)
        if int(used) != want:
            raise RuntimeError(f"paged_tree.cu ({streams} streams, {4 * int(nt)} tokens): compiled with {used} registers, its register "
                               f"split starts from {want} (kLaunchRegs): build with CUDA 12.9, or fit the split to this compiler")


def build(force: bool = False, verbose: bool = False, ptxas_info: bool = False) -> str:
    if not force and not ptxas_info and up_to_date():
        return LIB
    os.makedirs(BUILD_DIR, exist_ok=True)
    cc = nvcc()

    def compile_one(src):
        obj = os.path.join(BUILD_DIR, os.path.basename(src)[:-3] + ".o")
        counted = os.path.basename(src) == "paged_tree.cu"
        cmd = [cc, "-c", src, "-o", obj] + NVCC_FLAGS + (["-Xptxas", "-v"] if ptxas_info or counted else [])
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed on {os.path.basename(src)}:\n{r.stderr}")
        if counted:
            check_registers(r.stderr)
        return obj, r.stderr

    cflags, lflags = torch_flags()
    torch_obj = os.path.join(BUILD_DIR, "torch_ops.o")

    def compile_torch():
        r = subprocess.run(["g++", "-c", TORCH_SRC, "-o", torch_obj] + cflags, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"g++ failed on torch_ops.cpp:\n{r.stderr}")

    with cf.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        bindings = ex.submit(compile_torch)
        results = list(ex.map(compile_one, sources()))
        bindings.result()
    if verbose or ptxas_info:
        for _, err in results:
            if err.strip():
                print(err, file=sys.stderr)
    tmp = LIB + ".tmp"
    cmd = [cc, "-shared", "-o", tmp] + [o for o, _ in results] + ARCH + ["-lcudart"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stderr}")
    os.replace(tmp, LIB)
    tmp = TORCH_LIB + ".tmp"
    r = subprocess.run(["g++", "-shared", "-o", tmp, torch_obj] + lflags, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"linking the PyTorch bindings failed:\n{r.stderr}")
    os.replace(tmp, TORCH_LIB)
    with open(STAMP, "w") as f:
        f.write(source_digest() + "\n")
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True, ptxas_info="--ptxas" in sys.argv))
