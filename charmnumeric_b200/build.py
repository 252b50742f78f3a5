"""Build libcnb200.so in-tree with nvcc for sm_100a.

    python -m charmnumeric_b200.build [--force] [--verbose]

The device header and the exp table are embedded into the library as text, because every
kernel generated at run time includes them through NVRTC.
"""
import hashlib
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

HERE = Path(__file__).resolve().parent
CSRC = HERE / "csrc"
OUT = HERE / "libcnb200.so"
BUILD = HERE / "_build"
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
HOST_SOURCES = ["wire.cpp", "lower.cpp", "fuse.cpp", "regions.cpp", "decomp.cpp", "codegen.cpp", "jit.cpp", "comm.cpp", "context.cpp",
                "executor.cpp", "sequence.cpp", "capi.cpp"]
SEQUENCE_SOURCES = ["rms_norm.cu", "causal_conv.cu", "selective_scan.cu", "sample.cu"]
CUDA_SOURCES = ["kernels.cu", "noalloc.cu", "storage.cu"] + SEQUENCE_SOURCES


def _embed():
    """Write embedded_headers.cpp holding the texts NVRTC needs."""
    dev = (CSRC / "cn_device.cuh").read_text()
    tab = (CSRC / "cn_exp_table.inc").read_text()
    aot = hashlib.sha256((CSRC / "kernels.cu").read_bytes() + (CSRC / "kernels.hpp").read_bytes()).hexdigest()[:8]
    seq = hashlib.sha256(b"".join((CSRC / s).read_bytes() for s in SEQUENCE_SOURCES + ["sequence.cuh", "sequence.hpp"])).hexdigest()[:8]

    def lit(text):
        # split into chunks: one raw string literal must stay below compiler limits
        parts = [text[i:i + 8000] for i in range(0, len(text), 8000)]
        return "\n".join('R"CNB200(' + p + ')CNB200"' for p in parts)
    body = ('#include "jit.hpp"\nnamespace cn {\n'
            "const char* const kDeviceHeaderText =\n" + lit(dev) + ";\n"
            "const char* const kExpTableText =\n" + lit(tab) + ";\n"
            # the kernels built ahead of time (matvec, dot, halo copies) are identified in
            # profile labels by a digest of their source
            'const char* const kAotSourceDigest = "' + aot + '";\n'
            'const char* const kSequenceSourceDigest = "' + seq + '";\n}\n')
    path = BUILD / "embedded_headers.cpp"
    if not path.exists() or path.read_text() != body:
        path.write_text(body)
    return path


def _digest(paths):
    h = hashlib.sha256()
    for p in sorted(paths):
        h.update(p.name.encode())
        h.update(p.read_bytes())
    return h.hexdigest()


def build(force=False, verbose=False):
    BUILD.mkdir(exist_ok=True)
    cuda_sources = [s for s in CUDA_SOURCES if (CSRC / s).exists()]
    inputs = [CSRC / s for s in HOST_SOURCES + cuda_sources]
    inputs += list(CSRC.glob("*.hpp")) + list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.inc"))
    inputs += [HERE.parent / "include" / "cnb200.h", Path(__file__)]
    stamp = BUILD / "stamp"
    digest = _digest(inputs)
    if not force and OUT.exists() and stamp.exists() and stamp.read_text() == digest:
        return OUT
    emb = _embed()
    common = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC,-Wall,-Wno-unused-function",
              "-I", str(CSRC), "-I", str(BUILD)]
    def compile_one(src):
        obj = BUILD / (src.stem + ".o")
        if src.suffix == ".cu":
            cmd = [NVCC] + ARCH + common + ["-Xptxas", "-v", "-c", str(src), "-o", str(obj)]
        else:
            cmd = [NVCC, "-x", "cu"] + ARCH + common + ["-c", str(src), "-o", str(obj)]
        if verbose:
            print(" ".join(cmd))
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode:
            sys.stderr.write(res.stdout + res.stderr)
            res.check_returncode()
        if src.suffix == ".cu":
            (BUILD / (src.stem + ".ptxas.txt")).write_text(res.stderr)
        elif res.stderr:
            sys.stderr.write(res.stderr)
        if verbose and src.suffix == ".cu":
            print(res.stderr)
        return obj

    # the longest first: selective_scan.cu alone takes as long as all host sources together
    sources = [CSRC / s for s in reversed(cuda_sources)] + [CSRC / s for s in HOST_SOURCES] + [emb]
    with ThreadPoolExecutor(max_workers=max(1, min(8, os.cpu_count() or 1))) as pool:
        objs = list(pool.map(compile_one, sources))
    cmd = [NVCC, "-shared"] + ARCH + ["-o", str(OUT)] + [str(o) for o in objs] + ["-ldl", "-lpthread"]
    if verbose:
        print(" ".join(cmd))
    subprocess.run(cmd, check=True)
    stamp.write_text(digest)
    return OUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
