"""Compiles the CUDA library for sm_100a with nvcc (cross-compiles without a GPU).

    python -m cgadimpl_b200.build [--force] [--verbose]

Output: cgadimpl_b200/libagb_cuda.so and, next to it, libagb_cuda.ptxas.log with ptxas' resource usage
of every kernel (registers, spills, shared memory); both in-tree and git-ignored.
"""
import os
import re
import shutil
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
LIB = os.path.join(PKG, "libagb_cuda.so")
PTXAS_LOG = os.path.join(PKG, "libagb_cuda.ptxas.log")
OBJ = os.path.join(CSRC, "build")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    # No implicit multiply-add contraction: the kernels keep the reference's rounding points.  (This does
    # not cover the packed __fmul2_rn -> __fadd2_rn pair; see the caution in rmsnorm_staged.cuh.)
    "--fmad=false",
    "-Xcompiler", "-fPIC",
]
# The translation units, compiled side by side; agb_train.cu holds the operators at the end of a model.
UNITS = ["agb_cuda.cu", "agb_train.cu"]


def _nvcc():
    for c in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if c and os.path.exists(c):
            return c
    raise RuntimeError("nvcc not found")


def _sources():
    out = []
    for d in (CSRC, os.path.join(ROOT, "include", "agb")):
        for f in sorted(os.listdir(d)):
            if f.endswith((".cu", ".cuh", ".h")):
                out.append(os.path.join(d, f))
    return out


def _includes(path, seen=None):
    """`path` and the files of this tree that it includes, directly or not."""
    seen = {} if seen is None else seen
    if path in seen:
        return seen
    seen[path] = True
    for name in re.findall(r'^\s*#\s*include\s+"([^"]+)"', open(path).read(), flags=re.M):
        for base in (os.path.dirname(path), CSRC, os.path.join(ROOT, "include")):
            if os.path.exists(os.path.join(base, name)):
                _includes(os.path.join(base, name), seen)
                break
    return seen


def build(force: bool = False, verbose: bool = False) -> str:
    srcs = _sources()
    if not force and os.path.exists(LIB) and os.path.exists(PTXAS_LOG) and \
            all(os.path.getmtime(LIB) >= os.path.getmtime(s) for s in srcs):
        return LIB
    os.makedirs(OBJ, exist_ok=True)
    jobs = []
    for unit in UNITS:
        obj = os.path.join(OBJ, unit[:-3] + ".o")
        log = obj[:-2] + ".ptxas.log"
        if force or not os.path.exists(log) or not os.path.exists(obj) or \
                any(os.path.getmtime(obj) < os.path.getmtime(s) for s in _includes(os.path.join(CSRC, unit))):
            # written beside the target and renamed: a reader never sees a half-written file
            new = f"{obj}.{os.getpid()}.new"
            cmd = [_nvcc()] + NVCC_FLAGS + ["-Xptxas", "-v", "-I", os.path.join(ROOT, "include"), "-I", CSRC, "-c", "-o", new,
                                            os.path.join(CSRC, unit)]
            jobs.append((cmd, new, obj, log, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)))
    failed = []
    for cmd, new, obj, log, proc in jobs:
        out, err = proc.communicate()
        if verbose:
            sys.stderr.write(err)
        if proc.returncode != 0:
            failed.append(" ".join(cmd) + "\n" + out + err)
            continue
        with open(log, "w") as f:
            f.write(err)
        os.replace(new, obj)
    if failed:
        raise RuntimeError("nvcc failed:\n" + "\n".join(failed))
    objs = [os.path.join(OBJ, unit[:-3] + ".o") for unit in UNITS]
    tmp = f"{LIB}.{os.getpid()}.new"
    cmd = [_nvcc()] + NVCC_FLAGS[:2] + ["--shared", "-o", tmp] + objs
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("nvcc failed:\n" + " ".join(cmd) + "\n" + r.stdout + r.stderr)
    os.replace(tmp, LIB)
    with open(PTXAS_LOG, "w") as f:
        for obj in objs:
            f.write(open(obj[:-2] + ".ptxas.log").read())
    return LIB


def kernel_resources():
    """{mangled kernel name: {"registers": n, "spill_stores": bytes, "spill_loads": bytes}} from the last build."""
    build()
    out, name = {}, None
    for line in open(PTXAS_LOG):
        m = re.search(r"Compiling entry function '(\S+)'", line)
        if m:
            name = m.group(1)
            out[name] = {}
            continue
        if name is None:
            continue
        m = re.search(r"(\d+) bytes spill stores, (\d+) bytes spill loads", line)
        if m:
            out[name]["spill_stores"], out[name]["spill_loads"] = int(m.group(1)), int(m.group(2))
        m = re.search(r"Used (\d+) registers", line)
        if m:
            out[name]["registers"] = int(m.group(1))
    return out


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
