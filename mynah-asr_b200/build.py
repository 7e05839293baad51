"""Builds the CUDA library in-tree: mynah-asr_b200/libmynah_b200.so (sm_100a only)."""
from __future__ import annotations

import os
import re
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libmynah_b200.so")
SOURCES = ["util.cu", "hostcopy.cu", "gemm_tc.cu", "gemm_i8.cu", "gemm_skinny.cu", "dequant.cu", "elementwise.cu", "attention.cu", "attention_tc.cu", "subsampling.cu", "mel.cu",
           "qgemv.cu", "qgemv_mma.cu", "qstream_tc.cu", "decoder.cu", "decoder_aed.cu", "fewrow.cu", "align.cu", "vad.cu", "stream.cu", "model.cu", "loader.cu", "kv.cu", "kv_append.cu", "kv_step.cu", "kv_chunk.cu", "capi.cu"]
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
              "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr"]

# Kernels that deal their launch's registers out anew between their warps: they refuse to run where the compiler gave them fewer, so it is said here
REGISTERS = {"kv_chunk.cu": {"kv_chunk_kernelILi64E": 128, "kv_chunk_kernelILi128E": 168}}


def missing_registers(source: str, said: str) -> list:
    """What nvcc's report on a source (-Xptxas -v) says of kernels that need a certain number of registers and have another, or does not say."""
    wrong = []
    for kernel, need in REGISTERS.get(source, {}).items():
        found = re.findall(r"entry function '(\S*%s\S*)'(?:(?!entry function).)*?Used (\d+) registers" % kernel, said, re.S)
        wrong += [f"{name}: {have} registers, not {need}" for name, have in found if int(have) != need]
        if not found:
            wrong.append(f"{kernel}: no report")
    return wrong


def _stale(obj: str, deps) -> bool:
    if not os.path.exists(obj):
        return True
    t = os.path.getmtime(obj)
    return any(os.path.getmtime(d) > t for d in deps)


def build(verbose: bool = False, force: bool = False) -> str:
    nvcc = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
    objdir = os.path.join(HERE, "build")
    os.makedirs(objdir, exist_ok=True)
    headers = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".h", ".cuh"))]
    headers.append(os.path.join(HERE, "..", "include", "mynah_b200.h"))
    objs, procs = [], []
    for s in SOURCES:
        src = os.path.join(CSRC, s)
        if not os.path.exists(src):
            continue
        obj = os.path.join(objdir, s.replace(".cu", ".o"))
        objs.append(obj)
        if force or _stale(obj, [src] + headers):
            cmd = [nvcc] + NVCC_FLAGS + (["-Xptxas", "-v"] if verbose or s in REGISTERS else []) + ["-c", src, "-o", obj]
            procs.append((s, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    failed = False
    for s, p in procs:
        out, _ = p.communicate()
        if p.returncode != 0 or verbose:
            sys.stderr.write(f"--- {s}\n{out}\n")
        wrong = missing_registers(s, out) if p.returncode == 0 else []
        if wrong:
            sys.stderr.write(f"--- {s}\n" + "\n".join(wrong) + "\n")
            os.remove(os.path.join(objdir, s.replace(".cu", ".o")))
        failed |= p.returncode != 0 or bool(wrong)
    if failed:
        raise RuntimeError("the build failed")
    if procs or not os.path.exists(LIB):
        subprocess.check_call([nvcc, "-shared", "-o", LIB] + objs + ["-lcudart"])
    return LIB


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv, force="-f" in sys.argv))
