"""Build liblssab8_b200.so in place (nvcc, sm_100a only).

The library is two translation units, compiled side by side: csrc/capi.cu (quantisers, prefill,
decode) and csrc/serving.cu (the serving-step operators).  Floating-point flags are part of the contract, not tuning: no fast math, no FMA contraction, IEEE division and
denormals, so every binary32 operation in the fold is the single RN operation the contract names.
"""
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "liblssab8_b200.so")
UNITS = ["capi.cu", "serving.cu"]
SOURCES = UNITS + ["common.cuh", "host.cuh", "tcgen05.cuh", "prep.cuh", "prefill.cuh", "decode.cuh", "decode_tc.cuh",
                   "rotary.cuh", "tables.cuh", "paged.cuh", "t2_table.inc"]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "-ftz=false", "-prec-div=true", "-prec-sqrt=true", "-fmad=false",
]


def nvcc():
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if cand and (os.path.sep not in cand or os.path.exists(cand)):
            return cand
    return "nvcc"


def stale():
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    srcs = [os.path.join(CSRC, s) for s in SOURCES] + [os.path.join(HERE, "..", "include", "lssab8.h")]
    return any(os.path.getmtime(s) > t for s in srcs if os.path.exists(s))


def build(force=False, verbose=False):
    if not force and not stale():
        return LIB
    objs = [os.path.join(HERE, u.replace(".cu", ".o")) for u in UNITS]
    cmds = [[nvcc()] + NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else []) + ["-c", "-o", o, os.path.join(CSRC, u)]
            for u, o in zip(UNITS, objs)]
    jobs = [subprocess.Popen(c, cwd=CSRC, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True) for c in cmds]
    logs = [j.communicate()[0] for j in jobs]
    if all(j.returncode == 0 for j in jobs):
        r = subprocess.run([nvcc(), "-shared", "-o", LIB] + NVCC_FLAGS[:2] + objs, cwd=CSRC, capture_output=True, text=True)
        logs.append(r.stdout + r.stderr)
        jobs.append(r)
    for o in objs:
        if os.path.exists(o):
            os.remove(o)
    if any(j.returncode != 0 for j in jobs):
        sys.stderr.write("".join(logs))
        raise RuntimeError("nvcc failed building liblssab8_b200.so")
    if verbose:
        sys.stderr.write("".join(logs))
    return LIB


if __name__ == "__main__":
    build(force=True, verbose="-v" in sys.argv)
    print(LIB)
