"""Build the quipsharp_b200 CUDA library for sm_100a (in-tree).

    python -m quipsharp_b200.build_native [-v]

Writes quipsharp_b200/_lib/libquipsharp_b200.so and the Python extension
quipsharp_b200/_lib/_fast.so (host code only).  The codebook tables and the
odd-prime DFT constants are generated into quipsharp_b200/_build/qs_tables_gen.inc
from quipsharp_b200/codebooks/tables.py before compiling, so the device code
carries exactly the tables the Python codebook objects expose.
"""
from __future__ import annotations

import concurrent.futures as cf
import math
import os
import shutil
import struct
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG, "csrc")
BUILD = os.path.join(PKG, "_build")
LIBDIR = os.path.join(PKG, "_lib")
LIBNAME = "libquipsharp_b200.so"
REPO = os.path.dirname(PKG)

PRIMES = (3, 5, 7, 11, 13, 17, 19, 23, 29, 31, 37, 41, 43)
ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def _fp16_high_byte(v: float) -> int:
    lo, hi = struct.pack("<e", v)
    assert lo == 0, (v, lo)
    return hi


def _float_lit(v: float) -> str:
    r = repr(float(struct.unpack("<f", struct.pack("<f", v))[0]))
    return r + "f" if ("." in r or "e" in r) else r + ".0f"


def generate_tables_inc(path: str) -> None:
    sys.path.insert(0, REPO)
    from quipsharp_b200.codebooks.tables import e8p_abs_table_x2, e8_1bit_table_x2

    e8p = e8p_abs_table_x2()
    onebit = e8_1bit_table_x2()
    lines = ["// GENERATED by quipsharp_b200/build_native.py -- do not edit.", ""]

    def f32_array(name, rows, qual):
        vals = [_float_lit(v / 2.0) for r in rows for v in r]
        body = ",".join(vals)
        lines.append(f"{qual} float {name}[{len(vals)}] = {{{body}}};")

    def hb_array(name, rows):
        words = []
        for r in rows:
            hb = [_fp16_high_byte(v / 2.0) for v in r]
            lo = hb[0] | hb[1] << 8 | hb[2] << 16 | hb[3] << 24
            hi = hb[4] | hb[5] << 8 | hb[6] << 16 | hb[7] << 24
            words.append(f"{{0x{lo:08x}u,0x{hi:08x}u}}")
        lines.append(f"static __device__ const uint2 {name}[256] = {{{','.join(words)}}};")

    f32_array("kE8pAbsF32", e8p, "static __device__ const")
    f32_array("kE81BitF32", onebit, "static __device__ const")
    f32_array("kE8pAbsF32Host", e8p, "static const")
    f32_array("kE81BitF32Host", onebit, "static const")
    hb_array("kE8pHiBytes", e8p)
    hb_array("kE81BitHiBytes", onebit)
    cos_v, sin_v = [], []
    for p in PRIMES:
        for k in range(p):
            cos_v.append(_float_lit(math.cos(2.0 * math.pi * k / p)))
            sin_v.append(_float_lit(math.sin(2.0 * math.pi * k / p)))
    lines.append(f"static __constant__ float kDftCos[{len(cos_v)}] = {{{','.join(cos_v)}}};")
    lines.append(f"static __constant__ float kDftSin[{len(sin_v)}] = {{{','.join(sin_v)}}};")
    _write_if_changed(path, "\n".join(lines) + "\n")


TWIDDLE_N = 8192


def generate_twiddles_inc(path: str) -> None:
    """exp(-2 pi i e / 8192) for e < 8192 as float2 (cos, -sin), rounded from double:
    the twiddles of the decode-batch FFT row kernels (qs_xsmall.cu)."""
    vals = []
    for e in range(TWIDDLE_N):
        a = 2.0 * math.pi * e / TWIDDLE_N
        vals.append(f"{{{_float_lit(math.cos(a))},{_float_lit(-math.sin(a))}}}")
    small = []
    for e in range(16):  # w_32^e: the in-register DFTs' constants (constant-bank operands)
        a = 2.0 * math.pi * e / 32
        small.append(f"{{{_float_lit(math.cos(a))},{_float_lit(-math.sin(a))}}}")
    text = ("// GENERATED by quipsharp_b200/build_native.py -- do not edit.\n"
            f"static __device__ const float2 kTwiddle{TWIDDLE_N}[{TWIDDLE_N}] = {{{','.join(vals)}}};\n"
            f"static __constant__ float2 kTw32[16] = {{{','.join(small)}}};\n")
    _write_if_changed(path, text)


def _write_if_changed(path: str, text: str) -> None:
    old = open(path).read() if os.path.exists(path) else None
    if old != text:
        with open(path, "w") as f:
            f.write(text)


SOURCES = ["qs_abi.cu", "qs_decode.cu", "qs_transform.cu", "qs_pack.cu", "qs_gemv.cu",
           "qs_xform_a.cu", "qs_xform_b.cu", "qs_xform_c.cu", "qs_xform_d.cu", "qs_xform_e.cu", "qs_xform_f.cu",
           "qs_noalloc.cu", "qs_gemm_tc.cu", "qs_xform2.cu", "qs_tp.cu", "qs_fit.cu", "qs_xsmall.cu",
           "qs_cache.cu", "qs_beam.cu", "qs_attn_decode.cu", "qs_attn_window.cu"]


def _compile(src: str, obj: str, verbose: bool) -> None:
    cmd = [_nvcc(), *ARCH_FLAGS, "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC",
           "-Xcompiler", "-fvisibility=hidden", "--expt-relaxed-constexpr",
           "-I", BUILD, "-I", CSRC, "-I", os.path.join(REPO, "include"),
           "-c", src, "-o", obj]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if verbose or res.returncode != 0:
        sys.stdout.write(res.stdout)
        sys.stderr.write(res.stderr)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src}")


def build(verbose: bool = False, force: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    os.makedirs(LIBDIR, exist_ok=True)
    generate_tables_inc(os.path.join(BUILD, "qs_tables_gen.inc"))
    generate_twiddles_inc(os.path.join(BUILD, "qs_twiddle_gen.inc"))
    # every translation unit depends on its own source and on all shared headers
    headers = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if not f.endswith(".cu")] + \
        [os.path.join(BUILD, "qs_tables_gen.inc"), os.path.join(BUILD, "qs_twiddle_gen.inc"),
         os.path.join(REPO, "include", "quipsharp_b200.h")]
    newest_header = max(os.path.getmtime(d) for d in headers)
    objs, jobs = [], []
    for s in SOURCES:
        src = os.path.join(CSRC, s)
        obj = os.path.join(BUILD, s.replace(".cu", ".o"))
        objs.append(obj)
        newest_dep = max(newest_header, os.path.getmtime(src))
        if force or not os.path.exists(obj) or os.path.getmtime(obj) < newest_dep:
            jobs.append((src, obj))
    with cf.ThreadPoolExecutor(max_workers=max(1, min(len(jobs), os.cpu_count() or 1))) as ex:
        for fut in [ex.submit(_compile, s, o, verbose) for s, o in jobs]:
            fut.result()
    lib = os.path.join(LIBDIR, LIBNAME)
    if jobs or not os.path.exists(lib):
        cmd = [_nvcc(), *ARCH_FLAGS, "-shared", "-Xcompiler", "-fPIC", "-o", lib, *objs]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            sys.stderr.write(res.stdout + res.stderr)
            raise RuntimeError("link failed")
    build_fast(verbose, force)
    return lib


def build_fast(verbose: bool, force: bool) -> str | None:
    """The Python extension with the decoding operators' direct calls, linked to the library;
    None where there is no compiler or are no headers for it (the calls then go by ctypes)."""
    import sysconfig

    import torch
    src, out = os.path.join(CSRC, "qs_fast.cpp"), os.path.join(LIBDIR, "_fast.so")
    newest = max(os.path.getmtime(src), os.path.getmtime(os.path.join(REPO, "include", "quipsharp_b200.h")))
    # what it was built for: torch's C++ interface changes between versions
    stamp, built_for = os.path.join(BUILD, "_fast.built_for"), f"torch {torch.__version__}, Python {sys.version}\n"
    known = os.path.exists(stamp) and open(stamp).read() == built_for
    if not force and known and os.path.exists(out) and os.path.getmtime(out) >= newest:
        return out
    inc = os.path.join(os.path.dirname(torch.__file__), "include")
    cuda = os.path.join(os.path.dirname(os.path.dirname(_nvcc())), "include")
    cxx, python = os.environ.get("CXX") or "g++", sysconfig.get_paths()["include"]
    for what, there in (("a C++ compiler", shutil.which(cxx)), ("Python's headers", os.path.exists(os.path.join(python, "Python.h"))),
                        ("torch's headers", os.path.exists(os.path.join(inc, "ATen", "ATen.h")))):
        if not there:
            sys.stderr.write(f"{os.path.basename(out)} is not built, for want of {what}: decoding calls go by ctypes\n")
            if os.path.exists(out):  # older than what it calls
                os.remove(out)
            return None
    cmd = [cxx, "-O2", "-std=c++17", "-shared", "-fPIC",
           "-fvisibility=hidden", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-I", python, "-I", inc,
           "-I", os.path.join(inc, "torch", "csrc", "api", "include"), "-I", cuda,
           src, "-o", out, "-L", LIBDIR, f"-l:{LIBNAME}", "-Wl,-rpath,$ORIGIN",
           # torch's own libraries are loaded by the time this is
           "-L", os.path.join(os.path.dirname(inc), "lib"), "-ltorch_python",
           "-ltorch_cuda", "-ltorch_cpu", "-lc10_cuda", "-lc10"]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError(f"g++ failed on {src}")
    _write_if_changed(stamp, built_for)
    return out


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv, force="-f" in sys.argv))
