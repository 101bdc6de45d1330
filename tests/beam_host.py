"""Device functions of the beam selection compiled for the host from the kernels' own source, operation by
operation: fp32 arithmetic without contraction, CUDA's intrinsics as the IEEE operations that they stand for."""
from __future__ import annotations

import os
import re
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "gemma4.pas_b200", "csrc")

SHIM = r"""
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
using std::max;
using std::min;
#define __device__
#define __forceinline__ inline
#define __noinline__
static inline uint32_t __float_as_uint(float f) { uint32_t u; memcpy(&u, &f, 4); return u; }
static inline float __uint_as_float(uint32_t u) { float f; memcpy(&f, &u, 4); return f; }
static inline float __fadd_rn(float a, float b) { return a + b; }
static inline float __fsub_rn(float a, float b) { return a - b; }
static inline float __fmul_rn(float a, float b) { return a * b; }
static inline float __fmaf_rn(float a, float b, float c) { return fmaf(a, b, c); }
static inline float __frcp_rn(float a) { return 1.0f / a; }
static inline float __fdividef(float a, float b) { return a / b; }
// the hardware's approximations (2^-22 of 2^y, a subnormal result is 0; an ulp or so of log2)
static inline float ex2_approx(float y) { const double r = std::exp2((double)y); return r < 0x1p-126 ? 0.0f : (float)(r * (1 + 1.5e-7)); }
static inline float lg2_approx(float x) { return (float)(std::log2((double)x) * (1 + 1e-7)); }
"""


def between(text, first, last):
    a = text.index(first)
    return text[a:text.index(last, a)]


def function(text, head):
    """A function's text, from `head` to its closing brace in the first column (or on the same line)."""
    a = text.index(head)
    line = text[a:text.index("\n", a)]
    return line if line.rstrip().endswith("}") else text[a:text.index("\n}\n", a) + 3]


def build(tmp_path, name, main, extra=""):
    """An executable of the kernels' pair routines and rank, `extra` and a main()."""
    beam = open(os.path.join(CSRC, "g4s_beam.cu")).read()
    device = open(os.path.join(CSRC, "g4s_device.cuh")).read()
    code = SHIM + "\n".join(function(device, f"__device__ __forceinline__ {h}") for h in ("float pow2i", "uint32_t f2key", "float key2f"))
    code += "\n" + between(beam, "struct Pair {", "// What a logit adds to its row's base")
    code = re.sub(r'asm\("lg2\.approx\.ftz\.f32[^;]*;"[^;]*;', "y = lg2_approx(s.h);", code)
    code += between(beam, "// A pair as a whole number", "__device__ __forceinline__ uint64_t pair_bits")
    src, exe = str(tmp_path / f"{name}.cpp"), str(tmp_path / name)
    with open(src, "w") as f:
        f.write(code + extra + main)
    subprocess.run(["g++", "-std=c++17", "-O1", "-ffp-contract=off", "-fwrapv", "-o", exe, src], check=True)
    return exe


def run(exe, lines):
    r = subprocess.run([exe], input="\n".join(lines) + "\n", capture_output=True, text=True, check=True)
    return r.stdout.split("\n")[:-1]
