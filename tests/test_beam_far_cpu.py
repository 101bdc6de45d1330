"""Differences of softcapped logits as the selection takes them at low temperatures: the kernels' own routines on the
host, against 60 digits."""
import re
from decimal import Decimal, getcontext

import numpy as np
import pytest

import beam_host

MAIN = r"""
int main()
{
    double cap, T;
    float m, l;
    while (scanf("%lf %lf %a %a", &cap, &T, &m, &l) == 4) {
        BeamArgs a{};
        const double k = 1.4426950408889634074 / T, two = 2.0 * 1.4426950408889634074 / (double)(float)cap;
        a.softcap = (float)cap;
        a.invcap = (float)(1.0 / (double)a.softcap);
        a.two2[0] = (float)two;
        a.two2[1] = (float)(two - (double)a.two2[0]);
        a.capk2 = (float)(2.0 * a.softcap * k);
        a.sat = 64.0f * a.softcap;
        printf("%a %a\n", beam_below(a, m, l), beam_nothing(a, m));
    }
    return 0;
}
"""


@pytest.fixture(scope="module")
def exe(tmp_path_factory):
    text = open(beam_host.CSRC + "/g4s_beam.cu").read()
    device = open(beam_host.CSRC + "/g4s_device.cuh").read()
    extra = "\n".join(re.findall(r"^#define G4_(?:TH\d|L2E) .*$", device, re.M))
    extra += "\nstruct BeamArgs { float softcap, invcap, two2[2], capk2, sat; };\n"
    extra += beam_host.function(device, "__device__ __forceinline__ float tanh_poly")
    for name in ("beam_e2", "beam_below", "beam_nothing"):
        body = beam_host.function(text, f"__device__ __forceinline__ float {name}")
        extra += re.sub(r'asm\("lg2\.approx[^;]*;"[^;]*;', "lg = lg2_approx((2.0f - u) / u);", body)
    return beam_host.build(tmp_path_factory.mktemp("far"), "far", MAIN, extra)


def tanh(v):
    e = (-2 * abs(v)).exp()
    t = (1 - e) / (1 + e)
    return t if v >= 0 else -t


@pytest.mark.parametrize("cap,T", [(30.0, 0.4), (30.0, 1e-3), (30.0, 1e-6), (5.0, 0.01), (1e6, 0.02), (1e-6, 1e-9)])
def test_differences_are_exact_to_a_few_steps_of_themselves(exe, cap, T):
    getcontext().prec = 60
    rng = np.random.default_rng(int(1 / T))
    c = np.float32(cap)
    m = np.concatenate([rng.normal(0, 0.4, 300), rng.uniform(-12, 12, 300), rng.normal(0, 1e-4, 50), [0.0, 40.0, -40.0]]) * cap
    gap = np.concatenate([np.exp(rng.uniform(-16, 3, m.size - 1)), [0.0]]) * cap
    m = m.astype(np.float32)
    l = np.minimum((m - gap).astype(np.float32), m)
    rows = beam_host.run(exe, [f"{cap!r} {T!r} {float(a).hex()} {float(b).hex()}" for a, b in zip(m, l)])
    k = Decimal(1) / (Decimal(T) * Decimal(2).ln())
    cd = Decimal(float(c))
    for a, b, row in zip(m, l, rows):
        got, none = (float.fromhex(v) for v in row.split())
        want = cd * (tanh(Decimal(float(a)) / cd) - tanh(Decimal(float(b)) / cd)) * k
        # 27 roundings of 2^-24
        assert abs(Decimal(got) - want) <= Decimal(27 * 2.0**-24) * want + Decimal(1e-30), (a, b)
        # what lies below `none` adds under 2^-64 of the maximum's term
        if np.isfinite(none):
            below = cd * (tanh(Decimal(float(a)) / cd) - tanh(Decimal(none) / cd)) * k
            assert below > 64, (a, none)
            assert none < a


def test_the_largest_and_infinite_logits_give_no_nan(exe):
    big = float(np.finfo(np.float32).max)
    lines = [f"30.0 0.001 {m.hex()} {l}" for m in (big, 1e30, 0.0, -1e29, 1e-30)
             for l in (big.hex(), "0x0p+0", (-1e29).hex(), "-inf") if l == "-inf" or float.fromhex(l) <= m]
    for line, row in zip(lines, beam_host.run(exe, lines)):
        got, none = (float.fromhex(v) for v in row.split())
        assert got >= 0.0 and np.isfinite(got), line
        assert not np.isnan(none), line
