"""Beam search on the CPU: the argument checks of the entry points, the facts that the
selection and the fork rest on, and the accuracy that the kernels' comments state."""
import ctypes
import os
import re
import subprocess
from decimal import Decimal, getcontext

import numpy as np
import pytest

import beam_util

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "gemma4.pas_b200")
BEAM = open(os.path.join(PKG, "csrc", "g4s_beam.cu")).read()
f32 = np.float32


def test_arguments(tmp_path, g4):
    exe = str(tmp_path / "beam_args")
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    subprocess.run(["g++", "-std=c++17", "-x", "c++", "-O0", "-I", os.path.join(ROOT, "include"), "-I", f"{cuda}/include",
                    os.path.join(ROOT, "tests", "cpp", "beam_args.cpp"), "-o", exe, "-L", PKG, "-lg4sampler",
                    f"-Wl,-rpath,{PKG}", "-L", f"{cuda}/lib64", "-lcudart", f"-Wl,-rpath,{cuda}/lib64", "-ldl", "-lpthread"],
                   check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr


def test_records(g4):
    # as the C compiler lays them out on this platform, and as the Pascal records do
    assert ctypes.sizeof(g4.BeamParams) == 64
    assert [getattr(g4.BeamParams, f).offset for f in ("beams", "n_out", "temperature", "length_alpha", "pad_token", "n_eos",
                                                       "eos")] == [0, 4, 8, 16, 24, 28, 32]
    assert ctypes.sizeof(g4.BeamTensor) == 64 and g4.BeamTensor.seg_bytes.offset == 56
    assert ctypes.sizeof(g4.PagePool) == 40 and ctypes.sizeof(g4.PageCache) == 24
    assert ctypes.sizeof(g4.BeamPages) == 72 and g4.BeamPages.result.offset == 64
    p = g4.BeamParams()
    g4.load().g4s_beam_params_defaults(ctypes.byref(p))
    assert (p.beams, p.n_out, p.temperature, p.length_alpha, p.pad_token, p.n_eos) == (4, 4, 1.0, 0.0, 0, 3)
    assert list(p.eos)[:3] == [1, 106, 50]
    header = open(os.path.join(ROOT, "include", "g4sampler.h")).read()
    for name in ("BEAM_MAX", "BEAM_MAX_OUT", "BEAM_MAX_EOS", "BEAM_MAX_TENSORS", "PAGES_MAX_POOLS", "PAGES_MAX_SEQS"):
        assert int(re.search(rf"#define G4S_{name}\s+(\d+)", header).group(1)) == getattr(g4, name)


# ---------------------------------------------------------------------------
# selection
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("seed", range(40))
def test_the_best_tokens_lie_in_the_best_items(seed):
    """The N best tokens of several beams lie in the N items whose best tokens rank first, in those among each beam's
    N best items, above the beam's best item left out, and at or above the bound of any beam's N-th item."""
    rng = np.random.default_rng(seed)
    W, V, L = int(rng.integers(1, 5)), int(rng.integers(1, 80)), int(rng.integers(1, 9))
    N = int(rng.integers(1, 12))
    x = rng.integers(0, int(rng.integers(2, 30)), (W, V)).astype(float)  # ties
    base = rng.integers(0, 3, W) * 1.0
    order = lambda w, v, i: (-(base[w] + v), w, -v, i)
    tokens = sorted((order(w, x[w, i], i), w, i) for w in range(W) for i in range(V))[:N]
    items = []
    for w in range(W):
        mine = [(order(w, x[w, s:s + L].max(), s // L), w, s // L) for s in range(0, V, L)]
        items += sorted(mine, key=lambda t: t[0])[:N]
    items.sort()
    chosen = items[:N]
    places = {(w, it): j for j, (_, w, it) in enumerate(chosen)}
    bound = max([sorted(t[0][0] for t in items if t[1] == w)[N - 1] * -1 for w in range(W)
                 if sum(t[1] == w for t in items) == N], default=-np.inf)
    for key, w, i in tokens:
        assert (w, i // L) in places
        assert -key[0] >= bound or len(items) < N
        out = [t for t in items[N:] if t[1] == w]
        if out:  # a key at or above the best item left out
            assert x[w, i] >= max(-t[0][2] for t in out)
        # no more than N - j of the item in place j
        j = places[(w, i // L)]
        assert sum(1 for _, v, k in tokens if (v, k // L) == (w, i // L)) <= N - j


def coefficients(name):
    m = re.search(name + r"\[\d\] = \{([^}]*)\}", BEAM)
    return [float(v) for v in m.group(1).split(",")]


def test_folded_softcap_polynomial():
    c = coefficients("BEAM_TH")
    P = lambda q: q * (1 + q * q * (c[0] + q * q * (c[1] + q * q * (c[2] + q * q * c[3]))))
    q = np.linspace(1e-4, 0.5, 200001)
    assert np.abs(P(q) / np.tanh(q) - 1).max() < 1.6e-8
    # below -1/2: monotone, to -inf, and with the load's maximum at or above 0 and cap >= 28 T, 2047 other logits
    # anywhere there cost under 1e-7 of the load's sum
    q = np.linspace(0.5, 40, 400001)
    assert (np.diff(P(q)) > 0).all() and c[3] > 0
    for z in (28.0, 30.0, 60.0):
        true = np.exp(-z * np.tanh(q))
        off = np.abs(np.exp(-z * P(q)) - true)
        assert (2047 * off / (1 + 2047 * true)).max() < 1e-7


def split(x):
    h = f32(x)
    return h, f32(Decimal(x) - Decimal(float(h)))


class Pairs:
    """The kernels' sums of two fp32 numbers, operation by operation."""

    @staticmethod
    def fma(a, b, c):
        return f32(np.longdouble(a) * np.longdouble(b) + np.longdouble(c))

    @staticmethod
    def sum(a, b):
        s = f32(a + b)
        bb = f32(s - a)
        return s, f32(f32(a - f32(s - bb)) + f32(b - bb))

    @staticmethod
    def norm(a, b):
        s = f32(a + b)
        return s, f32(b - f32(s - a))

    @classmethod
    def mul(cls, a, b):
        p = f32(a[0] * b[0])
        return cls.norm(p, cls.fma(a[0], b[1], cls.fma(a[1], b[0], cls.fma(a[0], b[0], -p))))

    @classmethod
    def exp(cls, z):
        t = f32(np.rint(f32(z[0] * f32(5.770780087))))
        n = int(t)
        f = cls.sum(cls.fma(t, f32(-0.17328643798828125), z[0]), cls.fma(t, f32(-3.571516913e-07), z[1]))
        g = f32(f[0] * f[0])
        gl = cls.fma(f[0], f[0], -g)
        c = cls.fma(f[0], f32(1 / 720), f32(1 / 120))
        c = cls.fma(f[0], c, f32(1 / 24))
        c = cls.fma(f[0], c, f32(1 / 6))
        cubic = f32(f32(f[0] * g) * c)
        s = cls.sum(f[0], f32(f32(0.5) * g))
        s = cls.norm(s[0], f32(f32(s[1] + f[1]) + f32(cls.fma(f32(0.5), gl, f32(f[0] * f[1])) + cubic)))
        o = cls.sum(f32(1), s[0])
        e = cls.norm(o[0], f32(o[1] + s[1]))
        root = [(f32(1), f32(0)), (f32(1.189207077), f32(3.797635273e-08)), (f32(1.414213538), f32(2.420323497e-08)),
                (f32(1.681792855), f32(-2.475532668e-08))][n & 3]
        v = cls.mul(e, root)
        return tuple(f32(np.ldexp(float(x), n >> 2)) for x in v)

    @classmethod
    def log(cls, s):
        y = f32(f32(np.log2(float(s[0])) * (1 + 1e-7)) * f32(0.693147181))  # (a first value off by an ulp or so)
        u = cls.mul(s, cls.exp((f32(-y), f32(0))))
        d = f32(f32(u[0] - f32(1)) + u[1])
        return cls.norm(y, cls.fma(f32(f32(-0.5) * d), d, d))


def test_constants_of_the_pairs_are_the_kernels():
    getcontext().prec = 40
    for i in (1, 2, 3):
        h, l = split(Decimal(2) ** (Decimal(i) / 4))
        assert f"{h:.9f}f, {l:.9e}f" in BEAM
    ln2 = Decimal(2).ln()
    assert f"{f32(4 / ln2):.9f}f" in BEAM
    assert f"{f32(ln2 / 4 - Decimal(0.17328643798828125)):.9e}f" in BEAM


def test_pairs_are_as_exact_as_stated():
    rng = np.random.default_rng(0)
    value = lambda p: np.longdouble(float(p[0])) + np.longdouble(float(p[1]))
    for x in np.concatenate([rng.uniform(-60, 60, 1500), rng.uniform(-0.3, 0.3, 500)]):
        z = split(float(x))
        e = Pairs.exp(z)
        true = np.exp(value(z))
        assert abs(value(e) / true - 1) < 3e-11
    for x in np.concatenate([rng.uniform(1, 3e5, 500), 2.0 ** rng.uniform(-50, 50, 500)]):
        s = split(float(x))
        assert abs(value(Pairs.log(s)) - np.log(value(s))) < 1e-10
    # cap tanh(l / cap) / T from them
    for cap, T in ((30.0, 0.7), (30.0, 1.0), (5.0, 2.0)):
        inv, scale = split(1 / cap), split(cap / T)
        for l in np.concatenate([rng.normal(0, 8, 300), rng.uniform(-200, 200, 100), rng.normal(0, 0.01, 100)]).astype(f32):
            b = f32(2 * min(abs(l), f32(20 * cap)))
            z = f32(b * inv[0])
            e = Pairs.exp((z, Pairs.fma(b, inv[1], Pairs.fma(b, inv[0], -z))))
            d = Pairs.sum(e[0], f32(1))
            dl = f32(d[1] + e[1])
            w = f32(1 / d[0])
            off = f32(Pairs.fma(-d[0], w, f32(1)) - f32(dl * w))
            th = Pairs.sum(f32(1), f32(-2 * w))
            x = Pairs.mul(Pairs.norm(th[0], f32(th[1] - f32(f32(2 * w) * off))), scale)
            assert abs(float(value(x)) - cap / T * np.tanh(abs(float(l)) / cap)) < 3e-11 * cap / T


# ---------------------------------------------------------------------------
# pages
# ---------------------------------------------------------------------------
def test_writers_of_a_shared_page():
    """Of w writers of a page with r holds the first min(w, r - 1) copy it: the closed form that every sequence can
    evaluate for itself, against going through the sequences one by one."""
    rng = np.random.default_rng(1)
    for _ in range(1500):
        P, width, n_pages, n = (int(rng.integers(*r)) for r in ((1, 5), (1, 6), (3, 40), (1, 6)))
        lens = rng.integers(0, width * P + 1, n)
        tables = rng.integers(0, n_pages, (n, width))
        refs = np.zeros(n_pages, np.int64)
        for i in range(n):
            np.add.at(refs, tables[i, :-(-int(lens[i]) // P)], 1)
        refs += rng.random(n_pages) < 0.1
        src = rng.integers(-1, n, int(rng.integers(1, 9)))
        n_new, frozen = int(rng.integers(0, 4)), rng.random(src.size) < 0.3
        _, _, _, result, copies = beam_util.fork(tables, lens, refs, src, n_new, P, width, frozen)
        after = refs.copy()
        for i in range(n):
            np.add.at(after, tables[i, :-(-int(lens[i]) // P)], int((src == i).sum()) - 1)
        last = [int(tables[s, lens[s] // P]) if s >= 0 and n_new and lens[s] % P and not z else -1 for s, z in zip(src, frozen)]
        need, want = 0, []
        for j, s in enumerate(src):
            if s < 0 or not n_new or frozen[j]:
                continue
            c = last[j] >= 0 and last[:j].count(last[j]) < after[last[j]] - 1
            grown = -(-(int(lens[s]) + n_new) // P)
            if grown <= width:
                need += int(c) + grown - -(-int(lens[s]) // P)
                if c:
                    want.append((last[j], int(lens[s]) % P))
        free = int((after <= 0).sum())
        assert result[1] == max(0, need - free)
        if not any(result[1:]):
            assert result[0] == need and [(a, f) for a, _, f in copies] == want


def test_compaction_pairs_holes_with_pages_above():
    rng = np.random.default_rng(2)
    for _ in range(300):
        n = int(rng.integers(1, 60))
        refs = np.where(rng.random(n) < rng.random(), rng.integers(1, 4, n), -rng.integers(0, 2, n))
        _, new_refs, page_map, moves, result = beam_util.compact(np.zeros((0, 1), np.int64), [], refs, 4, 1)
        used = int((refs > 0).sum())
        below = int((refs[:used] > 0).sum())
        # the ranks a warp computes from the used pages below its own
        before = np.concatenate([[0], np.cumsum(refs > 0)])
        for k, (a, b) in enumerate(moves.reshape(-1, 2)):
            assert before[a] - below == k and b - before[b] == k
        assert result[:2] == [used, used - below] and (new_refs[:used] > 0).all() and not new_refs[used:].any()
