"""Beam selection's scores against 64 bits, at every temperature and softcap: row by row, with a bound of what each
row's own terms can be off by."""
import numpy as np
import pytest

import beam_util
from test_gpu_beam import LOW, Case, logits

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # half a step of fp32, relative


def bound(x, cap, T):
    """Of a row's log-sum-exp and of x(top), without the score's own rounding.

    The sum: a lane's packed sums take up to 32 terms of a 4 KiB load each and are joined over 2 + 5 steps, one more a
    load; the exponential is off by 2^-22 (4 U), in a term and where a sum moves to a new maximum (up to 8 loads of an
    item here) or to the row's.  A term's argument y is rounded to U |y|, which weighs E = sum p_i (x_top - x_i).
    The pairs: 3e-11 of cap / T, for the top and for the token.
    The arguments, up to cap / T = 64: s k is a product of a polynomial of s(l) / l, whose last step rounds to U and whose
    others to U of what they add (c = 1.3 up to cap / 2, 2 up to cap), or of the tanh with 4 roundings (c = 4); the
    maximum's own is common to all terms, so that each counts with the weight of the others.
    Beyond: below cap / 2, up to 512, only the polynomial's rest, under 0.0356 cap, is rounded (2.5 U of it, in a term
    and in the maximum's); else a difference has 27 roundings of itself (beam_below), which weighs E."""
    v = np.minimum(x[x > -1e30], -LOW["bf16"])
    s = cap * np.tanh(v / cap) if cap > 0 else v
    z = (s - s.max()) / T
    p = np.exp(z)
    p /= p.sum()
    E = float(np.sum(p * -z))
    total = (32 + 7 + 8 + 4 * (1 + 8 + 1)) * U + U * E
    if cap <= 0:
        return total + 2 * U * E
    total += 2 * 3e-11 * cap / T
    if cap / T <= 64:
        c = np.where(np.abs(v) <= cap / 2, 1.3, np.where(np.abs(v) <= cap, 2.0, 4.0))
        off = c * np.abs(s) / T * U
        i = int(np.argmax(v))
        return total + float(np.sum(p * off) - p[i] * off[i] + (1 - p[i]) * off[i])
    return total + (5 * 0.0356 * cap / T * U if cap / T <= 512 else 0.0) + 27 * U * E


def spread(rng, rows, V, cap, T):
    return logits(rng, rows, V)


def near(top, wide=3.0):
    """An eighth of the row within a few T of its largest, at `top` (in caps)."""
    def make(rng, rows, V, cap, T):
        x = rng.standard_normal((rows, V)) * 2.5 + min(top * cap, 0)
        x = np.minimum(x, top * cap - 1e-3 * cap)
        n = max(1, V // 8)
        np.put_along_axis(x, rng.integers(0, V, (rows, n)), top * cap - rng.exponential(wide * T, (rows, n)), 1)
        return x
    return make


KINDS = {"spread": spread, "below half the cap": near(0.45), "about half the cap": near(0.502), "below the cap": near(0.97),
         "about the cap": near(1.001), "twice the cap": near(2.0, 30.0), "saturated": near(9.0, 1e4), "negative": near(-0.3),
         "far negative": near(-1.2)}


def check(torch, g4, sampler, x, dtype, cap, T, N=3, **kw):
    """Every row a prompt of one beam: its N best tokens' scores, and their order."""
    c = Case(torch, g4, x, dtype, 1, N, scores=np.zeros(x.shape[0]), cap=cap, T=T, **kw)
    s, _, _, p, t = c.run(sampler)
    want = beam_util.select(c.x, c.scores, c.lens, c.done, 1, N, cap, T, 0.0, 7, fmax=-LOW[dtype])
    for r, cand in enumerate(want):
        n = min(N, len(cand))
        if n == 0:
            assert (t[r] == -1).all()
            continue
        assert t[r, :n].tolist() == [k[3] for k in cand[:n]], r
        tol = bound(c.x[r], cap, T)
        for i in range(n):
            assert abs(float(s[r, i]) - cand[i][1]) <= tol + U * abs(cand[i][1]), (r, i, s[r, i], cand[i][1], tol)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("cap,T", [(30.0, 2.0), (30.0, 1.0), (30.0, 0.5), (30.0, 0.46), (30.0, 0.2), (30.0, 0.06), (30.0, 0.05),
                                   (30.0, 1e-2), (30.0, 1e-3), (30.0, 1e-5), (5.0, 1.0), (5.0, 0.03), (1000.0, 3.0),
                                   (1000.0, 0.5), (2e4, 1.0), (1e6, 0.01), (1e-3, 1.0), (1e-3, 1e-5)])
def test_scores(sampler, g4, torch_cuda, cap, T, kind, dtype):
    rng = np.random.default_rng(int(cap * 7) + len(kind))
    for V, pad, offset in ((9000, 0, 0), (40003, 2, 1)):  # items of parts of a load and of one, aligned and not
        check(torch_cuda, g4, sampler, KINDS[kind](rng, 6, V, cap, T), dtype, cap, T, pad=pad, offset=offset)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["spread", "about half the cap", "about the cap"])
@pytest.mark.parametrize("cap,T", [(30.0, 1.0), (30.0, 0.1), (30.0, 1e-3)])
def test_scores_of_long_rows(g4, torch_cuda, cap, T, kind, dtype):
    """Items of several loads: their maxima move from one way through a load to another."""
    rng = np.random.default_rng(11)
    with g4.Sampler(0, 4, 700_000) as s:
        x = KINDS[kind](rng, 4, 700_000, cap, T)
        step = 2048 if dtype == "bf16" else 1024
        x[1] -= 30.0 * (np.arange(x.shape[1]) // step % 3 == 0)  # loads far below their neighbours
        x[2, ::step * 2] = 1.4 * cap
        x[3] = np.where(rng.random(x.shape[1]) < 1e-4, np.nan, x[3])
        check(torch_cuda, g4, s, x, dtype, cap, T)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T", [0.4, 1e-2, 1e-4])
def test_masks_at_low_temperatures(sampler, g4, torch_cuda, T, dtype):
    rng = np.random.default_rng(5)
    x = logits(rng, 12, 7001)
    x[0][rng.random(7001) < 0.97] = -np.inf
    x[1][rng.random(7001) < 0.5] = LOW[dtype]
    x[2][rng.random(7001) < 0.3] = np.nan
    x[3] = -np.inf
    x[4] = -25.0 - rng.random(7001)
    x[4][rng.random(7001) < 0.5] = -np.inf  # (masked among negative ones: no polynomial reaches below them)
    x[5, [7, 900]] = np.inf
    x[6] *= 40.0
    x[7] = np.where(np.arange(7001) == 5000, 3.0, -np.inf)
    x[8] = -9e29
    x[9] = 0.0
    x[10] = np.where(rng.random(7001) < 0.5, -0.0, 0.0)
    for offset in (0, 3):
        check(torch_cuda, g4, sampler, x, dtype, 30.0, T, N=5, offset=offset)


def test_refuses_what_the_pairs_cannot_tell_apart(sampler, g4, torch_cuda):
    c = Case(torch_cuda, g4, np.zeros((4, 64)), "f32", 4, 4)
    args = (c.ptr, g4.F32, 1, 64, 64)
    out = (c.state(c.d), c.state(c.out[:3]), c.out[3].data_ptr(), c.out[4].data_ptr())
    for cap, T in ((1e6, 0.009), (200.0, 1e-6)):
        assert sampler.beam_select(*args, cap, g4.make_beam_params(4, 4, T), *out, check=False) == g4.ERR_ARG
        assert "softcap" in sampler.last_error() and "temperature" in sampler.last_error()
    assert sampler.beam_select(*args, 0.0, g4.make_beam_params(4, 4, 1e-6), *out, check=False) == g4.OK
    torch_cuda.cuda.synchronize()
