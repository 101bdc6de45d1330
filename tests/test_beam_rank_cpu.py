"""The rank that beam selection orders by, score / max(length, 1)^alpha, over every accepted alpha and length:
the kernels' own routines on the host against 40 digits."""
from decimal import Decimal, getcontext

import numpy as np
import pytest

import beam_host

MAIN = r"""
int main()
{
    float score;
    int length, scaled;
    double alpha;
    while (scanf("%a %d %lf %d", &score, &length, &alpha, &scaled) == 4) {
        BeamRow r{};
        const float h = (float)alpha;
        r.inv = beam_length_power(max(length, 1), Pair{h, (float)(alpha - (double)h)});
        printf("%llu\n", (unsigned long long)beam_rank(r, Pair{score, score * 1.7e-8f}, scaled));
    }
    return 0;
}
"""


@pytest.fixture(scope="module")
def exe(tmp_path_factory):
    return beam_host.build(tmp_path_factory.mktemp("rank"), "rank", MAIN)


def ranks(exe, rows):
    return [int(v) for v in beam_host.run(exe, [f"{float(s).hex()} {n} {a!r} 1" for s, n, a in rows])]


def true(score, length, alpha):
    h = Decimal(float(np.float32(score)))
    low = Decimal(float(np.float32(np.float32(score) * np.float32(1.7e-8))))
    return (h + low) * (-(Decimal(alpha) * Decimal(max(length, 1)).ln())).exp()


@pytest.mark.parametrize("alpha", [0.6, 1.0, 2.0, 5.0, 8.0])
def test_ranks_order_as_the_scaled_scores(exe, alpha):
    getcontext().prec = 40
    rng = np.random.default_rng(int(alpha * 10))
    lengths = [0, 1, 2, 3, 50, 50000, 56000, 57000, 65000, 70000, 10**6, 2**30, 2**31 - 1]
    lengths += np.exp(rng.uniform(0, np.log(2**31 - 1), 200)).astype(int).tolist()
    rows = [(np.float32(s), n, alpha) for n in lengths
            for s in (-1e4, -37.5, -1e-3, -1e-30, 0.0, 1e-30, 2.5, 1e9, -float(rng.uniform(0.1, 100)))]
    key = ranks(exe, rows)
    want = [true(*r) for r in rows]
    at = sorted(range(len(rows)), key=lambda i: want[i])
    for a, b in zip(at, at[1:]):
        # 1e-9: the logarithm and the power are exact to 3e-11, times alpha
        if abs(want[b] - want[a]) > Decimal(1e-9) * max(abs(want[a]), abs(want[b])):
            assert key[b] > key[a], (rows[a], rows[b])


def test_one_length_keeps_the_order_of_the_scores(exe):
    """With one length the rank never falls as the score grows, neighbours among the fp32 numbers included."""
    rng = np.random.default_rng(3)
    for length, alpha in ((7, 0.6), (60000, 8.0), (2**31 - 1, 8.0), (1, 3.0)):
        s = np.float32(-np.exp(rng.uniform(-3, 8, 2000)))
        s = np.unique(np.concatenate([s, np.nextafter(s, np.float32(0)), np.nextafter(s, np.float32(-np.inf)),
                                      -np.exp2(np.arange(-5, 12)).astype(np.float32)]))
        key = ranks(exe, [(v, length, alpha) for v in s])
        assert all(b > a for a, b in zip(key, key[1:]))


def test_scores_of_1e30_or_more_keep_their_place(exe):
    key = ranks(exe, [(v, 9, 1.0) for v in (-np.inf, -3e38, -1e30, -1e20, -1.0, 0.0, 1.0, 1e20, 1e30, 3e38, np.inf)])
    assert key == sorted(set(key))
