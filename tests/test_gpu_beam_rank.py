"""Beam selection's length power where 1 / length^alpha leaves fp32's range."""
import numpy as np
import pytest

from test_gpu_beam import Case, logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("W,N", [(4, 8), (17, 20)])  # (from 16 beams on one warp a beam)
@pytest.mark.parametrize("alpha", [2.5, 5.0, 8.0])
def test_the_longest_beams_come_where_their_scaled_scores_stand(sampler, g4, torch_cuda, W, N, alpha):
    rng = np.random.default_rng(int(alpha) + W)
    G = 6
    ladder = [50_000, 56_000, 57_000, 65_000, 70_000, 1_000_000, 3, 2**30, 2**31 - 3]
    lens = np.array([ladder[int(i)] for i in rng.integers(0, len(ladder), G * W)])
    lens[:4] = [65_000, 70_000, 56_500, 50_000]  # one group of close lengths
    done = rng.random(G * W) < 0.3
    # scores in proportion to the power, so that beams of every length meet
    scores = -np.minimum((lens / 50_000.0) ** min(alpha, 3.0) * rng.uniform(1.0, 3.0, G * W), 1e6)
    c = Case(torch_cuda, g4, logits(rng, G * W, 2500), "f32", W, N, scores=scores, lens=lens, done=done, alpha=alpha)
    c.check(c.run(sampler))


def test_a_long_poor_beam_does_not_win(sampler, g4, torch_cuda):
    """Four beams of one length and one score but for a poor one: scaled, the order is that of the scores."""
    x = np.tile(logits(np.random.default_rng(1), 1, 1000), (4, 1))
    for length in (50_000, 56_500, 65_000, 70_000, 1_000_000):
        c = Case(torch_cuda, g4, x, "f32", 4, 4, scores=[-5.0, -1.0, -50.0, -2.0], lens=np.full(4, length),
                 done=np.ones(4), alpha=8.0)
        _, _, _, p, _ = c.run(sampler)
        assert p[0].tolist() == [1, 3, 0, 2], length
