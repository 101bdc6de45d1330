"""A search whose page pool runs short in some steps, and recovers as the integration notes say: pages are freed, and
g4s_pages_fork grows the rows as they are (src[j] = j, or -1 where the step left no beam), with the ended beams
frozen and the tables in the other buffer once more."""
import numpy as np
import pytest

from test_gpu_pages import Search

pytestmark = pytest.mark.gpu


class Shortage(Search):
    def __init__(self, torch, g4, sampler, G, W, P, seed, free):
        super().__init__(torch, g4, sampler, G, W, 97, P, seed, 0.6)
        self.held = (self.refs == 0).nonzero()[:, 0].tolist()  # by a prefix cache, all but `free`
        self.held = self.held[free:] if free is not None else []
        self.refs[self.held] = 1
        self.i, self.recoveries = 0, 0

    def model(self, t):
        super().model()
        if t == 3:  # one beam of the first prompt goes on, the others have no token left
            self.logits[1:self.W] = -float("inf")

    def advance(self, t, stream):
        self.model(t)
        self.step(self.i, stream.cuda_stream)
        short = self.result.tolist()
        assert short[2:] == [0, 0] and (short[1] == 0 or short[0] == 0)
        if short[1]:
            # the fork alone is done: as many pages as are missing are given up by the other holder
            self.recoveries += 1
            give, self.held = self.held[:short[1]], self.held[short[1]:]
            self.refs[give] = 0
            self.i += 1
            a, b = self.tab[self.i % 2], self.tab[1 - self.i % 2]
            rows = self.G * self.W
            src = self.torch.arange(rows, dtype=self.torch.int32, device="cuda")
            src[self.par < 0] = -1
            self.s.pages_fork(self.cache, rows, a.data_ptr(), self.plens.data_ptr(), self.refs.data_ptr(), rows,
                              src.data_ptr(), 1, b.data_ptr(), self.plens.data_ptr(), self.refs.data_ptr(),
                              self.result.data_ptr(), frozen_ptr=self.done.data_ptr(), stream=stream.cuda_stream)
            assert self.result.tolist()[1:] == [0, 0, 0]
        self.write(self.i)
        self.i += 1

    def sequences(self):
        tab, lens, pool = self.tab[self.i % 2].cpu().numpy(), self.plens.cpu().numpy(), self.pool.cpu().numpy()
        count = np.zeros(self.n_pages, np.int64)
        out = []
        for r in range(self.G * self.W):
            n = int(lens[r])
            out.append([int(pool[tab[r, t // self.P], t % self.P]) for t in range(n)])
            count[tab[r, :-(-n // self.P)]] += 1
        count[self.held] += 1
        assert np.array_equal(count, self.refs.cpu().numpy())  # nothing leaked
        return out


@pytest.mark.parametrize("G,W,P,free", [(1, 4, 4, 0), (3, 5, 3, 4), (2, 8, 16, 1)])
def test_a_search_goes_on_after_a_shortage(sampler, g4, torch_cuda, G, W, P, free):
    torch = torch_cuda
    rich = Shortage(torch, g4, sampler, G, W, P, 31 * G + W, None)
    poor = Shortage(torch, g4, sampler, G, W, P, 31 * G + W, free)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        for t in range(12):
            for s in (rich, poor):
                s.advance(t, stream)
            for name in ("scores", "lens", "done", "par", "tok", "plens", "last"):
                assert torch.equal(getattr(rich, name), getattr(poor, name)), (t, name)
            assert rich.sequences() == poor.sequences(), t
    torch.cuda.synchronize()
    assert rich.recoveries == 0 and poor.recoveries > 0
