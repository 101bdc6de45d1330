"""Beam search's selection and state reordering on the GPU against their plain 64-bit forms."""
import ctypes

import numpy as np
import pytest

import beam_util

pytestmark = pytest.mark.gpu

LOW = {"f32": np.finfo(np.float32).min, "bf16": -3.3895313892515355e38}


@pytest.fixture(scope="module")
def big(g4, torch_cuda):
    """A context for rows longer than 512 units."""
    s = g4.Sampler(device=0, max_rows=40, max_vocab=1 << 20)
    yield s
    s.close()


def tolerance(cap, T, score):
    """Bound of |score - 64-bit score|.  Softcapped logits are off by under 2.2e-7 cap, over T.  A row's sum of
    positive terms: each of a lane's four sums takes at most 8 * 4 (a 2 KiB unit of bf16, 4 units), 2 + 5 joins of
    them and of the lanes, 2^-24 each; the exponential 2^-22 there and in the joins of items; its argument's 2^-24 |y|
    weighs at most log 2^18 = 13.  The score rounds once."""
    return 2.2e-7 * max(cap, 0.0) / T + (32 + 7 + 8 + 13) * 2.0 ** -24 + np.abs(score) * 2.0 ** -24


class Case:
    """Inputs on the host and the device, and the call."""

    def __init__(self, torch, g4, x, dtype, W, N, scores=None, lens=None, done=None, cap=30.0, T=1.0, alpha=0.0,
                 pad=0, offset=0, pad_token=7, seed=0):
        rng = np.random.default_rng(seed)
        self.torch, self.g4, self.dtype, self.W, self.N = torch, g4, dtype, W, N
        self.rows, self.V = x.shape
        self.G = self.rows // W
        self.cap, self.T, self.alpha, self.pad_token = cap, T, alpha, pad_token
        self.stride = self.V + pad
        t = torch.from_numpy(np.ascontiguousarray(x, np.float32))
        buf = torch.full((self.rows * self.stride + offset,), 1e6, dtype=torch.float32)
        view = buf[offset:].view(self.rows, self.stride)
        view[:, :self.V] = t
        self.buf = buf.to(torch.float32 if dtype == "f32" else torch.bfloat16).cuda()
        self.ptr = self.buf.data_ptr() + offset * self.buf.element_size()
        self.x = self.buf[offset:].view(self.rows, self.stride)[:, :self.V].double().cpu().numpy()
        self.scores = (-rng.exponential(3.0, self.rows) if scores is None else np.asarray(scores)).astype(np.float32)
        self.lens = (rng.integers(1, 40, self.rows) if lens is None else np.asarray(lens)).astype(np.int32)
        self.done = (np.zeros(self.rows) if done is None else np.asarray(done)).astype(np.uint8)
        self.d = [torch.from_numpy(v).cuda() for v in (self.scores, self.lens, self.done)]
        n = self.G * N
        self.out = [torch.full((n + 3,), -77.0, device="cuda"), torch.full((n + 3,), -77, dtype=torch.int32, device="cuda"),
                    torch.full((n + 3,), 77, dtype=torch.uint8, device="cuda"),
                    torch.full((n + 3,), -77, dtype=torch.int32, device="cuda"),
                    torch.full((n + 3,), -77, dtype=torch.int32, device="cuda")]
        self.params = g4.make_beam_params(W, N, T, alpha, pad_token, beam_util.EOS)

    def state(self, t):
        return self.g4.BeamState(*(v.data_ptr() for v in t))

    def run(self, sampler, stream=None, in_place=False):
        after = self.d if in_place else self.out[:3]
        self.torch.cuda.synchronize()
        sampler.beam_select(self.ptr, self.g4.F32 if self.dtype == "f32" else self.g4.BF16, self.G, self.V, self.stride,
                            self.cap, self.params, self.state(self.d), self.state(after), self.out[3].data_ptr(),
                            self.out[4].data_ptr(), stream=stream)
        self.torch.cuda.synchronize()
        return self.got(after)

    def got(self, after=None):
        after = self.out[:3] if after is None else after
        n = self.G * self.N
        s, l, d, p, t = (v.cpu().numpy() for v in (*after, *self.out[3:]))
        for v, w in zip((self.out[0], *self.out[3:]), (-77.0, -77, -77)):
            assert (v.cpu().numpy()[n:] == w).all(), "wrote behind the last group"
        return tuple(v[:n].reshape(self.G, self.N) for v in (s, l, d, p, t))

    def check(self, got):
        want = beam_util.select(self.x, self.scores, self.lens, self.done, self.W, self.N, self.cap, self.T, self.alpha,
                                self.pad_token, fmax=-LOW[self.dtype])
        s, l, d, p, t = got
        for g in range(self.G):
            cand = want[g]
            n = min(self.N, len(cand))
            assert (p[g, n:] == -1).all() and (t[g, n:] == -1).all() and (s[g, n:] == -np.inf).all()
            assert (l[g, n:] == 0).all() and (d[g, n:] == 0).all()
            by = {(c[2], c[3]): c for c in cand}
            seen = set()
            for i in range(n):
                key = (int(p[g, i]), int(t[g, i]))
                assert key in by and key not in seen, (g, i, key)
                seen.add(key)
                rank, score, _, _, length, ended = by[key]
                tol = tolerance(self.cap, self.T, score)
                with np.errstate(over="ignore"):
                    if np.isfinite(np.float32(score)):
                        assert abs(float(s[g, i]) - score) <= tol, (g, i, s[g, i], score, tol)
                    else:
                        assert s[g, i] == np.float32(score)
                assert (int(l[g, i]), int(d[g, i])) == (length, ended), (g, i)
                # the place is the 64-bit order's wherever the ranks differ by more than the scores may be off
                slack = 2 * tol * max(abs(rank / score), 0.0) if score and np.isfinite(score) else 0.0
                if key != (cand[i][2], cand[i][3]):
                    assert abs(rank - cand[i][0]) <= slack, (g, i, key, cand[i])
                    assert rank != cand[i][0], ("equal ranks out of order", g, i, key, cand[i])


def logits(rng, rows, V, scale=2.5):
    x = rng.standard_normal((rows, V)) * scale
    if V > 64:
        at = rng.integers(0, V, (rows, 12))
        np.put_along_axis(x, at, rng.uniform(5, 16, (rows, 12)), 1)
    return x


SHAPES = [  # G, W, N, V, pad, offset
    (1, 1, 1, 1, 0, 0),
    (2, 1, 1, 2, 0, 0),
    (1, 4, 8, 3, 1, 0),         # fewer candidates than places
    (3, 2, 5, 31, 1, 1),
    (2, 5, 10, 511, 1, 0),
    (2, 4, 4, 512, 0, 0),
    (2, 3, 6, 513, 3, 2),
    (1, 8, 16, 1023, 1, 0),
    (2, 8, 16, 1024, 0, 0),
    (2, 2, 64, 1025, 7, 0),
    (2, 32, 64, 2049, 7, 8),
    (5, 7, 14, 32003, 2, 0),
    (2, 32, 32, 20000, 0, 0),
    (1, 4, 4, 262144, 0, 0),
    (3, 4, 8, 100001, 7, 0),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_select_shapes(sampler, g4, torch_cuda, dtype, shape):
    G, W, N, V, pad, offset = shape
    rng = np.random.default_rng(V * 7 + W)
    c = Case(torch_cuda, g4, logits(rng, G * W, V), dtype, W, N, pad=pad, offset=offset)
    c.check(c.run(sampler))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("offset", range(8))
def test_select_row_ends_at_every_alignment(sampler, g4, torch_cuda, dtype, offset):
    """Rows that end in, at and behind a load, from every place of 16 bytes on; what stands beside them is never seen."""
    rng = np.random.default_rng(offset)
    for i, V in enumerate((2, 9, 255, 1023, 1024, 1025, 1031, 2047, 2048, 2049, 4103, 6145)):
        x = logits(rng, 6, V, 2.5 if i % 3 else 30.0)  # (above the cap too: element by element)
        c = Case(torch_cuda, g4, x, dtype, 3, 5, pad=(0, 1, 2, 3, 5, 7)[(i + offset) % 6], offset=offset, alpha=0.5,
                 cap=30.0 if i % 2 else 0.0)
        rows = c.buf[offset:].view(6, c.stride)
        for beside in (1e6, np.inf, np.nan):
            c.buf[:offset] = beside
            rows[:, V:] = beside
            c.check(c.run(sampler))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_select_equal_rows_at_any_offset_score_equal(sampler, g4, torch_cuda, dtype):
    """A row's sums do not depend on where it starts: one prompt's beams of equal logits tie bit for bit."""
    for V, pad in ((97, 0), (2047, 4), (5003, 2), (40001, 0)):
        x = np.tile(logits(np.random.default_rng(V), 1, V), (8, 1))
        c = Case(torch_cuda, g4, x, dtype, 8, 16, pad=pad, scores=np.full(8, -3.0), lens=np.full(8, 2), offset=1)
        s, _, _, p, t = c.run(sampler)
        assert p[0].tolist() == list(range(8)) * 2 and len(set(t[0, :8])) == len(set(t[0, 8:])) == 1
        assert len(set(s[0, :8].tolist())) == len(set(s[0, 8:].tolist())) == 1


@pytest.mark.parametrize("max_vocab", [1, 900, 5000, 20000])
def test_select_in_a_small_context(g4, torch_cuda, max_vocab):
    """The statistics' room is sized by the context's vocabulary."""
    s = g4.Sampler(device=0, max_rows=12, max_vocab=max_vocab)
    rng = np.random.default_rng(max_vocab)
    for dtype, offset in (("f32", 0), ("f32", 3), ("bf16", 0), ("bf16", 7)):
        c = Case(torch_cuda, g4, logits(rng, 12, max_vocab), dtype, 4, 6, pad=1, offset=offset)
        c.check(c.run(s))
    s.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cap,T,alpha", [(0.0, 1.0, 0.0), (30.0, 0.5, 0.6), (0.0, 1.7, 1.0), (5.0, 1.0, 2.0),
                                         (1000.0, 0.3, 0.0), (30.0, 1e-3, 0.0), (0.01, 1.0, 0.0)])
def test_select_parameters(sampler, g4, torch_cuda, dtype, cap, T, alpha):
    rng = np.random.default_rng(5)
    done = np.arange(24) % 5 == 2
    c = Case(torch_cuda, g4, logits(rng, 24, 5003, 4.0), dtype, 6, 9, cap=cap, T=T, alpha=alpha, done=done, pad=1)
    c.check(c.run(sampler))


def mask(x, kind, rng, dtype):
    V = x.shape[1]
    if kind == "most":
        x[rng.random(x.shape) < 0.97] = -np.inf
    elif kind == "lowest":
        x[rng.random(x.shape) < 0.5] = LOW[dtype]
    elif kind == "nan":
        x[rng.random(x.shape) < 0.3] = np.nan
    elif kind == "empty rows":
        x[::3] = -np.inf
        x[1] = LOW[dtype]
        x[4] = np.nan
    elif kind == "empty group":
        x[:4] = -np.inf
    elif kind == "all":
        x[:] = -np.inf
    elif kind == "one token":
        keep = rng.integers(0, V, x.shape[0])
        y = np.full_like(x, -np.inf)
        y[np.arange(x.shape[0]), keep] = x[np.arange(x.shape[0]), keep]
        x = y
    elif kind == "inf":
        x[0, 3] = x[0, V - 1] = np.inf
        x[5, :] = np.where(rng.random(V) < 0.01, np.inf, x[5, :])
    elif kind == "large":
        x *= 40.0  # far beyond the softcap
    elif kind == "huge":
        x[1, 7] = 3e38
        x[2, 9] = -9e29
    return x


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cap", [30.0, 0.0])
@pytest.mark.parametrize("kind", ["most", "lowest", "nan", "empty rows", "empty group", "all", "one token", "inf", "large",
                                  "huge"])
def test_select_masks(sampler, g4, torch_cuda, dtype, cap, kind):
    rng = np.random.default_rng(11)
    x = mask(logits(rng, 12, 3001), kind, rng, dtype)
    c = Case(torch_cuda, g4, x, dtype, 4, 8, cap=cap, pad=7)
    c.check(c.run(sampler))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("W,N", [(4, 8), (32, 64), (1, 64), (8, 3)])
@pytest.mark.parametrize("kind", ["equal", "few values", "zeros", "block"])
def test_select_ties(sampler, g4, torch_cuda, dtype, kind, W, N):
    rng = np.random.default_rng(3)
    V = 9001
    x = np.zeros((2 * W, V))
    if kind == "few values":
        x = np.tile(rng.integers(0, 3, V).astype(float), (2 * W, 1))
    elif kind == "zeros":
        x = np.where(rng.random((2 * W, V)) < 0.5, -0.0, 0.0)  # equal, whatever the sign
    elif kind == "block":
        x[:, 1000:1500] = 2.0  # the best tokens side by side, more than places
    # the same score: continuations of equal rank are told apart by beam and id
    c = Case(torch_cuda, g4, x, dtype, W, N, scores=np.full(2 * W, -1.5), lens=np.full(2 * W, 3), pad=1)
    got = c.run(sampler)
    c.check(got)
    want = beam_util.select(c.x, c.scores, c.lens, c.done, W, N, c.cap, c.T, c.alpha, 7)
    for g in range(2):
        assert [(int(a), int(b)) for a, b in zip(got[3][g], got[4][g])] == [(k[2], k[3]) for k in want[g][:N]]


def test_select_dead_and_ended_beams(sampler, g4, torch_cuda):
    rng = np.random.default_rng(2)
    W, N = 4, 6
    x = logits(rng, 5 * W, 4000)
    scores = -rng.exponential(2.0, 5 * W)
    scores[1:4] = -np.inf                      # a first step: one beam lives
    scores[4:8] = -np.inf                      # no beam
    scores[8] = np.nan
    done = np.zeros(5 * W)
    done[12:16] = 1                            # all have ended
    done[[17, 18]] = 1
    scores[17] = -np.inf                       # ended and dead
    scores[18] = -0.01                         # the ended one leads
    lens = np.full(5 * W, 9)
    lens[12] = 0
    for alpha in (0.0, 1.0):
        c = Case(torch_cuda, g4, x, "f32", W, N, scores=scores, done=done, lens=lens, alpha=alpha)
        got = c.run(sampler)
        c.check(got)
        assert (got[3][1] == -1).all()
        assert sorted(got[3][3][:4]) == [12, 13, 14, 15] and (got[4][3][:4] == 7).all()
        assert got[3][4][0] == 18 and got[2][4][0] == 1 and got[1][4][0] == 9


def test_select_end_tokens(sampler, g4, torch_cuda):
    x = np.full((2, 200), -5.0)
    x[0, 106], x[0, 3], x[1, 50], x[1, 1] = 9.0, 8.0, 9.0, 8.5
    c = Case(torch_cuda, g4, x, "f32", 2, 4, scores=[-1.0, -1.0])
    s, l, d, p, t = c.run(sampler)
    c.check((s, l, d, p, t))
    assert {int(k): int(v) for k, v in zip(t[0], d[0])} == {106: 1, 3: 0, 50: 1, 1: 1}


@pytest.mark.parametrize("dtype,V", [("f32", 262145), ("f32", 600001), ("bf16", 1 << 20), ("bf16", 524289)])
def test_select_long_rows(big, g4, torch_cuda, dtype, V):
    rng = np.random.default_rng(V)
    x = logits(rng, 6, V)
    x[2, V - 5:] = [14.0, 15.0, 16.0, 17.0, 18.0]
    c = Case(torch_cuda, g4, x, dtype, 3, 6, pad=(-V) % 8)
    c.check(c.run(big))
    x[:, 70000:] = 1.0
    c = Case(torch_cuda, g4, x, dtype, 3, 6, pad=3, cap=0.0)
    c.check(c.run(big))


def test_select_equal_rows_tie_whatever_their_alignment(sampler, g4, torch_cuda):
    # rows 8 bytes apart in alignment hold the same logits: the lower beam comes first
    rng = np.random.default_rng(9)
    x = np.tile(logits(rng, 1, 30002), (4, 1))
    for dtype in ("f32", "bf16"):
        c = Case(torch_cuda, g4, x, dtype, 4, 8, scores=np.full(4, -2.0), lens=np.full(4, 5))
        s, _, _, p, t = c.run(sampler)
        assert p[0].tolist() == [0, 1, 2, 3, 0, 1, 2, 3]
        assert len(set(t[0][:4])) == 1 and (s[0][:4] == s[0][0]).all()


def test_select_in_place_and_twice(sampler, g4, torch_cuda):
    rng = np.random.default_rng(4)
    c = Case(torch_cuda, g4, logits(rng, 12, 5000), "bf16", 4, 4, alpha=0.7)
    first = c.run(sampler)
    again = c.run(sampler)
    for a, b in zip(first, again):
        assert np.array_equal(a, b)  # bit for bit
    inplace = c.run(sampler, in_place=True)
    for a, b in zip(first, inplace):
        assert np.array_equal(a, b)


def test_select_other_stream_and_graph(sampler, g4, torch_cuda):
    torch = torch_cuda
    rng = np.random.default_rng(6)
    x = logits(rng, 12, 5000)
    c = Case(torch, g4, x, "f32", 4, 8, pad=4)
    want = c.run(sampler)
    s = torch.cuda.Stream()
    assert all(np.array_equal(a, b) for a, b in zip(want, c.run(sampler, stream=s.cuda_stream)))
    for v in c.out:
        v.fill_(-77 if v.dtype != torch.uint8 else 77)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        sampler.beam_select(c.ptr, g4.F32, c.G, c.V, c.stride, c.cap, c.params, c.state(c.d), c.state(c.out[:3]),
                            c.out[3].data_ptr(), c.out[4].data_ptr(), stream=s.cuda_stream)
    g.replay()
    torch.cuda.synchronize()
    assert all(np.array_equal(a, b) for a, b in zip(want, c.got()))
    # other logits in the same buffer
    y = logits(rng, 12, 5000)
    c.buf.view(12, c.stride)[:, :5000] = torch.from_numpy(y.astype(np.float32)).cuda()
    c.x = y.astype(np.float32).astype(np.float64)
    g.replay()
    torch.cuda.synchronize()
    c.check(c.got())


# ---------------------------------------------------------------------------
# reordering
# ---------------------------------------------------------------------------
def reorder_want(x, parents, W, live):
    """x [planes, rows, heads, max_len, dim]: positions below `live` by parent."""
    want = x.copy()
    for j, p in enumerate(parents):
        if p // W == j // W and p >= 0:
            want[:, j, :, :live] = x[:, p, :, :live]
    return want


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("G,W,planes,heads,max_len,live,dim", [
    (1, 1, 1, 1, 1, 1, 1), (2, 3, 2, 2, 5, 3, 7), (3, 4, 3, 2, 9, 9, 16), (2, 8, 2, 1, 17, 5, 6), (2, 16, 1, 3, 8, 7, 8),
    (1, 32, 2, 2, 6, 6, 10), (5, 5, 4, 2, 33, 32, 64), (2, 2, 1, 1, 4000, 3999, 3)])
@pytest.mark.parametrize("esize", [1, 2, 4])
def test_reorder(sampler, g4, torch_cuda, in_place, G, W, planes, heads, max_len, live, dim, esize):
    torch = torch_cuda
    rng = np.random.default_rng(W * 100 + live)
    dt = {1: np.uint8, 2: np.int16, 4: np.int32}[esize]
    R = G * W
    x = rng.integers(0, 127, (planes, R, heads, max_len, dim)).astype(dt)
    hist = rng.integers(0, 1000, (R, 11)).astype(np.int32)
    parents = (np.arange(R) // W * W + rng.integers(0, W, R)).astype(np.int32)
    if R > 3:
        parents[1], parents[R - 1] = -1, parents[R - 1]
    src = torch.from_numpy(x).cuda()
    dst = src if in_place else torch.from_numpy(np.full_like(x, 99)).cuda()
    h = torch.from_numpy(hist).cuda()
    block = heads * max_len * dim * esize
    tens = g4.beam_tensors([
        g4.BeamTensor(src.data_ptr(), dst.data_ptr(), block, planes, R * block, heads, max_len * dim * esize,
                      live * dim * esize),
        g4.BeamTensor(h.data_ptr(), h.data_ptr(), 44, 1, 0, 1, 0, 5 * 4)])
    dp = torch.from_numpy(parents).cuda()
    torch.cuda.synchronize()
    sampler.beam_reorder(dp.data_ptr(), G, W, tens)
    torch.cuda.synchronize()
    want = reorder_want(x, parents, W, live)
    if not in_place:
        keep = np.full_like(x, 99)
        for j, p in enumerate(parents):
            if p >= 0:
                keep[:, j, :, :live] = want[:, j, :, :live]
        want = keep
    assert np.array_equal(dst.cpu().numpy(), want)
    hw = hist.copy()
    for j, p in enumerate(parents):
        if p >= 0:
            hw[j, :5] = hist[p, :5]
    assert np.array_equal(h.cpu().numpy(), hw)


def test_reorder_the_most_tensors(sampler, g4, torch_cuda):
    torch = torch_cuda
    rng = np.random.default_rng(8)
    G, W = 3, 4
    parents = (np.arange(G * W) // W * W + rng.integers(0, W, G * W)).astype(np.int32)
    host, dev, tens = [], [], []
    for i in range(g4.BEAM_MAX_TENSORS):
        n = (1, 4, 16, 5, 4096, 1028, 333)[i % 7]  # bytes a row, every width
        host.append(rng.integers(0, 256, (G * W, n), dtype=np.uint8))
        dev.append(torch.from_numpy(host[-1].copy()).cuda())
        tens.append(g4.BeamTensor(dev[-1].data_ptr(), dev[-1].data_ptr(), n, 1, 0, 1, 0, n))
    d = torch.from_numpy(parents).cuda()
    torch.cuda.synchronize()
    sampler.beam_reorder(d.data_ptr(), G, W, g4.beam_tensors(tens))
    torch.cuda.synchronize()
    for h, v in zip(host, dev):
        assert np.array_equal(v.cpu().numpy(), h[parents])


def test_reorder_ignores_parents_of_other_groups(sampler, g4, torch_cuda):
    torch = torch_cuda
    x = torch.arange(8 * 4, dtype=torch.int32, device="cuda").view(8, 4)
    y = torch.full_like(x, -5)
    parents = torch.tensor([3, 4, 1, -2147483648, 7, 8, 2147483647, 4], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    sampler.beam_reorder(parents.data_ptr(), 2, 4, [g4.BeamTensor(x.data_ptr(), y.data_ptr(), 16, 1, 0, 1, 0, 16)])
    torch.cuda.synchronize()
    want = np.full((8, 4), -5)
    for j, p in ((0, 3), (2, 1), (4, 7), (7, 4)):
        want[j] = np.arange(4) + 4 * p
    assert np.array_equal(y.cpu().numpy(), want)


def test_reorder_nothing_to_do(sampler, g4, torch_cuda):
    torch = torch_cuda
    x = torch.ones(4, 4, dtype=torch.int32, device="cuda")
    parents = torch.zeros(4, dtype=torch.int32, device="cuda")
    assert sampler.beam_reorder(parents.data_ptr(), 1, 4, []) == g4.OK
    assert sampler.beam_reorder(parents.data_ptr(), 1, 4,
                                [g4.BeamTensor(x.data_ptr(), x.data_ptr(), 16, 1, 0, 1, 0, 0)]) == g4.OK


def test_refusals(sampler, g4, torch_cuda):
    c = Case(torch_cuda, g4, np.zeros((8, 64)), "f32", 4, 4)
    P, T = c.out[3].data_ptr(), c.out[4].data_ptr()

    def call(code, what, dtype=0, G=2, V=64, stride=64, cap=30.0, params=None, before=None, after=None, ptr=c.ptr, parents=P):
        rc = sampler.beam_select(ptr, dtype, G, V, stride, cap, params or c.params, before or c.state(c.d),
                                 after or c.state(c.out[:3]), parents, T, check=False)
        assert rc == code and what in sampler.last_error(), (rc, sampler.last_error())

    mk = g4.make_beam_params
    call(g4.ERR_ARG, "non-NULL", ptr=None)
    call(g4.ERR_ARG, "non-NULL", parents=None)
    call(g4.ERR_ARG, "dtype", dtype=2)
    call(g4.ERR_ARG, "beams", params=mk(0, 4))
    call(g4.ERR_ARG, "beams", params=mk(33, 4))
    call(g4.ERR_ARG, "n_out", params=mk(4, 65))
    call(g4.ERR_ARG, "n_out", params=mk(4, 0))
    call(g4.ERR_ARG, "groups", G=0)
    call(g4.ERR_ARG, "vocab", V=0)
    call(g4.ERR_CAPACITY, "exceed", G=257)
    call(g4.ERR_CAPACITY, "exceed", V=262145, stride=262145)
    call(g4.ERR_ARG, "row_stride", stride=63)
    call(g4.ERR_ARG, "aligned", ptr=c.ptr + 2)
    for T_ in (0.0, -1.0, float("nan"), float("inf"), 1e-7):
        call(g4.ERR_ARG, "temperature", params=mk(4, 4, T_))
    for a in (-0.5, float("nan"), 9.0):
        call(g4.ERR_ARG, "length_alpha", params=mk(4, 4, 1.0, a))
    for cap in (float("nan"), float("inf"), 1e-7):
        call(g4.ERR_ARG, "softcap", cap=cap)
    bad = mk(4, 4)
    bad.n_eos = 9
    call(g4.ERR_ARG, "n_eos", params=bad)
    no_lens = g4.BeamState(c.d[0].data_ptr(), None, None)
    call(g4.ERR_ARG, "lens", before=no_lens)
    call(g4.ERR_ARG, "lens", before=no_lens, after=g4.BeamState(c.out[0].data_ptr(), None, None), params=mk(4, 4, 1.0, 0.5))
    call(g4.ERR_ARG, "overlaps", after=c.state(c.d), params=mk(4, 3))
    call(g4.ERR_ARG, "overlaps", after=g4.BeamState(c.d[0].data_ptr() + 4, None, None))
    with pytest.raises(ValueError):
        mk(4, 4, eos=range(9))
    # lens and done may be left out
    assert sampler.beam_select(c.ptr, 0, 2, 64, 64, 30.0, c.params, no_lens, g4.BeamState(c.out[0].data_ptr(), None, None),
                               P, T, check=False) == g4.OK

    x = c.d[0].data_ptr()
    ok = dict(src=x, dst=x, row_stride=4, segs0=1, stride0=0, segs1=1, stride1=0, seg_bytes=4)
    for change, what in (({"src": None}, "NULL"), ({"row_stride": 3}, "row_stride"), ({"seg_bytes": -1}, "negative"),
                         ({"segs0": 0}, "no segment"), ({"segs1": 2}, "overlap"), ({"stride0": -4, "segs0": 2}, "negative")):
        t = {**ok, **change}
        rc = sampler.beam_reorder(P, 2, 4, [g4.BeamTensor(*(t[f] for f, _ in g4.BeamTensor._fields_))], check=False)
        assert rc == g4.ERR_ARG and what in sampler.last_error(), (change, sampler.last_error())
    assert sampler.beam_reorder(None, 2, 4, [], check=False) == g4.ERR_ARG
    assert sampler.beam_reorder(P, 2, 33, [], check=False) == g4.ERR_ARG
    t = g4.BeamTensor(x, x, 1 << 41, 1, 0, 1, 0, 1 << 40)
    assert sampler.beam_reorder(P, 2, 4, [t], check=False) == g4.ERR_CAPACITY
    with pytest.raises(g4.G4SError):
        sampler.beam_reorder(P, 0, 4, [])
    torch_cuda.cuda.synchronize()
    assert ctypes.sizeof(g4.BeamParams) == 64


def test_select_many_beams_with_length_penalty(sampler, g4, torch_cuda):
    # one warp a beam from 16 beams on
    rng = np.random.default_rng(12)
    for W, N in ((15, 30), (16, 7), (17, 64), (31, 33)):
        c = Case(torch_cuda, g4, logits(rng, 2 * W, 3000), "f32", W, N, alpha=0.9, done=rng.random(2 * W) < 0.2, T=0.8)
        c.check(c.run(sampler))


def test_select_rows_over_4_gib_apart(sampler, g4, torch_cuda):
    torch = torch_cuda
    rng = np.random.default_rng(13)
    stride, V, W = 600_000_000, 5001, 4  # 2.4 GB a row: the last starts over 2^31 elements in
    buf = torch.empty(5 * stride + V, device="cuda")
    c = Case(torch, g4, logits(rng, 5, V), "f32", 5, 10)
    for r in range(5):
        buf[r * stride:r * stride + V] = c.buf.view(5, V)[r]
    c.buf, c.ptr, c.stride = buf, buf.data_ptr(), stride
    c.check(c.run(sampler))
    del buf, c
    torch.cuda.empty_cache()


def test_select_two_contexts_at_once(g4, torch_cuda):
    torch = torch_cuda
    rng = np.random.default_rng(14)
    with g4.Sampler(0, 64, 40000) as a, g4.Sampler(0, 64, 40000) as b:
        ca = Case(torch, g4, logits(rng, 60, 33000), "f32", 6, 12)
        cb = Case(torch, g4, logits(rng, 60, 33000), "bf16", 5, 5)
        sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
        torch.cuda.synchronize()
        for _ in range(20):
            for s, c, st, dt in ((a, ca, sa, g4.F32), (b, cb, sb, g4.BF16)):
                s.beam_select(c.ptr, dt, c.G, c.V, c.stride, c.cap, c.params, c.state(c.d), c.state(c.out[:3]),
                              c.out[3].data_ptr(), c.out[4].data_ptr(), stream=st.cuda_stream)
        torch.cuda.synchronize()
        ca.check(ca.got())
        cb.check(cb.got())


def test_select_between_sampler_calls(sampler, g4, torch_cuda, oracle):
    # the selection shares the context's item statistics with the full-vocabulary path, and starts behind it
    torch = torch_cuda
    rng = np.random.default_rng(15)
    x = logits(rng, 8, 20000).astype(np.float32)
    c = Case(torch, g4, x, "f32", 4, 4)
    dx = torch.from_numpy(x).cuda()
    u = torch.full((8,), 0.3, dtype=torch.float64, device="cuda")
    tok = torch.zeros(8, dtype=torch.int32, device="cuda")
    p = g4.make_params(1.0, 0, 0.95)
    torch.cuda.synchronize()
    sampler.sample(dx.data_ptr(), g4.F32, 8, 20000, 20000, p, 30.0, u.data_ptr(), tok.data_ptr())
    torch.cuda.synchronize()
    want = tok.cpu().numpy().copy()
    first = c.run(sampler)
    for _ in range(5):
        tok.fill_(-1)
        torch.cuda.synchronize()
        sampler.sample(dx.data_ptr(), g4.F32, 8, 20000, 20000, p, 30.0, u.data_ptr(), tok.data_ptr())
        sampler.beam_select(c.ptr, g4.F32, c.G, c.V, c.stride, c.cap, c.params, c.state(c.d), c.state(c.out[:3]),
                            c.out[3].data_ptr(), c.out[4].data_ptr())
        torch.cuda.synchronize()
        assert np.array_equal(tok.cpu().numpy(), want)
        assert all(np.array_equal(p, q) for p, q in zip(first, c.got()))
    c.check(first)


def test_select_on_the_lm_heads_logits(g4, torch_cuda, oracle):
    """The LM head's logits (kept with out_logits) searched without leaving the device."""
    torch = torch_cuda
    rng = np.random.default_rng(16)
    V, H, rows = 4096, 256, 8
    blocks = rng.integers(0, 256, (V, H // 32, 18), dtype=np.uint8)
    blocks[:, :, :2] = (rng.uniform(0.001, 0.02, (V, H // 32)).astype(np.float16)).view(np.uint8).reshape(V, H // 32, 2)
    db = torch.from_numpy(blocks.reshape(-1).copy()).cuda()
    nib = torch.zeros(V * H // 2, dtype=torch.uint8, device="cuda")
    sc = torch.zeros(V * H // 32, dtype=torch.int16, device="cuda")
    hidden = torch.from_numpy(rng.standard_normal((rows, H)).astype(np.float32)).cuda()
    out = torch.zeros(rows, V, device="cuda")
    tok = torch.zeros(rows, dtype=torch.int32, device="cuda")
    with g4.Sampler(0, rows, V) as s:
        torch.cuda.synchronize()
        g4.q4_repack(db.data_ptr(), V, H, nib.data_ptr(), sc.data_ptr())
        torch.cuda.synchronize()
        c = Case(torch, g4, np.zeros((rows, V)), "f32", 4, 8)
        s.lmhead_sample(hidden.data_ptr(), rows, H, nib.data_ptr(), sc.data_ptr(), V, g4.make_params(0.0, 4, 1.0), 30.0, 0,
                        tok.data_ptr(), logits_ptr=out.data_ptr())
        c.ptr, c.stride = out.data_ptr(), V
        got = c.run(s)
        c.x = out.double().cpu().numpy()
        c.check(got)


def test_reorder_rows_over_4_gib_apart(sampler, g4, torch_cuda):
    torch = torch_cuda
    buf = torch.empty(3 * 2_200_000_000 + 64, dtype=torch.uint8, device="cuda")
    row = 2_200_000_000
    for r in range(3):
        buf[r * row:r * row + 64] = r + 1
    parents = torch.tensor([2, 0, 0], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    sampler.beam_reorder(parents.data_ptr(), 1, 3, [g4.BeamTensor(buf.data_ptr(), buf.data_ptr(), row, 2, 32, 1, 0, 32)])
    torch.cuda.synchronize()
    assert [int(buf[r * row + 63]) for r in range(3)] == [3, 1, 1]
    del buf
    torch.cuda.empty_cache()


def test_select_extreme_scores(sampler, g4, torch_cuda):
    rng = np.random.default_rng(17)
    x = logits(rng, 12, 3000)
    scores = np.array([0.0, -1e9, -1e9, -1e9, 5.0, np.inf, -3.0, -2.0, -3e38, -1e30, 1e20, -7.0])
    c = Case(torch_cuda, g4, x, "f32", 4, 6, scores=scores)
    s, l, d, p, t = c.run(sampler)
    want = beam_util.select(c.x, c.scores, c.lens, c.done, 4, 6, 30.0, 1.0, 0.0, 7)
    # beams held back by a large negative score come in their own order behind the first
    assert p[0].tolist() == [k[2] for k in want[0][:6]] and t[0].tolist() == [k[3] for k in want[0][:6]]
    # +inf takes every place, best logits first
    assert (p[1] == 5).all() and (s[1] == np.inf).all()
    assert t[1].tolist() == np.lexsort((np.arange(3000), -c.x[5]))[:6].tolist()
    assert p[2][0] == 10 and np.isfinite(s[2]).all()
