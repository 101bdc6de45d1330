"""The paged cache's fork and compaction on the GPU against their sequential definitions, and a
whole beam search over a paged cache against one that keeps token lists."""
import numpy as np
import pytest

import beam_util

pytestmark = pytest.mark.gpu


class Cache:
    """Random pools of several layouts: (segments, bytes a position, spare bytes a segment, spare bytes a page)."""

    def __init__(self, torch, g4, rng, n_pages, P, width, layouts=((1, 32, 0, 0), (2, 20, 4, 8), (3, 7, 3, 1))):
        self.torch, self.P, self.n_pages, self.width, self.layouts = torch, P, n_pages, width, layouts
        self.host, self.dev, pools = [], [], []
        for segs, token, spare, page_spare in layouts:
            seg = P * token + spare
            page = segs * seg + page_spare
            h = rng.integers(0, 256, n_pages * page, dtype=np.uint8)
            d = torch.from_numpy(h.copy()).cuda()
            self.host.append(h)
            self.dev.append(d)
            pools.append(g4.PagePool(d.data_ptr(), page, segs, seg, token))
        self.c = g4.page_cache(pools, P, n_pages, width)

    def moved(self, copies):
        """The pools after the copies (from, to, filled positions)."""
        out = []
        for h, (segs, token, spare, page_spare) in zip(self.host, self.layouts):
            seg = self.P * token + spare
            v = h.copy().reshape(self.n_pages, segs * seg + page_spare)
            for a, b, fill in copies:
                for s in range(segs):
                    v[b, s * seg:s * seg + fill * token] = h.reshape(self.n_pages, -1)[a, s * seg:s * seg + fill * token]
            out.append(v.reshape(-1))
        return out

    def check(self, copies):
        for w, d in zip(self.moved(copies), self.dev):
            assert np.array_equal(d.cpu().numpy(), w)


def scattered(rng, n, lens, P, width, n_pages, share=0.5):
    """Tables of sequences that share prefixes (and last pages) with the one before."""
    ids = rng.permutation(n_pages)
    tables = np.full((n, width), -1, np.int64)
    refs = np.zeros(n_pages, np.int64)
    at = 0
    for i, ln in enumerate(lens):
        k = -(-int(ln) // P)
        common = 0
        if i and rng.random() < share:
            prev = -(-int(lens[i - 1]) // P)
            common = int(rng.integers(0, min(k, prev) + 1))
            tables[i, :common] = tables[i - 1, :common]
        tables[i, common:k] = ids[at:at + k - common]
        at += k - common
        refs[tables[i, :k]] += 1
    assert at <= n_pages
    return tables, refs, ids[at:]


def run_fork(torch, g4, sampler, cache, tables, lens, refs, src, n_new, frozen=None, alias=False, stream=None):
    cu = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()
    n_in, n_out, width = len(lens), len(src), cache.width
    dt, dl, dr, ds = cu(tables), cu(lens), cu(refs), cu(src)
    ot = torch.full((n_out + 1, width), -9, dtype=torch.int32, device="cuda")
    ol = dl if alias and n_out <= n_in else torch.full((n_out + 1,), -9, dtype=torch.int32, device="cuda")
    orf = dr if alias else torch.full((len(refs) + 1,), -9, dtype=torch.int32, device="cuda")
    res = torch.full((5,), -9, dtype=torch.int32, device="cuda")
    fz = torch.from_numpy(np.asarray(frozen, np.uint8)).cuda() if frozen is not None else None
    torch.cuda.synchronize()
    sampler.pages_fork(cache.c, n_in, dt.data_ptr(), dl.data_ptr(), dr.data_ptr(), n_out, ds.data_ptr(), n_new,
                       ot.data_ptr(), ol.data_ptr(), orf.data_ptr(), res.data_ptr(),
                       frozen_ptr=fz.data_ptr() if fz is not None else 0, stream=stream)
    torch.cuda.synchronize()
    want_t, want_l, want_r, want, copies = beam_util.fork(np.asarray(tables), np.asarray(lens), np.asarray(refs), src, n_new,
                                                         cache.P, width, frozen)
    assert res.tolist() == want + [-9]
    got = ot.cpu().numpy()
    assert np.array_equal(got[:n_out], want_t)
    assert (got[n_out] == -9).all()
    assert np.array_equal(ol.cpu().numpy()[:n_out], want_l)
    assert np.array_equal(orf.cpu().numpy()[:len(refs)], want_r)
    cache.check(copies)
    return want, copies


@pytest.mark.parametrize("n_new", [0, 1, 5, 40])
@pytest.mark.parametrize("n_in,n_out,P,width,n_pages", [
    (1, 1, 1, 64, 100), (3, 5, 4, 32, 200), (8, 8, 16, 12, 120), (40, 70, 8, 30, 3000), (300, 1000, 16, 9, 9000),
    (5, 0, 16, 12, 120), (4, 4, 7, 60, 20011)])
def test_fork(sampler, g4, torch_cuda, n_in, n_out, P, width, n_pages, n_new):
    rng = np.random.default_rng(n_in * 1000 + n_new)
    cache = Cache(torch_cuda, g4, rng, n_pages, P, width)
    most = max(1, min(width * P - n_new, (n_pages // (2 * max(n_in, 1))) * P, 17 * P))
    lens = rng.integers(0, most + 1, n_in)
    tables, refs, rest = scattered(rng, n_in, lens, P, width, n_pages)
    refs[rest[:5]] += 1          # held elsewhere
    if n_in and lens[0]:
        refs[tables[0, -(-int(lens[0]) // P) - 1]] += 1  # a last page held elsewhere too
    src = rng.integers(-1, n_in, n_out)
    for alias in (False, True):
        cache = Cache(torch_cuda, g4, rng, n_pages, P, width)
        run_fork(torch_cuda, g4, sampler, cache, tables, lens, refs, src, n_new, alias=alias)
    cache = Cache(torch_cuda, g4, rng, n_pages, P, width)
    run_fork(torch_cuda, g4, sampler, cache, tables, lens, refs, src, n_new, frozen=rng.random(n_out) < 0.4)


def test_fork_many_copies_of_one(sampler, g4, torch_cuda):
    rng = np.random.default_rng(1)
    for held in (0, 1):
        cache = Cache(torch_cuda, g4, rng, 500, 16, 8)
        tables = np.full((2, 8), -1)
        tables[0, :3] = [7, 400, 33]
        tables[1, :1] = [44]
        refs = np.zeros(500, np.int64)
        refs[[7, 400, 33, 44]] = 1
        refs[33] += held
        got, copies = run_fork(torch_cuda, g4, sampler, cache, tables, [37, 16], refs, [0] * 64 + [-1, 1], 1)
        assert got[0] == 64 + held and len(copies) == 63 + held


def test_fork_short_of_pages_or_table(sampler, g4, torch_cuda):
    rng = np.random.default_rng(2)
    tables = np.full((2, 4), -1)
    tables[0, :3], tables[1, :4] = [0, 1, 2], [3, 4, 5, 6]
    refs = np.array([1] * 7 + [0, 1])
    for src, n_new, lens in (([0, 0, 0, 1], 1, [10, 15]),   # one free page, two copies
                             ([0, 1], 1, [12, 16]),          # the second's table is full
                             ([0, 1], 20, [12, 16]), ([0, 0, 0, 1], 4, [12, 12])):
        cache = Cache(torch_cuda, g4, rng, 9, 4, 4)
        got, copies = run_fork(torch_cuda, g4, sampler, cache, tables, lens, refs, src, n_new)
        assert (got[1] or got[2]) and got[0] == 0 and not copies
    # every page of the freed sequence can be taken at once
    cache = Cache(torch_cuda, g4, rng, 9, 4, 8)
    t8 = np.full((2, 8), -1)
    t8[:, :4] = tables
    got, _ = run_fork(torch_cuda, g4, sampler, cache, t8, [12, 16], refs, [0], 20)
    assert got == [5, 0, 0, 0]


def test_fork_bad_inputs(sampler, g4, torch_cuda):
    rng = np.random.default_rng(3)
    tables = np.array([[0, 1, 2, -1], [3, 99, 5, -1], [-7, 6, 7, -1], [8, 9, -1, -1]])
    refs = np.array([1] * 10 + [0] * 10)
    for src, lens in (([0, 1, 2, 3], [10, 10, 10, 6]), ([0, 4, 2147483647, 3], [10, 10, 10, 6]),
                      ([0, 1, -5, -2147483648], [10, -3, 10, 17]), ([3, 3, 2, 0], [-1, 17, 2147483647, 6])):
        for n_new in (0, 2):
            cache = Cache(torch_cuda, g4, rng, 20, 4, 4)
            got, copies = run_fork(torch_cuda, g4, sampler, cache, tables, lens, refs, src, n_new)
            assert got[3] > 0 and got[0] == 0
    # bad entries behind a sequence's end do not count
    cache = Cache(torch_cuda, g4, rng, 20, 4, 4)
    got, _ = run_fork(torch_cuda, g4, sampler, cache, tables, [10, 4, 0, 6], refs, [0, 1, 2, 3], 1)
    assert got[3] == 0 and got[0] == 2
    # counts below zero are free pages
    refs[12:14] = -3
    cache = Cache(torch_cuda, g4, rng, 20, 4, 4)
    run_fork(torch_cuda, g4, sampler, cache, tables, [10, 4, 0, 6], refs, [0, 0, 0, 3], 6)


def test_fork_large_tables(sampler, g4, torch_cuda):
    rng = np.random.default_rng(4)
    n, P, width, n_pages = 256, 16, 600, 60000
    lens = rng.integers(0, 580 * P, n)
    lens = (lens * (0.7 * n_pages * P / lens.sum())).astype(np.int64)
    cache = Cache(torch_cuda, g4, rng, n_pages, P, width, layouts=((1, 16, 0, 0),))
    tables, refs, _ = scattered(rng, n, lens, P, width, n_pages)
    src = np.arange(n) // 8 * 8 + rng.integers(0, 8, n)
    run_fork(torch_cuda, g4, sampler, cache, tables, lens, refs, src, 3)


def test_fork_more_sequences_than_threads(g4, torch_cuda):
    s = g4.Sampler(device=0, max_rows=8192, max_vocab=64)
    rng = np.random.default_rng(6)
    n, P, width, n_pages = 3000, 3, 5, 30000
    lens = rng.integers(0, width * P - 1, n)
    cache = Cache(torch_cuda, g4, rng, n_pages, P, width, layouts=((1, 4, 0, 0),))
    tables, refs, _ = scattered(rng, n, lens, P, width, n_pages)
    for n_out in (1025, 8192):
        src = rng.integers(-1, n, n_out)
        src[-40:] = src[0]  # a parent whose children are far apart
        c = Cache(torch_cuda, g4, rng, n_pages, P, width, layouts=((1, 4, 0, 0),))
        run_fork(torch_cuda, g4, s, c, tables, lens, refs, src, 1, frozen=rng.random(n_out) < 0.2)
    s.close()


def run_compact(torch, g4, sampler, cache, tables, lens, refs, alias):
    cu = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()
    n, n_pages = len(lens), cache.n_pages
    dt, dl, dr = cu(tables), cu(lens), cu(refs)
    ot = dt if alias else dt.clone().fill_(-9)
    orf = dr if alias else torch.full((n_pages,), -9, dtype=torch.int32, device="cuda")
    mp = torch.full((n_pages + 1,), -9, dtype=torch.int32, device="cuda")
    mv = torch.full((n_pages + 1,), -9, dtype=torch.int32, device="cuda")
    res = torch.full((5,), -9, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    sampler.pages_compact(cache.c, n, dt.data_ptr(), dl.data_ptr(), dr.data_ptr(), ot.data_ptr(), orf.data_ptr(),
                          mp.data_ptr(), mv.data_ptr(), res.data_ptr())
    torch.cuda.synchronize()
    wt, wr, wm, wv, want = beam_util.compact(np.asarray(tables), np.asarray(lens), np.asarray(refs), cache.P, cache.width)
    assert res.tolist() == want + [-9]
    got = ot.cpu().numpy()
    for i, ln in enumerate(lens):
        k = -(-min(max(int(ln), 0), cache.width * cache.P) // cache.P)
        assert np.array_equal(got[i, :k], wt[i, :k])
        assert np.array_equal(got[i, k:], np.asarray(tables)[i, k:] if alias else np.full(cache.width - k, -9))
    assert np.array_equal(orf.cpu().numpy(), wr)
    assert mp.tolist() == wm.tolist() + [-9]
    assert mv.tolist() == wv.tolist() + [-9] * (n_pages + 1 - len(wv))
    cache.check([(a, b, cache.P) for a, b in wv.reshape(-1, 2)])
    return want


@pytest.mark.parametrize("alias", [False, True])
@pytest.mark.parametrize("n,P,width,n_pages,fill", [(1, 4, 5, 1, 1.0), (1, 4, 5, 7, 0.5), (3, 16, 8, 31, 0.9), (5, 8, 40, 255, 0.4),
                                                    (6, 8, 40, 257, 0.97), (20, 4, 70, 4001, 0.2), (64, 16, 40, 20000, 0.1)])
def test_compact(sampler, g4, torch_cuda, n, P, width, n_pages, fill, alias):
    rng = np.random.default_rng(n_pages)
    most = max(1, min(width, int(n_pages * fill / n)))
    lens = rng.integers(0, most * P + 1, n)
    tables, refs, rest = scattered(rng, n, lens, P, width, n_pages)
    refs[rest[::3]] = 2
    refs[rest[1::7]] = -1
    cache = Cache(torch_cuda, g4, rng, n_pages, P, width)
    run_compact(torch_cuda, g4, sampler, cache, tables, lens, refs, alias)


def test_compact_full_empty_and_compact_pools(sampler, g4, torch_cuda):
    rng = np.random.default_rng(8)
    for refs in (np.zeros(300), np.ones(300), np.r_[np.ones(100), np.zeros(200)], np.r_[np.zeros(200), np.ones(100)],
                 np.r_[np.zeros(299), 1], np.r_[0, np.ones(299)]):
        cache = Cache(torch_cuda, g4, rng, 300, 4, 3)
        run_compact(torch_cuda, g4, sampler, cache, np.full((0, 3), -1), [], refs.astype(np.int64), False)


def test_compact_bad_inputs(sampler, g4, torch_cuda):
    rng = np.random.default_rng(9)
    refs = np.zeros(40, np.int64)
    refs[[30, 31, 5]] = 1
    tables = np.array([[30, 31, -1], [5, 99, -4], [12, -1, -1]])
    for alias in (False, True):
        cache = Cache(torch_cuda, g4, rng, 40, 4, 3)
        got = run_compact(torch_cuda, g4, sampler, cache, tables, [8, 2147483647, 1], refs, alias)
        assert got == [3, 3, 0, 4]
        cache = Cache(torch_cuda, g4, rng, 40, 4, 3)
        assert run_compact(torch_cuda, g4, sampler, cache, tables, [8, 4, -2147483648], refs, alias)[3] == 1


def test_pages_refusals(sampler, g4, torch_cuda):
    torch = torch_cuda
    x = torch.zeros(4096, dtype=torch.int32, device="cuda")
    p = x.data_ptr()

    def fork(code, what, pool=None, P=4, n_pages=8, width=2, n_in=2, n_out=2, n_new=1, tables=p, lens=p + 256, refs=p + 512,
             src=p + 768, ot=p + 1024, ol=p + 1280, orf=p + 1536, res=p + 1792, pools=None):
        pools = pools if pools is not None else [g4.PagePool(p + 4096, 64, 1, 0, 16)] if pool is None else [g4.PagePool(*pool)]
        rc = sampler.pages_fork(g4.page_cache(pools, P, n_pages, width), n_in, tables, lens, refs, n_out, src, n_new, ot,
                                ol, orf, res, check=False)
        assert rc == code and what in sampler.last_error(), (rc, sampler.last_error())

    fork(g4.ERR_ARG, "page_tokens", P=0)
    fork(g4.ERR_ARG, "n_pages", n_pages=0)
    fork(g4.ERR_ARG, "max_seq_pages", width=0)
    fork(g4.ERR_ARG, "2^30", width=1 << 20, P=1 << 12)
    fork(g4.ERR_ARG, "n_pools", pools=[g4.PagePool(p, 64, 1, 0, 16)] * 97)
    fork(g4.ERR_ARG, "NULL data", pool=(None, 64, 1, 0, 16))
    fork(g4.ERR_ARG, "size", pool=(p, 64, 0, 0, 16))
    fork(g4.ERR_ARG, "size", pool=(p, 64, 1, 0, 0))
    fork(g4.ERR_ARG, "overlap", pool=(p, 63, 1, 0, 16))
    fork(g4.ERR_ARG, "overlap", pool=(p, 128, 2, 60, 16))
    fork(g4.ERR_CAPACITY, "vectors", pool=(p, 1 << 42, 1, 0, 1 << 36))
    fork(g4.ERR_ARG, "n_in", n_in=-1)
    fork(g4.ERR_CAPACITY, "n_out", n_out=1025)
    fork(g4.ERR_ARG, "n_new", n_new=-1)
    for name in ("tables", "lens", "refs", "src", "ot", "ol", "orf", "res"):
        fork(g4.ERR_ARG, "non-NULL", **{name: None})
    fork(g4.ERR_ARG, "out->tables", ot=p)
    fork(g4.ERR_ARG, "out->tables", ot=p + 12)
    fork(g4.ERR_ARG, "refs or lens", orf=p + 516)
    fork(g4.ERR_ARG, "refs or lens", ol=p + 260)
    rc = sampler.pages_compact(g4.page_cache([], 4, 8, 2), 2, p, p + 256, p + 512, p + 8, p + 1024, p + 2048, p + 3000,
                               p + 3500, check=False)
    assert rc == g4.ERR_ARG and "overlap" in sampler.last_error()
    rc = sampler.pages_compact(g4.page_cache([], 4, 8, 2), 2, p, p + 256, p + 512, p + 800, p + 1024, None, p + 3000,
                               p + 3500, check=False)
    assert rc == g4.ERR_ARG and "page_map" in sampler.last_error()


# ---------------------------------------------------------------------------
# a whole search
# ---------------------------------------------------------------------------
class Search:
    """A toy model whose logits depend on the last two tokens, searched on the GPU: token ids are what its paged
    cache and its dense state hold, so that both can be read back and compared with the beams' histories."""

    def __init__(self, torch, g4, sampler, G, W, V, P, seed, alpha):
        self.torch, self.g4, self.s, self.G, self.W, self.V, self.P = torch, g4, sampler, G, W, V, P
        rng = np.random.default_rng(seed)
        self.A = rng.standard_normal((V, V)).astype(np.float32) * 3
        self.B = rng.standard_normal((V, V)).astype(np.float32)
        R, self.width, self.n_pages = G * W, 24, 40 * G * W
        i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32, device="cuda")
        self.dA, self.dB = torch.from_numpy(self.A).cuda(), torch.from_numpy(self.B).cuda()
        self.logits = torch.zeros(R, V, device="cuda")
        self.pool = torch.full((self.n_pages, P), -1, dtype=torch.int32, device="cuda")
        self.cache = g4.page_cache([g4.PagePool(self.pool.data_ptr(), P * 4, 1, 0, 4)], P, self.n_pages, self.width)
        self.tab = [i32(R, self.width), i32(R, self.width)]
        self.plens, self.refs, self.result = i32(R), i32(self.n_pages), i32(4)
        self.prompt = rng.integers(2, V, (G, 5))
        self.scores = torch.full((R,), -np.inf, device="cuda")
        self.scores[::W] = 0.0
        self.lens, self.done = i32(R), torch.zeros(R, dtype=torch.uint8, device="cuda")
        self.par, self.tok = i32(R), i32(R)
        self.prev = torch.from_numpy(np.repeat(self.prompt[:, -2], W).astype(np.int32)).cuda()
        self.last = torch.from_numpy(np.repeat(self.prompt[:, -1], W).astype(np.int32)).cuda()
        # the prompt in the first beam's pages; the others start empty
        pages = -(-5 // P)
        for g in range(G):
            ids = torch.arange(g * pages, (g + 1) * pages, dtype=torch.int32, device="cuda")
            self.tab[0][g * W, :pages] = ids
            self.refs[ids.long()] = 1
            self.plens[g * W] = 5
            flat = np.full(pages * P, -1)
            flat[:5] = self.prompt[g]
            self.pool[ids.long()] = torch.from_numpy(flat.reshape(pages, P).astype(np.int32)).cuda()
        self.params = g4.make_beam_params(W, W, 0.9, alpha, pad_token=0, eos=(1,))
        # dense state: the row's previous token, moved in place
        self.dense = g4.beam_tensors([g4.BeamTensor(self.last.data_ptr(), self.last.data_ptr(), 4, 1, 0, 1, 0, 4)])
        self.state = g4.BeamState(self.scores.data_ptr(), self.lens.data_ptr(), self.done.data_ptr())

    def model(self):
        self.logits.copy_(self.dA[self.last.long()] + self.dB[self.prev.long()])

    def step(self, i, stream):
        g4 = self.g4
        a, b = self.tab[i % 2], self.tab[1 - i % 2]
        pages = g4.beam_pages(self.cache, g4.PageTables(a.data_ptr(), self.plens.data_ptr(), self.refs.data_ptr()),
                              g4.PageTables(b.data_ptr(), self.plens.data_ptr(), self.refs.data_ptr()), 1,
                              self.result.data_ptr())
        self.s.beam_step(self.logits.data_ptr(), g4.F32, self.G, self.V, self.V, 30.0, self.params, self.state, self.state,
                         self.par.data_ptr(), self.tok.data_ptr(), self.dense, pages, stream=stream)

    def write(self, i):
        """What the model does next: the token's entry at the new position, its state."""
        torch = self.torch
        tab = self.tab[1 - i % 2]
        live = self.par >= 0
        grown = live & (self.done == 0)
        pos = (self.plens.long() - 1).clamp(min=0)
        page = tab.gather(1, (pos // self.P)[:, None])[:, 0].long()
        at = page * self.P + pos % self.P
        flat = self.pool.view(-1)
        sel = grown.nonzero()[:, 0]
        flat[at[sel]] = self.tok[sel]
        self.prev.copy_(self.last)
        self.last.copy_(torch.where(live, self.tok, self.last))

    def before(self):
        """The beams' scores, lengths and end flags, as the next step takes them."""
        return [t.cpu().numpy().copy() for t in (self.scores, self.lens, self.done)]

    def follow(self, hists, before, alpha):
        """Checks the step taken from `before` against 64 bits, and returns the beams' new token lists.

        The oracle starts every step from the device's own scores, not from its own of the steps before: two paths
        that use the same transitions in another order (this model has such cycles) have one score in exact arithmetic
        and, with 12 roundings to fp32 in another order, two on the device, up to 12 eps / 2 * |score| < 1e-5 apart.
        Either may then come first, and 12 steps of 64 bits cannot say which.  Within a step a score is off by 2e-5 at
        most, so a place's rank is its 64-bit one or differs from it by at most 4e-5 / length^alpha <= 4e-5."""
        scores, lens, done = before
        W, new = self.W, []
        got = [t.cpu().numpy() for t in (self.scores, self.lens, self.done, self.par, self.tok)]
        for g in range(self.G):
            live = [r for r in range(g * W, (g + 1) * W) if scores[r] > -np.inf]
            x = np.stack([self.A[hists[r][-1]] + self.B[hists[r][-2]] for r in live]).astype(np.float64)
            cand = beam_util.select(x, scores[live], lens[live], done[live], len(live), W, 30.0, 0.9, alpha, 0, (1,))[0]
            by = {(live[c[2]], c[3]): c for c in cand}
            assert len(cand) >= W
            for w in range(W):
                sc, ln, dn, par, tok = (v[g * W + w] for v in got)
                rank, score, _, _, length, ended = by.pop((int(par), int(tok)))  # (each at most once)
                assert abs(float(sc) - score) <= 2e-5, (g, w)
                assert (int(ln), int(dn)) == (length, ended), (g, w)
                assert abs(rank - cand[w][0]) <= 4e-5, (g, w)
                new.append(hists[par] + ([] if done[par] else [int(tok)]))
        return new


@pytest.mark.parametrize("G,W,P,alpha,graph", [(1, 4, 4, 0.0, False), (3, 5, 3, 0.8, False), (2, 8, 16, 0.6, True), (2, 1, 2, 0.0, True)])
def test_search(sampler, g4, torch_cuda, G, W, P, alpha, graph):
    torch = torch_cuda
    s = Search(torch, g4, sampler, G, W, 97, P, 31 * G + W, alpha)
    steps = 12
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        graphs = {}
        hists = [list(map(int, s.prompt[r // W])) for r in range(G * W)]
        for i in range(steps):
            was = s.before()
            if graph:
                # two graphs, one a table buffer, captured once and replayed in turn
                s.model()
                if i % 2 not in graphs:
                    g = torch.cuda.CUDAGraph()
                    stream.synchronize()
                    with torch.cuda.graph(g, stream=stream):
                        s.step(i, stream.cuda_stream)
                    graphs[i % 2] = g
                graphs[i % 2].replay()
            else:
                s.model()
                s.step(i, stream.cuda_stream)
            s.write(i)
            assert s.result.tolist()[1:] == [0, 0, 0]
            hists = s.follow(hists, was, alpha)
    torch.cuda.synchronize()
    tab, lens = s.tab[steps % 2].cpu().numpy(), s.plens.cpu().numpy()
    pool = s.pool.cpu().numpy()
    held = np.zeros(s.n_pages, np.int64)
    for g in range(G):
        for w in range(W):
            r = g * W + w
            hist, done = hists[r], bool(s.done[r])
            n = int(lens[r])
            got = [int(pool[tab[r, t // P], t % P]) for t in range(n)]
            # an ended beam's end token has no position of its own
            assert got == (hist[:-1] if done else hist), (g, w)
        for w in range(W):
            held[tab[g * W + w, :-(-int(lens[g * W + w]) // P)]] += 1
    assert np.array_equal(held, s.refs.cpu().numpy())  # nothing leaked


def test_step_refusals(sampler, g4, torch_cuda):
    torch = torch_cuda
    s = Search(torch, g4, sampler, 1, 4, 97, 4, 1, 0.0)
    before = [t.clone() for t in (s.scores, s.lens, s.refs, s.par)]
    args = (s.logits.data_ptr(), g4.F32, 1, 97, 97, 30.0)
    ptrs = (s.par.data_ptr(), s.tok.data_ptr())
    rc = sampler.beam_step(*args, g4.make_beam_params(4, 8), s.state, g4.BeamState(s.lens.data_ptr(), None, None), *ptrs,
                           check=False)
    assert rc == g4.ERR_ARG and "n_out" in sampler.last_error()
    t = s.tab[0].data_ptr()
    same = g4.PageTables(t, s.plens.data_ptr(), s.refs.data_ptr())
    rc = sampler.beam_step(*args, s.params, s.state, s.state, *ptrs, s.dense,
                           g4.beam_pages(s.cache, same, same, 1, s.result.data_ptr()), check=False)
    assert rc == g4.ERR_ARG and "tables" in sampler.last_error()
    rc = sampler.beam_step(*args, s.params, s.state, s.state, *ptrs, [g4.BeamTensor(None, None, 4, 1, 0, 1, 0, 4)], check=False)
    assert rc == g4.ERR_ARG and "NULL" in sampler.last_error()
    torch.cuda.synchronize()
    for a, b in zip(before, (s.scores, s.lens, s.refs, s.par)):
        assert torch.equal(a, b)  # nothing was launched


def test_tables_without_pools(sampler, g4, torch_cuda):
    rng = np.random.default_rng(20)
    lens = rng.integers(0, 100, 9)
    tables, refs, rest = scattered(rng, 9, lens, 8, 20, 300)
    refs[rest[:40]] = 1
    cache = Cache(torch_cuda, g4, rng, 300, 8, 20, layouts=())
    run_fork(torch_cuda, g4, sampler, cache, tables, lens, refs, rng.integers(-1, 9, 12), 3)
    run_compact(torch_cuda, g4, sampler, cache, tables, lens, refs, False)
    run_fork(torch_cuda, g4, sampler, cache, np.full((0, 20), -1), [], refs, [-1, -1], 3)


def test_the_most_pools(sampler, g4, torch_cuda):
    rng = np.random.default_rng(9)
    layouts = tuple((1 + i % 3, (4, 16, 1, 20)[i % 4], i % 5, i % 2) for i in range(g4.PAGES_MAX_POOLS))
    P, width, n_pages = 4, 6, 60
    lens = rng.integers(1, width * P - 2, 6)
    cache = Cache(torch_cuda, g4, rng, n_pages, P, width, layouts=layouts)
    tables, refs, _ = scattered(rng, 6, lens, P, width, n_pages)
    run_fork(torch_cuda, g4, sampler, cache, tables, lens, refs, [0, 0, 1, 3, 3, 3], 1)
    cache = Cache(torch_cuda, g4, rng, n_pages, P, width, layouts=layouts)
    assert run_compact(torch_cuda, g4, sampler, cache, tables, lens, refs, False)[1] > 0


def test_pages_over_4_gib_in(g4, sampler, torch_cuda):
    torch = torch_cuda
    P, token, n_pages = 4, 1 << 18, 5000  # pages of 1 MiB
    pool = torch.zeros(n_pages * P * token, dtype=torch.uint8, device="cuda")
    page = pool.view(n_pages, P, token)
    page[4990, :3] = 7
    page[4991, :1] = 9
    cache = g4.page_cache([g4.PagePool(pool.data_ptr(), P * token, 1, 0, token)], P, n_pages, 2)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
    tables, lens = i32([[4990, -1], [4991, -1]]), i32([3, 1])
    refs = torch.ones(n_pages, dtype=torch.int32, device="cuda")
    refs[4999] = 0
    ot, ol, orf, res = i32([[-9, -9], [-9, -9]]), i32([0, 0]), torch.zeros_like(refs), i32([0, 0, 0, 0])
    src = i32([0, 0])
    torch.cuda.synchronize()
    sampler.pages_fork(cache, 2, tables.data_ptr(), lens.data_ptr(), refs.data_ptr(), 2, src.data_ptr(), 1, ot.data_ptr(),
                       ol.data_ptr(), orf.data_ptr(), res.data_ptr())
    torch.cuda.synchronize()
    # the second sequence's page is freed: it is the lowest free one, and takes the copy
    assert res.tolist() == [1, 0, 0, 0] and ot.tolist() == [[4991, -9], [4990, -9]] and ol.tolist() == [4, 4]
    assert bool((page[4991, :3] == 7).all()) and bool((page[4991, 3] == 0).all())
    del pool, page
    torch.cuda.empty_cache()


def test_fork_into_a_graph(sampler, g4, torch_cuda):
    """A captured fork and compaction, replayed on other tables in the same memory."""
    torch = torch_cuda
    rng = np.random.default_rng(21)
    n, P, width, n_pages = 6, 8, 12, 200
    cache = Cache(torch, g4, rng, n_pages, P, width)
    cu = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()
    lens = rng.integers(1, 50, n)
    tables, refs, _ = scattered(rng, n, lens, P, width, n_pages)
    dt, dl, dr, ds = cu(tables), cu(lens), cu(refs), cu(np.zeros(n))
    ot, ol, orf, res = cu(np.full((n, width), -9)), cu(np.zeros(n)), cu(np.zeros(n_pages)), cu(np.zeros(4))
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        sampler.pages_fork(cache.c, n, dt.data_ptr(), dl.data_ptr(), dr.data_ptr(), n, ds.data_ptr(), 2, ot.data_ptr(),
                           ol.data_ptr(), orf.data_ptr(), res.data_ptr(), stream=stream.cuda_stream)
    for k in range(4):
        lens = rng.integers(0, 80, n)
        tables, refs, _ = scattered(rng, n, lens, P, width, n_pages)
        src = rng.integers(-1, n, n)
        for d, h in ((dt, tables), (dl, lens), (dr, refs), (ds, src)):
            d.copy_(cu(h))
        for d, h in zip(cache.dev, cache.host):
            d.copy_(torch.from_numpy(h))
        ot.fill_(-9)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        wt, wl, wr, want, copies = beam_util.fork(tables, lens, refs, src, 2, P, width)
        assert res.tolist() == want and np.array_equal(ot.cpu().numpy(), wt) and np.array_equal(ol.cpu().numpy(), wl)
        assert np.array_equal(orf.cpu().numpy(), wr)
        cache.check(copies)


def test_fork_repeated_in_place_leaks_nothing(sampler, g4, torch_cuda):
    """A long run of forks, growth, frees and compactions in place: the counts are what the tables hold."""
    torch = torch_cuda
    rng = np.random.default_rng(22)
    n, P, width, n_pages = 12, 4, 40, 400
    cache = Cache(torch, g4, rng, n_pages, P, width, layouts=((1, 16, 0, 0),))
    cu = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()
    tab = [cu(np.full((n, width), -1)), cu(np.full((n, width), -1))]
    lens, refs, res = cu(np.zeros(n)), cu(np.zeros(n_pages)), cu(np.zeros(4))
    mp, mv = cu(np.zeros(n_pages)), cu(np.zeros(n_pages))
    for k in range(120):
        a, b = tab[k % 2], tab[1 - k % 2]
        src = np.arange(n) if k == 0 else rng.integers(0, n, n)
        if k % 17 == 16:
            src[rng.integers(0, n, 5)] = -1
        ds = cu(src)
        torch.cuda.synchronize()
        sampler.pages_fork(cache.c, n, a.data_ptr(), lens.data_ptr(), refs.data_ptr(), n, ds.data_ptr(), int(rng.integers(0, 4)),
                           b.data_ptr(), lens.data_ptr(), refs.data_ptr(), res.data_ptr())
        if k % 10 == 9:
            sampler.pages_compact(cache.c, n, b.data_ptr(), lens.data_ptr(), refs.data_ptr(), b.data_ptr(), refs.data_ptr(),
                                  mp.data_ptr(), mv.data_ptr(), res.data_ptr())
        torch.cuda.synchronize()
        assert res.tolist()[3] == 0
        L, T = lens.cpu().numpy(), b.cpu().numpy()
        held = np.zeros(n_pages, np.int64)
        for i in range(n):
            np.add.at(held, T[i, :-(-int(L[i]) // P)], 1)
        assert np.array_equal(held, refs.cpu().numpy()), k
        if L.max() > width * P - 8:
            lens.zero_()
            refs.zero_()
