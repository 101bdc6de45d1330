"""Beam search on the GPU: its selection, the reordering of its states, and the pages of its cache.

Four operators of a beam-search decode step, each at sizes from one prompt to a full batch:

  select    the best continuations of every prompt's beams over beams x vocabulary
  reorder   the beams' dense states gathered by the selected parents
  fork      a paged cache forked by the selected parents: shared pages counted,
            the partly filled last page copied on write, room for the next tokens,
            pages that no sequence holds any more freed
  compact   a paged cache's used pages moved to the lowest ids

`own` chooses between the plain torch form of each (False) and the library's calls (True).
"""
import functools
import math
import os
import sys

import numpy as np
import torch

own = False

MASKED = -1e30  # a logit at or below this is masked (as on the sampler's top-K path)
EOS = (1, 106, 50)  # the model family's end tokens


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _select(name, dtype, groups, beams, out, vocab, pad, softcap, temperature, alpha, masked, done):
    """One beam-search selection.  pad: elements between the rows' ends and the next start; masked:
    share of the vocabulary that a grammar forbids; done: every done-th beam has ended (0: none)."""
    return {"op": "select", "name": name, "dtype": dtype, "groups": groups, "beams": beams, "out": out,
            "vocab": vocab, "pad": pad, "softcap": softcap, "temperature": temperature, "alpha": alpha,
            "masked": masked, "done": done}


def _reorder(name, dtype, groups, beams, layers, heads, max_len, live, dim):
    """Dense caches [layers][rows][heads][max_len][dim] (two of them) and the rows' token history."""
    return {"op": "reorder", "name": name, "dtype": dtype, "groups": groups, "beams": beams, "layers": layers,
            "heads": heads, "max_len": max_len, "live": live, "dim": dim}


def _fork(name, dtype, groups, beams, pools, segs, page_tokens, width, pages, prompt_lo, prompt_hi, grown, new):
    """A paged cache of `pools` pools of `pages` pages; prompts of prompt_lo..prompt_hi tokens shared by a
    group's beams, `grown` tokens of each beam's own, room asked for `new` more."""
    return {"op": "fork", "name": name, "dtype": dtype, "groups": groups, "beams": beams, "pools": pools,
            "segs": segs, "page_tokens": page_tokens, "width": width, "pages": pages, "prompt_lo": prompt_lo,
            "prompt_hi": prompt_hi, "grown": grown, "new": new}


def _compact(name, dtype, seqs, pools, page_tokens, width, pages, length, used):
    """A fragmented cache: `seqs` sequences of about `length` tokens scattered over the `pages` pages, of
    which a share `used` is held (by the sequences, and by a prefix cache that only counts them)."""
    return {"op": "compact", "name": name, "dtype": dtype, "seqs": seqs, "pools": pools,
            "page_tokens": page_tokens, "width": width, "pages": pages, "length": length, "used": used}


def listed():
    return [
        # an interactive answer with 4 beams: one prompt, latency counts
        _select("select, one prompt, 4 beams", "f32", 1, 4, 4, 262144, 0, 30.0, 1.0, 0.0, 0.0, 0),
        # offline decoding of a batch, candidates for 2 x beams as schemes with finished lists keep
        _select("select, 32 prompts x 8 beams, bf16", "bf16", 32, 8, 16, 262144, 0, 30.0, 1.0, 0.0, 0.0, 0),
        # the same in fp32 with a length penalty and beams that have ended
        _select("select, 32 prompts x 8 beams, fp32, ended beams", "f32", 32, 8, 8, 262144, 0, 30.0, 1.0, 0.6, 0.0, 5),
        # constrained decoding: a grammar leaves a tenth of the vocabulary
        _select("select, grammar, 16 prompts x 4 beams", "bf16", 16, 4, 4, 262144, 0, 30.0, 0.8, 0.0, 0.9, 0),
        # a small odd vocabulary without softcap in rows that no vector load fits
        _select("select, odd vocabulary, 7 prompts x 5 beams", "f32", 7, 5, 10, 32003, 2, 0.0, 0.7, 1.0, 0.0, 6),
        # the 512-position window caches of one prompt's beams, early in the window
        _reorder("reorder, one prompt, 4 beams", "bf16", 1, 4, 4, 2, 512, 33, 256),
        # a batch whose windows are almost full
        _reorder("reorder, 8 prompts x 8 beams", "bf16", 8, 8, 8, 2, 512, 509, 256),
        # one prompt's beams over a small page pool
        _fork("fork, one prompt, 4 beams", "bf16", 1, 4, 4, 1, 16, 256, 1024, 300, 300, 21, 1),
        # a batch over a large pool
        _fork("fork, 32 prompts x 8 beams", "bf16", 32, 8, 4, 1, 16, 512, 12288, 500, 4000, 137, 1),
        # long sequences in large pages, heads before positions, several drafted tokens at once
        _fork("fork, 8 prompts x 6 beams, long", "f32", 8, 6, 6, 2, 64, 640, 4096, 9000, 30000, 777, 5),
        # a small pool after a few sequences ended
        _compact("compact, small pool", "bf16", 7, 4, 16, 64, 512, 300, 0.4),
        # a large pool, over half of it held
        _compact("compact, large pool", "bf16", 64, 4, 16, 512, 8192, 1000, 0.6),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["select", "select", "reorder", "fork", "fork", "compact"])
    if op == "select":
        dtype = rng.choice(["f32", "bf16"])
        beams = rng.randint(1, 16)
        vocab = _log(rng, 1000, 262144)
        most = 250_000_000 // (vocab * beams * (4 if dtype == "f32" else 2))
        groups = _log(rng, 1, max(1, min(64, most)))
        return {k: v for k, v in _select("", dtype, groups, beams, rng.choice([beams, 2 * beams]), vocab,
                                         rng.choice([0, 0, 1, 8, 37]), rng.choice([0.0, 30.0]),
                                         rng.choice([1.0, round(rng.uniform(0.5, 1.5), 2)]),
                                         rng.choice([0.0, 0.6, 1.0]), rng.choice([0.0, 0.0, 0.5, 0.95]),
                                         rng.choice([0, 0, 4, 7])).items() if k != "name"}
    if op == "reorder":
        heads, dim, max_len = rng.randint(1, 4), rng.choice([16, 40, 64, 128, 256]), _log(rng, 32, 1024)
        groups, beams, layers = _log(rng, 1, 16), rng.randint(2, 16), rng.randint(1, 8)
        most = 130_000_000 // (heads * dim * max_len * layers)
        beams = max(2, min(beams, most))
        groups = max(1, min(groups, most // beams))
        return {k: v for k, v in _reorder("", rng.choice(["bf16", "f32"]), groups, beams, layers, heads, max_len,
                                          rng.randint(1, max_len), dim).items() if k != "name"}
    if op == "fork":
        groups, beams = _log(rng, 1, 32), rng.randint(2, 12)
        page = rng.choice([8, 16, 32, 64])
        lo = _log(rng, 1, 2000)
        hi = lo + _log(rng, 1, 2000)
        grown = _log(rng, 1, 300)
        new = rng.choice([0, 1, 1, 1, 4, 17])
        need = int(1.1 * groups * ((hi + page - 1) // page + 1 + beams * ((grown + 2 * new) // page + 4))) + 64
        return {k: v for k, v in _fork("", rng.choice(["bf16", "f32"]), groups, beams, rng.randint(1, 6),
                                       rng.choice([1, 1, 2]), page, (hi + grown + new) // page + 2 + rng.randint(0, 99),
                                       need + rng.randint(0, need), lo, hi, grown, new).items() if k != "name"}
    pages, page = _log(rng, 64, 8192), rng.choice([8, 16, 32])
    length = _log(rng, 20, 1000)
    used = round(rng.uniform(0.2, 0.9), 2)
    seqs = max(1, int(pages * used * 0.7) // ((length + page - 1) // page + 1))
    seqs = min(seqs, 64)
    pools = rng.randint(1, 4 if page <= 16 else 2)
    return {k: v for k, v in _compact("", rng.choice(["bf16", "bf16", "f32"] if pools <= 2 else ["bf16"]), seqs, pools,
                                      page, (2 * length + page - 1) // page + 2, pages, length, used).items()
            if k != "name"}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
_T = {"f32": torch.float32, "bf16": torch.bfloat16}
HEAD_DIM = {1: 512, 2: 256}  # elements of one position and segment: two heads of 256 together, or apart


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def _prepare_select(case, seed):
    g = _gen(seed)
    G, W, V = case["groups"], case["beams"], case["vocab"]
    R, stride = G * W, V + case["pad"]
    x = torch.randn(R, stride, device="cuda", generator=g).mul_(2.5)
    # a few likely tokens a row, as a trained model gives
    at = torch.randint(0, V, (R, 24), device="cuda", generator=g)
    x.scatter_reduce_(1, at, torch.rand(R, 24, device="cuda", generator=g).mul_(10.0).add_(5.0), "amax")
    if case["masked"] > 0:
        x.masked_fill_(torch.rand(R, stride, device="cuda", generator=g) < case["masked"], -math.inf)
    logits = x.to(_T[case["dtype"]])
    rng = np.random.default_rng(seed)
    lens = rng.integers(3, 60, size=(G, 1)).repeat(W, 1)
    done = np.zeros((G, W), np.uint8)
    if case["done"]:
        done.reshape(-1)[case["done"] - 1::case["done"]] = 1
        lens = np.where(done > 0, np.maximum(1, lens - rng.integers(1, 20, size=(G, W))), lens)
    scores = -lens * rng.uniform(0.5, 1.0, (G, 1)) - rng.exponential(2.0, (G, W))
    st = {"case": case, "logits": logits, "stride": stride,
          "scores": torch.from_numpy(scores.astype(np.float32)).cuda(), "lens": _i32(lens),
          "done": torch.from_numpy(done).cuda()}
    N = case["out"]
    st["out"] = {"scores": torch.empty(G, N, device="cuda"), "parents": torch.empty(G, N, dtype=torch.int32, device="cuda"),
                 "tokens": torch.empty(G, N, dtype=torch.int32, device="cuda"),
                 "lens": torch.empty(G, N, dtype=torch.int32, device="cuda"),
                 "done": torch.empty(G, N, dtype=torch.uint8, device="cuda")}
    return st


def _parents(rng, G, W):
    """Parents [G, W] as beam search picks them: about half of the beams survive, some several times."""
    keep = max(1, (W + 1) // 2)
    out = np.empty((G, W), np.int64)
    for g in range(G):
        alive = rng.permutation(W)[:keep]
        p = np.concatenate([alive, alive[rng.integers(0, keep, W - keep)]])
        out[g] = g * W + rng.permutation(p)
    return out


def _prepare_reorder(case, seed):
    g = _gen(seed)
    L, H, M, D = case["layers"], case["heads"], case["max_len"], case["dim"]
    R = case["groups"] * case["beams"]
    kv = torch.randn(2, L, R, H, M, D, device="cuda", generator=g).to(_T[case["dtype"]])
    hist = torch.randint(0, 262144, (R, M), device="cuda", generator=g, dtype=torch.int32)
    rng = np.random.default_rng(seed)
    return {"case": case, "kv": kv, "hist": hist, "parents": _i32(_parents(rng, case["groups"], case["beams"]).reshape(-1)),
            "out": {"kv": torch.zeros_like(kv), "hist": torch.zeros_like(hist)}}


def _prompt_len(case, g):
    lo, hi = case["prompt_lo"], case["prompt_hi"]
    return lo + int((hi - lo) * ((g * 0.6180339887) % 1.0))


def _prepare_fork(case, seed):
    G, W, P = case["groups"], case["beams"], case["page_tokens"]
    rng = np.random.default_rng(seed)
    ids = rng.permutation(case["pages"])  # a pool that has been in use for a while: pages in no order
    table = np.full((G * W, case["width"]), -1, np.int64)
    lens = np.empty(G * W, np.int64)
    refs = np.zeros(case["pages"], np.int64)
    at = 0
    for g in range(G):
        shared = _prompt_len(case, g) // P  # whole pages of the prompt are shared
        total = _prompt_len(case, g) + case["grown"]
        pages = (total + P - 1) // P
        common = ids[at:at + shared]
        at += shared
        for w in range(W):
            r = g * W + w
            table[r, :shared] = common
            table[r, shared:pages] = ids[at:at + pages - shared]
            at += pages - shared
            lens[r] = total
            refs[table[r, :pages]] += 1
    refs[ids[at:at + case["pages"] // 50]] += 1  # pages held by a prefix cache
    src = _parents(rng, G, W).reshape(-1)
    D = HEAD_DIM[case["segs"]]
    pools = torch.randn(case["pools"], case["pages"], case["segs"], P, D, device="cuda", generator=_gen(seed),
                        dtype=torch.float32 if case["dtype"] == "f32" else torch.bfloat16)
    return {"case": case, "pools": pools, "table": _i32(table), "lens": _i32(lens), "refs": _i32(refs),
            "src": _i32(src),
            "out": {"table": torch.full((G * W, case["width"]), -1, dtype=torch.int32, device="cuda"),
                    "lens": torch.zeros(G * W, dtype=torch.int32, device="cuda"),
                    "refs": torch.zeros(case["pages"], dtype=torch.int32, device="cuda"),
                    "result": torch.zeros(4, dtype=torch.int32, device="cuda")}}


def _compact_lens(case):
    return [max(1, int(case["length"] * (0.5 + (i * 0.6180339887) % 1.0))) for i in range(case["seqs"])]


def _prepare_compact(case, seed):
    P = case["page_tokens"]
    rng = np.random.default_rng(seed)
    ids = rng.permutation(case["pages"])
    lens = _compact_lens(case)
    table = np.full((case["seqs"], case["width"]), -1, np.int64)
    refs = np.zeros(case["pages"], np.int64)
    at = 0
    for i, n in enumerate(lens):
        pages = (n + P - 1) // P
        pages = min(pages, case["pages"] - at)
        lens[i] = min(n, pages * P)
        table[i, :pages] = ids[at:at + pages]
        at += pages
    refs[ids[:at]] = 1
    extra = max(0, int(case["pages"] * case["used"]) - at)
    refs[ids[at:at + extra]] = 2  # held by a prefix cache
    D = HEAD_DIM[1]
    pools = torch.randn(case["pools"], case["pages"], 1, P, D, device="cuda", generator=_gen(seed),
                        dtype=torch.float32 if case["dtype"] == "f32" else torch.bfloat16)
    n = case["pages"]
    return {"case": case, "pools": pools, "table": _i32(table), "lens": _i32(lens), "refs": _i32(refs),
            "out": {"table": torch.full((case["seqs"], case["width"]), -1, dtype=torch.int32, device="cuda"),
                    "refs": torch.zeros(n, dtype=torch.int32, device="cuda"),
                    "map": torch.zeros(n, dtype=torch.int32, device="cuda"),
                    "moves": torch.zeros(n, dtype=torch.int32, device="cuda"),
                    "result": torch.zeros(4, dtype=torch.int32, device="cuda")}}


def prepare(case, seed):
    return {"select": _prepare_select, "reorder": _prepare_reorder, "fork": _prepare_fork,
            "compact": _prepare_compact}[case["op"]](case, seed)


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _softcap(x, cap):
    return cap * torch.tanh(x / cap) if cap > 0 else x


def _plain_select(s):
    c = s["case"]
    G, W, N, V, T = c["groups"], c["beams"], c["out"], c["vocab"], c["temperature"]
    raw = s["logits"][:, :V].float()
    raw = torch.where(raw > MASKED, raw, -math.inf)
    raw = raw.clamp(max=torch.finfo(torch.float32).max) + 0.0
    x = torch.where(raw == -math.inf, raw, _softcap(raw, c["softcap"]))
    top = x.amax(1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    # the sum and what decides between candidates in 64 bits
    norm = torch.exp((x - top) / T).sum(1, dtype=torch.float64).log()
    # each row's best by raw logit, then by the lower id: one whole number orders both
    bits = raw.view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).to(torch.int64)
    key = (key << 32) | (0x7FFFFFFF - torch.arange(V, device=raw.device))
    n = min(N, V)
    ids = 0x7FFFFFFF - (torch.topk(key, n, dim=1).values & 0x7FFFFFFF)
    best = raw.gather(1, ids)
    logp = (_softcap(best.double(), c["softcap"]) - top.double()) / T - norm[:, None]
    scores, lens, done = s["scores"].double().view(-1, 1), s["lens"].view(-1, 1), s["done"].view(-1, 1) > 0
    first = torch.arange(n, device=raw.device) == 0
    cand = torch.where(done, torch.where(first, scores, -math.inf), scores + logp)
    cand = torch.where((best == -math.inf) & ~done, -math.inf, cand)
    ids = torch.where(done, 0, ids)
    after = lens + (~done).int()
    rank = cand * after.clamp(min=1).double() ** -c["alpha"]
    rank, cand, ids = (t.reshape(G, W * n) for t in (rank, cand, ids))
    rank, at = torch.sort(rank, dim=1, descending=True, stable=True)
    rank, at = rank[:, :N], at[:, :N]
    if W * n < N:
        rank = torch.nn.functional.pad(rank, (0, N - W * n), value=-math.inf)
        at = torch.nn.functional.pad(at, (0, N - W * n))
    none = rank == -math.inf
    row = torch.arange(G, device=raw.device)[:, None] * W + at // n
    token = ids.gather(1, at)
    ended = torch.isin(token, torch.tensor(EOS, device=raw.device)) | done.view(-1)[row]
    return {"scores": torch.where(none, -math.inf, cand.gather(1, at)).float(),
            "parents": torch.where(none, -1, row).int(), "tokens": torch.where(none, -1, token).int(),
            "lens": torch.where(none, 0, after.view(-1)[row]).int(), "done": (ended & ~none).to(torch.uint8)}


def _plain_reorder(s):
    n, p, out = s["case"]["live"], s["parents"], s["out"]
    out["kv"][..., :n, :] = s["kv"][..., :n, :].index_select(2, p)
    out["hist"][:, :n] = s["hist"][:, :n].index_select(0, p)
    return out


def _plain_fork(s):
    c, out, dev = s["case"], s["out"], s["table"].device
    P, new, refs, src = c["page_tokens"], c["new"], s["refs"].long(), s["src"].long()
    col = torch.arange(c["width"], device=dev)
    held = lambda lens: col < ((lens + P - 1) // P)[:, None]  # noqa: E731
    # the new sequences hold their parents' pages, the old ones none
    table, lens = s["table"].long()[src], s["lens"].long()[src]
    one = torch.ones((), dtype=torch.int64, device=dev)
    old = s["table"].long()
    refs = refs.index_put((old[held(s["lens"].long())],), -one, accumulate=True)
    refs = refs.index_put((table[held(lens)],), one, accumulate=True)
    # a partly filled last page that another holds too is copied; the last of its writers keeps it
    part = (lens % P != 0) & (new > 0)
    last = table.gather(1, (lens // P).clamp(max=c["width"] - 1)[:, None])[:, 0]
    same = (last[:, None] == last[None, :]) & part[:, None] & part[None, :]
    before = same.tril(-1).sum(1)
    copy = part & (before < refs[last] - 1)
    grow = (lens + new + P - 1) // P - (lens + P - 1) // P
    need = copy.long() + grow
    free = torch.nonzero(refs <= 0)[:, 0]
    start = need.cumsum(0) - need
    taken = need.sum()
    # the copied page's new id goes into the last page's column, the grown ones behind it
    shift = col[None, :] - (lens // P)[:, None] - torch.where(part & ~copy, 1, 0)[:, None]
    mine = (shift >= 0) & (shift < need[:, None])
    table = torch.where(mine, free[(start[:, None] + shift).clamp(0, free.numel() - 1)], table)
    refs = refs.index_put((last[copy],), -one, accumulate=True)
    refs[free[:taken]] = 1
    keep = held(lens + new)
    out["table"].copy_(torch.where(keep, table, out["table"].long()))
    out["lens"].copy_(lens + new)
    out["refs"].copy_(refs)
    out["result"].copy_(torch.stack([taken, 0 * taken, 0 * taken, 0 * taken]))
    # the filled positions of the copied pages
    a, b = last[copy], free[start[copy]]
    filled = (torch.arange(P, device=dev)[None, :] < (lens % P)[copy][:, None])[None, :, None, :, None]
    s["pools"][:, b] = torch.where(filled, s["pools"][:, a], s["pools"][:, b])
    return {**out, "pools": s["pools"]}


def _plain_compact(s):
    c, out, dev = s["case"], s["out"], s["table"].device
    refs = s["refs"]
    used = refs > 0
    n = used.sum()
    page = torch.arange(c["pages"], device=dev)
    a, b = torch.nonzero(used & (page >= n))[:, 0], torch.nonzero(~used & (page < n))[:, 0]
    to = torch.where(used, page, -1)
    to[a] = b
    out["map"].copy_(to)
    out["moves"][:2 * a.numel()] = torch.stack([a, b], 1).reshape(-1).int()
    out["result"].copy_(torch.stack([n, (used & (page >= n)).sum(), 0 * n, 0 * n]))
    moved = torch.where(page < n, refs, 0)
    moved[b] = refs[a]
    out["refs"].copy_(moved)
    P = c["page_tokens"]
    held = torch.arange(c["width"], device=dev) < ((s["lens"] + P - 1) // P)[:, None]
    out["table"].copy_(torch.where(held, to[s["table"].long().clamp(min=0)], out["table"].long()))
    s["pools"][:, b] = s["pools"][:, a]
    return {**out, "pools": s["pools"]}


# ---------------------------------------------------------------------------
# the library's calls
# ---------------------------------------------------------------------------
@functools.lru_cache(None)
def _library():
    """The context that a user's program keeps."""
    at = os.path.join(os.getcwd(), "gemma4.pas_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import g4sampler

    return g4sampler, g4sampler.Sampler(device=_device(), max_rows=1024, max_vocab=262144)


@functools.lru_cache(None)
def _device():
    """The context's device."""
    return torch.cuda.current_device()


def _stream():
    """The current stream, on which the inputs were made and the results are read.  The legacy default stream's
    handle is 0, which the library takes for its context's own stream; 1 names it.  (By the raw handle: a Stream
    object a call takes 3 us, as long as the smallest operator.)"""
    return torch._C._cuda_getCurrentRawStream(_device()) or 1


def _own_select(s):
    c, o = s["case"], s["out"]
    g4, sampler = _library()
    if "plan" not in s:
        s["plan"] = (g4.make_beam_params(c["beams"], c["out"], c["temperature"], c["alpha"], pad_token=0, eos=EOS),
                     g4.BeamState(s["scores"].data_ptr(), s["lens"].data_ptr(), s["done"].data_ptr()),
                     g4.BeamState(o["scores"].data_ptr(), o["lens"].data_ptr(), o["done"].data_ptr()))
    params, before, after = s["plan"]
    sampler.beam_select(s["logits"].data_ptr(), g4.F32 if c["dtype"] == "f32" else g4.BF16, c["groups"], c["vocab"],
                        s["stride"], c["softcap"], params, before, after, o["parents"].data_ptr(), o["tokens"].data_ptr(),
                        stream=_stream())
    return o


def _own_reorder(s):
    c, o = s["case"], s["out"]
    g4, sampler = _library()
    if "plan" not in s:
        e, M, D, H = s["kv"].element_size(), c["max_len"], c["dim"], c["heads"]
        R = c["groups"] * c["beams"]
        # K and V of every layer are 2 * layers planes of [rows][heads][max_len][dim]
        kv = g4.BeamTensor(s["kv"].data_ptr(), o["kv"].data_ptr(), H * M * D * e, 2 * c["layers"], R * H * M * D * e,
                           H, M * D * e, c["live"] * D * e)
        hist = g4.BeamTensor(s["hist"].data_ptr(), o["hist"].data_ptr(), M * 4, 1, 0, 1, 0, c["live"] * 4)
        s["plan"] = g4.beam_tensors([kv, hist])
    sampler.beam_reorder(s["parents"].data_ptr(), c["groups"], c["beams"], s["plan"], stream=_stream())
    return o


def _cache(g4, s):
    c = s["case"]
    n, size, e = c["pools"], s["pools"].stride(1), s["pools"].element_size()
    segs, D = s["pools"].shape[2], s["pools"].shape[4]
    return g4.page_cache([g4.PagePool(s["pools"][i].data_ptr(), size * e, segs, s["pools"].stride(2) * e, D * e)
                          for i in range(n)], c["page_tokens"], c["pages"], c["width"])


def _own_fork(s):
    c, o = s["case"], s["out"]
    g4, sampler = _library()
    if "plan" not in s:
        s["plan"] = _cache(g4, s)
    rows = c["groups"] * c["beams"]
    sampler.pages_fork(s["plan"], rows, s["table"].data_ptr(), s["lens"].data_ptr(), s["refs"].data_ptr(), rows,
                       s["src"].data_ptr(), c["new"], o["table"].data_ptr(), o["lens"].data_ptr(),
                       o["refs"].data_ptr(), o["result"].data_ptr(), stream=_stream())
    return {**o, "pools": s["pools"]}


def _own_compact(s):
    c, o = s["case"], s["out"]
    g4, sampler = _library()
    if "plan" not in s:
        s["plan"] = _cache(g4, s)
    sampler.pages_compact(s["plan"], c["seqs"], s["table"].data_ptr(), s["lens"].data_ptr(), s["refs"].data_ptr(),
                          o["table"].data_ptr(), o["refs"].data_ptr(), o["map"].data_ptr(), o["moves"].data_ptr(),
                          o["result"].data_ptr(), stream=_stream())
    return {**o, "pools": s["pools"]}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"select": _own_select, "reorder": _own_reorder, "fork": _own_fork, "compact": _own_compact}[op](state)
    return {"select": _plain_select, "reorder": _plain_reorder, "fork": _plain_fork, "compact": _plain_compact}[op](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    if case["op"] == "select":
        rows = case["groups"] * case["beams"]
        live = rows - (rows // case["done"] if case["done"] else 0)
        e = 4 if case["dtype"] == "f32" else 2
        # one exponential, one sum and one comparison a logit, and the softcap's tanh
        return {"bytes": live * case["vocab"] * e + rows * 9 + case["groups"] * case["out"] * 17,
                "flops": live * case["vocab"] * (6 if case["softcap"] > 0 else 4)}
    if case["op"] == "reorder":
        e = 4 if case["dtype"] == "f32" else 2
        row = 2 * case["layers"] * case["heads"] * case["live"] * case["dim"] * e + case["live"] * 4
        keep = max(1, (case["beams"] + 1) // 2)  # distinct parents are read once
        return {"bytes": case["groups"] * (keep + case["beams"]) * row, "flops": 0}
    token = case["pools"] * 512 * (4 if case["dtype"] == "f32" else 2)
    if case["op"] == "fork":
        G, W, P = case["groups"], case["beams"], case["page_tokens"]
        keep = max(1, (W + 1) // 2)
        lens = [_prompt_len(case, g) + case["grown"] for g in range(G)]
        fill = sum(n % P for n in lens) if case["new"] else 0  # positions of each group's partly filled pages
        entries = sum((n + P - 1) // P for n in lens) * W
        # a page that k sequences take is copied k - 1 times; tables read and written, counts too
        copied = (W - keep) * fill * token
        return {"bytes": copied + min(copied, keep * fill * token) + entries * 8 + case["pages"] * 8, "flops": 0}
    # used pages at or above the count of used pages move: a share 1 - used of them
    P = case["page_tokens"]
    held = min(sum((n + P - 1) // P for n in _compact_lens(case)), case["pages"])
    used = max(held, int(case["pages"] * case["used"]))
    moved = used * (1 - used / case["pages"])
    return {"bytes": 2 * moved * P * token + held * 8 + case["pages"] * 12, "flops": 0}


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    """The selection's scores; the other operators move bytes and compute no number."""
    if case["op"] != "select":
        return None
    s = prepare(case, seed)
    G, W, N, V = case["groups"], case["beams"], case["out"], case["vocab"]
    alpha = case["alpha"]
    found = []
    for g in range(G):
        z = s["logits"][g * W:(g + 1) * W, :V].to(torch.float64)
        allowed = z > MASKED
        if case["softcap"] > 0:
            e = torch.exp(-2.0 * z.abs() / case["softcap"])
            z = torch.sign(z) * case["softcap"] * (1.0 - e) / (1.0 + e)
        z = torch.where(allowed, z / case["temperature"], torch.full_like(z, -math.inf))
        logp = z - torch.logsumexp(z, 1, keepdim=True)
        total = s["scores"][g].to(torch.float64)[:, None] + torch.nan_to_num(logp, nan=-math.inf)
        ended = s["done"][g] > 0
        total[ended] = -math.inf
        total[ended, 0] = s["scores"][g].to(torch.float64)[ended]
        length = s["lens"][g].to(torch.float64) + (~ended).to(torch.float64)
        share = torch.pow(torch.clamp(length, min=1.0), alpha)[:, None]
        value, at = torch.topk((total / share).reshape(-1), min(N, W * V))
        score = total.reshape(-1)[at]
        score[value == -math.inf] = -math.inf
        found.append(torch.nn.functional.pad(score, (0, N - score.numel()), value=-math.inf))
    return {"scores": torch.stack(found), "parents": None, "tokens": None, "lens": None, "done": None}
