"""Plain 64-bit forms of the beam-search operators, written from their definitions,
which the GPU tests compare with."""
from __future__ import annotations

import numpy as np

NEG = -np.inf
EOS = (1, 106, 50)


def select(logits, scores, lens, done, W, N, cap, T, alpha, pad=0, eos=EOS, fmax=float(np.finfo(np.float32).max)):
    """g4s_beam_select of [rows, V] float64 logits: a list per group of (rank, score, row, token, len, done),
    every candidate in order (not only the first N).  fmax: what +inf counts as."""
    rows, V = logits.shape
    out = []
    for g in range(rows // W):
        rank, score, row, raw, tok = [], [], [], [], []
        for r in range(g * W, (g + 1) * W):
            if not scores[r] > NEG:
                continue
            length = int(lens[r]) + (0 if done[r] else 1)
            norm = float(max(length, 1)) ** alpha
            if done[r]:
                rank.append(np.array([float(scores[r]) / norm]))
                score.append(np.array([float(scores[r])]))
                raw.append(np.array([0.0]))
                tok.append(np.array([pad]))
                row.append(np.array([r]))
                continue
            x = logits[r]
            ok = np.nonzero(x > -1e30)[0]
            if ok.size == 0:
                continue
            v = np.minimum(x[ok], fmax) + 0.0
            s = cap * np.tanh(v / cap) if cap > 0 else v
            m = s.max()
            with np.errstate(over="ignore"):
                logp = (s - m) / T - np.log(np.sum(np.exp((s - m) / T)))
            sc = float(scores[r]) + logp
            # only the row's best N can be among the group's: by raw logit, then id
            keep = np.lexsort((ok, -v))[:N]
            rank.append(sc[keep] / norm)
            score.append(sc[keep])
            raw.append(v[keep])
            tok.append(ok[keep])
            row.append(np.full(keep.size, r))
        if not rank:
            out.append([])
            continue
        rank, score, row, raw, tok = (np.concatenate(z) for z in (rank, score, row, raw, tok))
        order = np.lexsort((tok, -raw, row, -rank))
        out.append([(rank[i], score[i], int(row[i]), int(tok[i]),
                     int(lens[row[i]]) + (0 if done[row[i]] else 1),
                     int(bool(done[row[i]]) or int(tok[i]) in eos)) for i in order])
    return out


def fork(tables, lens, refs, src, n_new, P, width, frozen=None, out_tables=None):
    """g4s_pages_fork, sequence by sequence.  Returns tables, lens, refs, result, copies."""
    n_pages = len(refs)
    refs = refs.astype(np.int64).copy()
    ok_len = lambda n: 0 <= n <= width * P
    pages = lambda n: -(-n // P)
    bad = 0
    kids = np.zeros(len(lens), np.int64)
    cur = []
    for s in src:
        if s < 0:
            cur.append(-1)
        elif s >= len(lens) or not ok_len(lens[s]):
            cur.append(-1)
            bad += 1
        else:
            cur.append(int(lens[s]))
            kids[s] += 1
    for i, n in enumerate(lens):
        if ok_len(n):
            for p in tables[i, :pages(n)]:
                if 0 <= p < n_pages:
                    refs[p] += kids[i] - 1
    out = np.full((len(src), width), -9, np.int64) if out_tables is None else out_tables.astype(np.int64).copy()
    for j, n in enumerate(cur):
        if n > 0:
            row = tables[src[j], :pages(n)]
            out[j, :pages(n)] = row
            bad += int(((row < 0) | (row >= n_pages)).sum())
    new_lens = np.array([max(n, 0) for n in cur], np.int64)
    over = 0
    plan = []  # (sequence, copied page or -1, new pages)
    left = refs.copy()
    for j, n in enumerate(cur):
        if n < 0 or n_new == 0 or (frozen is not None and frozen[j]):
            continue
        copy = -1
        if n % P:
            p = int(out[j, n // P])
            if 0 <= p < n_pages and left[p] > 1:
                copy = p
                left[p] -= 1
        if pages(n + n_new) > width:
            over += 1
            if copy >= 0:
                left[copy] += 1  # what it would have done no longer matters: nothing is taken
            continue
        plan.append((j, copy, pages(n + n_new) - pages(n)))
    need = sum((c >= 0) + k for _, c, k in plan)
    free = np.nonzero(refs <= 0)[0]
    short = max(0, need - free.size)
    copies = []
    result = [0, short, over, bad]
    if not (short or over or bad):
        result[0] = need
        at = 0
        for j, copy, grow in plan:
            n = cur[j]
            if copy >= 0:
                out[j, n // P] = free[at]
                copies.append((copy, int(free[at]), n % P))
                refs[copy] -= 1
                refs[free[at]] = 1
                at += 1
            for k in range(grow):
                out[j, pages(n) + k] = free[at]
                refs[free[at]] = 1
                at += 1
            new_lens[j] = n + n_new
        # sequences without a plan entry (frozen, empty) keep their length
    return out, new_lens, refs, result, copies


def compact(tables, lens, refs, P, width):
    """g4s_pages_compact: tables, refs, map, moves, result."""
    n_pages = len(refs)
    used = np.nonzero(refs > 0)[0]
    U = used.size
    frm = used[used >= U]
    holes = np.array([p for p in range(U) if refs[p] <= 0], np.int64)
    page_map = np.full(n_pages, -1, np.int64)
    page_map[used] = used
    page_map[frm] = holes
    new_refs = np.zeros(n_pages, np.int64)
    new_refs[page_map[used]] = refs[used]
    out = tables.astype(np.int64).copy()
    bad = 0
    for i, n in enumerate(lens):
        m = min(max(int(n), 0), width * P)
        bad += m != n
        for c in range(-(-m // P)):
            p = tables[i, c]
            if 0 <= p < n_pages:
                out[i, c] = page_map[p]
                bad += page_map[p] < 0
            else:
                bad += 1
    return out, new_refs, page_map, np.stack([frm, holes], 1).reshape(-1), [U, frm.size, 0, bad]
