"""NumPy restatement of the operators over shared pages, a shared prefix and selected key blocks: integers exactly, attention
in 64 bits.  The rules are those of include/dtattn.h."""
from __future__ import annotations

import numpy as np


def references(table, num_pages):
    slots = table[(table >= 0) & (table < num_pages)]
    return np.bincount(slots, minlength=num_pages).astype(np.int32)


def fork(table, lengths, refs, parents):
    """(table, lengths, refs) after the sequences continue their parents."""
    B, P = len(lengths), len(refs)
    new_t, new_l, new_r = np.full_like(table, -1), np.zeros_like(lengths), refs.copy()
    for b in range(B):
        for page in table[b]:
            if 0 <= page < P:
                new_r[page] -= 1
    for b in range(B):
        if 0 <= parents[b] < B:
            new_t[b], new_l[b] = table[parents[b]], lengths[parents[b]]
            for page in new_t[b]:
                if 0 <= page < P:
                    new_r[page] += 1
    return new_t, new_l, new_r


def reserve(pools, table, lengths, refs, n_new, page):
    """(pools, table, refs, short) once every sequence has pages of its own for its next n_new tokens.  pools: arrays
    [num_pages, heads, rows, ...], page / rows tokens to a row."""
    pools, table, refs = [x.copy() for x in pools], table.copy(), refs.copy()
    B, P, capacity = len(lengths), len(refs), table.shape[1] * page
    before_t, before_r = table.copy(), refs.copy()
    free = [i for i in range(P) if refs[i] <= 0]
    seen, short, source = {}, 0, [x.copy() for x in pools]
    for b in range(B):
        t = min(max(int(lengths[b]), 0), capacity)
        end = min(t + n_new, capacity)
        if t >= end:
            continue
        for s in range(t // page, (end - 1) // page + 1):
            old = int(before_t[b, s])
            shared = 0 <= old < P and before_r[old] > 1
            if 0 <= old < P:
                if not shared:
                    continue
                rank = seen.get(old, 0)
                seen[old] = rank + 1
                if rank >= before_r[old] - 1:
                    continue
                refs[old] -= 1
            elif s == t // page and t % page:  # tokens that found no page are lost
                short += 1
                continue
            if not free:
                table[b, s] = -1
                short += 1
                continue
            new = free.pop(0)
            table[b, s] = new
            refs[new] = 1
            if shared and s == t // page and t % page:
                for x, y in zip(source, pools):
                    rows = -(-(t % page) // (page // x.shape[2]))
                    y[new, :, :rows] = x[old, :, :rows]
    return pools, table, refs, short


def compact(pools, table, refs):
    """(pools, table, refs, used)."""
    P, used = len(refs), int((refs > 0).sum())
    to = np.arange(P)
    holes = [i for i in range(used) if refs[i] <= 0]
    late = [i for i in range(used, P) if refs[i] > 0]
    pools, refs = [x.copy() for x in pools], refs.copy()
    for a, b in zip(late, holes):
        to[a] = b
        for x in pools:
            x[b] = x[a]
        refs[b], refs[a] = refs[a], 0
    inside = (table >= 0) & (table < P)
    return pools, np.where(inside, to[np.where(inside, table, 0)], table).astype(np.int32), refs, used


def attend(q, k, v, scale):
    """q [heads, D] over k, v [n, D] in 64 bits: (O, LSE, sum of P |V|, largest sum of |q| |k|); no key: 0 and -inf."""
    if len(k) == 0:
        return np.zeros((len(q), v.shape[1])), np.full(len(q), -np.inf), np.zeros((len(q), v.shape[1])), 0.0
    with np.errstate(all="ignore"):
        s = scale * (q @ k.T)
        m = s.max(1, keepdims=True)
        p = np.exp(s - m)
        z = p.sum(1, keepdims=True)
        p = p / z
        size = abs(scale) * float((np.abs(q) @ np.abs(k).T).max())
        return p @ v, (m + np.log(z))[:, 0], p @ np.abs(v), size


def rows_of(x, table, b, tokens):
    """[tokens, Hkv, D] of sequence b: the given token indices of a padded (table None) or paged cache."""
    tokens = np.asarray(tokens, dtype=np.int64)
    if table is None:
        return x[b][:, tokens].swapaxes(0, 1)
    page = x.shape[2]
    return x[table[b, tokens // page], :, tokens % page]


def bounds(k, lo, hi, table, lengths, n_new, block):
    """(k_min, k_max) once the blocks of the last n_new tokens are refreshed."""
    lo, hi = lo.copy(), hi.copy()
    for b, n in enumerate(lengths):
        n = int(n)
        if n_new <= 0 or n <= 0:
            continue
        for j in range(max(n - n_new, 0) // block, -(-n // block)):
            tokens = np.arange(j * block, min((j + 1) * block, n))
            if table is not None:
                page = k.shape[2]
                slot, at = int(table[b, j * block // page]), j * block % page // block
                if not 0 <= slot < len(k):
                    continue
                rows = k[slot][:, j * block % page:][:, :len(tokens)]
            else:
                slot, at, rows = b, j, k[b][:, tokens]
            nan = np.isnan(rows)
            lo[slot, :, at] = np.where(nan, np.inf, rows).min(1)
            hi[slot, :, at] = np.where(nan, -np.inf, rows).max(1)
    return lo, hi


def select(q, lo, hi, table, lengths, keep, recent, block, sign=1.0):
    """[B, Hkv, keep / block] block indices.  q [B, Hq, D], bounds in 64 bits."""
    B, hq, d = q.shape
    h = lo.shape[1]
    keep, recent = keep // block, recent // block
    out = np.full((B, h, keep), -1, dtype=np.int32)
    for b in range(B):
        blocks = -(-int(lengths[b]) // block)
        for i in range(h):
            if blocks <= keep:
                out[b, i, :blocks] = np.arange(blocks)
                continue
            cand = blocks - recent
            if table is None:
                l, u = lo[b, i, :cand], hi[b, i, :cand]
            else:
                per = lo.shape[2]
                j = np.arange(cand)
                l, u = lo[table[b, j // per], i, j % per], hi[table[b, j // per], i, j % per]
            best = np.full(cand, -np.inf)
            for row in sign * q[b, i * (hq // h):(i + 1) * (hq // h)]:
                with np.errstate(all="ignore"):
                    s = (row * np.where(row > 0, u, l)).sum(1)
                best = np.fmax(best, s)
            best = best.astype(np.float32)
            best = np.where(np.isnan(best), -np.inf, best)
            order = np.argsort(-best, kind="stable")[:keep - recent]
            out[b, i] = np.concatenate([np.sort(order), np.arange(cand, blocks)])
    return out
