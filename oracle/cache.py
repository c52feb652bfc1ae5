"""fp64 NumPy restatement of the 8-bit KV cache and of eviction by attention weight (include/dtattn.h).

No counterpart in the reference (its Llama port keeps no KV cache, python/dtorch/test/modules/llama.py:126-156), so
these are pinned by their definitions alone: plain loops, one block, head or row after another.
"""
from __future__ import annotations

import numpy as np

from .sdpa import e4m3fn_decode, e4m3fn_encode


def block_scale(amax: float) -> float:
    """The smallest power of two s >= 2^-126 with amax <= 448 s, for a block that has an amax (1 for amax = 0)."""
    if amax == 0:
        return 1.0
    k = -126
    while amax > 448.0 * 2.0 ** k:
        k += 1
    return 2.0 ** k


def _encode(x: np.ndarray, s: float) -> np.ndarray:
    bad = ~np.isfinite(x)
    codes = e4m3fn_encode((np.where(bad, 0.0, x) / s).astype(np.float32))
    return np.where(bad, np.uint8(0x7F), codes)


def append_fp8(codes, scale, table, lengths, new, block):
    """One of K and V, in place: codes uint8 [slots, H, rows, D], scale [slots, H, rows / block], new float64
    [B, H, n, D]; table [B, max_pages] or None.  Does not advance lengths."""
    slots, heads, rows, _ = codes.shape
    capacity = rows * table.shape[1] if table is not None else rows
    for b in range(new.shape[0]):
        start = max(int(lengths[b]), 0)
        end = min(start + new.shape[2], capacity)
        t = start
        while t < end:
            t0 = t // block * block
            stop = min(end, t0 + block)
            slot, r0 = (int(table[b, t0 // rows]), t0 % rows) if table is not None else (b, t0)
            if 0 <= slot < slots:
                for h in range(heads):
                    x = new[b, h, t - start:stop - start]
                    fin = np.abs(x[np.isfinite(x)])
                    amax = float(fin.max(initial=0.0))
                    s = block_scale(amax) if amax > 0 else 2.0 ** -126  # no value to hold: no scale is too small
                    if t > t0:
                        old = float(scale[slot, h, r0 // block])
                        s = s if np.isnan(old) else max(s, old)
                        if s != old:
                            was = codes[slot, h, r0:r0 + t - t0]
                            val = e4m3fn_decode(was)
                            bad = np.isnan(val)
                            again = e4m3fn_encode((np.where(bad, 0.0, val) * (old / s)).astype(np.float32))
                            codes[slot, h, r0:r0 + t - t0] = np.where(bad, was, again)
                    codes[slot, h, r0 + t - t0:r0 + stop - t0] = _encode(x, s)
                    scale[slot, h, r0 // block] = s
            t = stop


def values(codes, scale, table=None, b=None, n=None):
    """float64 values of a cache's codes, or [H, n, D] of sequence b's first n tokens."""
    if b is None:
        return e4m3fn_decode(codes) * np.repeat(np.asarray(scale, dtype=np.float64), codes.shape[2] // scale.shape[2], 2)[..., None]
    rows, block = codes.shape[2], codes.shape[2] // scale.shape[2]
    t = np.arange(n)
    slot = np.clip(table[b, t // rows], 0, codes.shape[0] - 1) if table is not None else np.full(n, b)
    r = t % rows if table is not None else t
    x = e4m3fn_decode(codes[slot, :, r]) * np.asarray(scale, dtype=np.float64)[slot, :, r // block][..., None]  # [n, H, D]
    return x.transpose(1, 0, 2)


def attend(q, k, v, scale):
    """One kv head: q [G, D], k and v [n, D] -> (O, LSE, A) with A = softmax |V|, what relative errors of P are relative to."""
    with np.errstate(invalid="ignore"):
        s = q @ k.T * scale
        m = s.max(-1, keepdims=True)
        p = np.exp(s - m)
        z = p.sum(-1, keepdims=True)
        return p @ v / z, (m + np.log(z))[:, 0], p @ np.abs(v) / z


def decode_fp8(q, kc, vc, ks, vs, lengths, table=None, scale=None):
    """q [B, Hq, D] -> (O, LSE, A, M): M [B, Hq] bounds sum_d |q_d k_d| * |scale| over the keys."""
    B, hq, d = q.shape
    hkv = kc.shape[1]
    g = hq // hkv
    scale = d ** -0.5 if scale is None else scale
    o, a = np.zeros((B, hq, d)), np.zeros((B, hq, d))
    lse, mag = np.full((B, hq), -np.inf), np.zeros((B, hq))
    cap = kc.shape[2] * (table.shape[1] if table is not None else 1)
    for b in range(B):
        n = min(max(int(lengths[b]), 0), cap)
        if n == 0:
            continue
        k, v = values(kc, ks, table, b, n), values(vc, vs, table, b, n)
        for h in range(hkv):
            r = slice(h * g, (h + 1) * g)
            o[b, r], lse[b, r], a[b, r] = attend(q[b, r], k[h], v[h], scale)
            mag[b, r] = (np.abs(q[b, r]) @ np.abs(k[h]).T).max(-1) * abs(scale)
    return o, lse, a, mag


def attention_weights(weights, q, k, lse, lengths=None, causal=False, q_offset=0, scale=None):
    """In place: weights [B, Hkv, S], q [B, Hq, L, D], k [B, Hkv, S, D] values, lse [B, Hq, L]."""
    B, hq, L, d = q.shape
    hkv, S = k.shape[1], k.shape[2]
    scale = d ** -0.5 if scale is None else scale
    for b in range(B):
        n = S if lengths is None else min(max(int(lengths[b]), 0), S)
        for h in range(hq):
            hk = h // (hq // hkv)
            for i in range(L):
                if lse[b, h, i] == -np.inf or (causal and lengths is not None and i + q_offset >= n):
                    continue
                top = min(n, max(i + q_offset + 1, 0)) if causal else n
                weights[b, hk, :top] += np.exp(k[b, hk, :top] @ q[b, h, i] * scale - lse[b, h, i])


def evict(arrays, scales, weights, lengths, keep, recent, block, scale_block=1):
    """In place: arrays of [B, H, S, ...], scales of [B, H, S / scale_block], weights float32 [B, H, S]; returns kept."""
    B, H, S = weights.shape
    kb, rb = keep // block, recent // block
    kept = np.full((B, H, kb), -1, dtype=np.int32)
    for b in range(B):
        n = min(max(int(lengths[b]), 0), S)
        blocks = -(-n // block)
        if blocks <= kb:
            kept[b, :, :blocks] = np.arange(blocks)
            continue
        for h in range(H):
            cand = blocks - rb
            with np.errstate(invalid="ignore"):
                w = weights[b, h, :cand * block].astype(np.float64).reshape(cand, block).sum(1).astype(np.float32)
            w = np.where(np.isnan(w), -np.inf, w)
            best = sorted(range(cand), key=lambda i: (-w[i], i))[:kb - rb]
            chosen = sorted(best) + list(range(cand, blocks))
            kept[b, h] = chosen
            at = np.concatenate([np.arange(i * block, min((i + 1) * block, n)) for i in chosen])
            for x in arrays:
                x[b, h, :len(at)] = x[b, h, at].copy()
            weights[b, h, :len(at)] = weights[b, h, at].copy()
            weights[b, h, len(at):n] = 0
            for s in scales:
                per = block // scale_block
                src = np.concatenate([np.arange(i * per, min((i + 1) * per, -(-n // scale_block))) for i in chosen])
                s[b, h, :len(src)] = s[b, h, src].copy()
        lengths[b] = keep - block + n - (blocks - 1) * block
    return kept
