"""Decode over a shared prefix, attention weights of cached tokens, and eviction by
them, restated in numpy, in 64 bits, a row at a time.

No counterpart in the reference, which has no KV cache.
"""
from __future__ import annotations

import numpy as np

PAGE = 16


def rows(pool, pages, n, h):
    """The first n rows of head h along a list of pages."""
    return pool[np.asarray(pages, np.int64), h].reshape(-1, pool.shape[-1])[:n]


def attend(q, k, v, half):
    """(o, lse, p, tol_o, tol_l, tol_p) of query rows q [G, D] over k, v [n, D], float64, for kernels that

    - add D products of a score in 32 bits: off by d = (D + 4) 2^-24 sum |q k| / sqrt(D), so a weight by a
      factor of 2 d (its own score and the sum's), by 2^-20 for the exponentials, the argument's scaling
      (|s| 2^-23) and the joins, and a term 2^-22 |s| of the largest score's size for the latter;
    - round weights relative to their largest to 16 bits for the product with V: half a step (`half`), or 2^-25
      of the largest below fp16's normal numbers;
    - round o to 16 bits: half a step, or 2^-25 below the normal numbers.
    """
    D = q.shape[-1]
    if len(k) == 0:
        z = np.zeros(q.shape)
        return z, np.full(len(q), -np.inf), np.zeros((len(q), 0)), z, np.zeros(len(q)), np.zeros((len(q), 0))
    s = q @ k.T / np.sqrt(D)
    m = s.max(1, keepdims=True)
    e = np.exp(s - m)
    z = e.sum(1, keepdims=True)
    p = e / z
    o, lse = p @ v, (m + np.log(z))[:, 0]
    d = (D + 4) * 2.0 ** -24 * (np.abs(q) @ np.abs(k).T).max(1) / np.sqrt(D)
    rel = 2 * d + 2.0 ** -20 + 2.0 ** -22 * np.abs(s).max(1)
    av = p @ np.abs(v)
    tol_o = (half + rel[:, None]) * av + 2.0 ** -25 * np.abs(v).sum(0) + half * np.abs(o) + 2.0 ** -25
    return o, lse, p, tol_o, rel + 2.0 ** -22 * np.abs(lse), p * rel[:, None] + 2.0 ** -30


def attend_exact(s, v, half, p_half):
    """attend() for products s [G, n] = q k that the kernels have exactly, whatever their size: what bounds the weights
    are the differences to the largest, x = (s - max) / sqrt(D) in units of log 2, not the scores. With u = 2^-24:

    - the scale is off by 3 u, its product with the difference and a sum with a constant by u each, an exponential by
      2 u, where a weight is taken in parts (in its wave, up to eight new maxima, waves, chunks, 32 lanes of a join) each
      of them and a product: u (5 |x| + 80) in all;
    - a sum of n weights, and of n products, in up to 16 parts: (n / 16 + 64) u;
    - P is off by p_half of itself, or 2^-25 of the largest below fp16's normal numbers; O by half of itself.
    """
    if s.shape[1] == 0:
        return attend(np.zeros((len(s), v.shape[-1])), v, v, half)
    D, u = v.shape[-1], 2.0 ** -24
    m = s.max(1, keepdims=True)
    x = (s - m) / np.sqrt(D) / np.log(2)
    e = np.exp2(x)
    z = e.sum(1, keepdims=True)
    p = e / z
    o, lse = p @ v, (m / np.sqrt(D) + np.log(z))[:, 0]
    rel = p * u * (5 * np.abs(np.maximum(x, -200)) + 80)
    adds = (s.shape[1] / 16 + 64) * u
    w = rel.sum(1, keepdims=True) + adds
    av = p @ np.abs(v)
    tol_o = rel @ np.abs(v) + (w + half) * np.abs(o) + (adds + p_half) * av + 2.0 ** -25 * (np.abs(v).sum(0) / z + 1)
    return o, lse, p, tol_o, w[:, 0] + 8 * u * np.abs(lse), rel + p * w + 2.0 ** -126


def decode_shared(q, k_pool, v_pool, prefix, prefix_len, table, ctx, half):
    """(o [B, H, D], lse [B, H], tol_o, tol_l)."""
    B, H, D = q.shape
    Hkv = k_pool.shape[1]
    G = H // Hkv
    o, lse, to, tl = np.zeros((B, H, D)), np.zeros((B, H)), np.zeros((B, H, D)), np.zeros((B, H))
    for h in range(Hkv):
        g = slice(h * G, (h + 1) * G)
        pre = [rows(x, prefix[:-(-prefix_len // PAGE)], prefix_len, h) for x in (k_pool, v_pool)]
        for b in range(B):
            own = [rows(x, table[b, :-(-ctx[b] // PAGE)], ctx[b], h) for x in (k_pool, v_pool)]
            k, v = (np.concatenate(x) for x in zip(pre, own))
            o[b, g], lse[b, g], _, to[b, g], tl[b, g], _ = attend(q[b, g], k, v, half)
    return o, lse, to, tl


def decode_weights(q, k_pool, v_pool, table, ctx, weights, half):
    """(o, lse, w, tol_o, tol_l, tol_w)."""
    B, H, D = q.shape
    Hkv = k_pool.shape[1]
    G = H // Hkv
    o, lse, to, tl = np.zeros((B, H, D)), np.zeros((B, H)), np.zeros((B, H, D)), np.zeros((B, H))
    w = weights.astype(np.float64)
    tw = np.zeros(w.shape)
    for b in range(B):
        n = ctx[b]
        for h in range(Hkv):
            g = slice(h * G, (h + 1) * G)
            k, v = (rows(x, table[b, :-(-n // PAGE)], n, h) for x in (k_pool, v_pool))
            o[b, g], lse[b, g], p, to[b, g], tl[b, g], tp = attend(q[b, g], k, v, half)
            w[b, h, :n] += p.sum(0)
            tw[b, h, :n] = tp.sum(0) + (G + 1) * 2.0 ** -24 * w[b, h, :n]   # the sum's roundings
    return o, lse, w, to, tl, tw


def evict(k_pool, v_pool, table, ctx, weights, new_table, keep, recent):
    """(k_pool, v_pool, kept, new_weights, new_lens, bad) after the call, by a plain sort."""
    k_pool, v_pool = k_pool.copy(), v_pool.copy()
    num_pages, Hkv = k_pool.shape[:2]
    B = len(ctx)
    kept = np.full((B, Hkv, keep), -1, np.int32)
    new_w = np.zeros((B, Hkv, PAGE * new_table.shape[1]), np.float32)
    lens, bad = np.zeros(B, np.int32), np.zeros(B, np.int32)
    for b in range(B):
        n = int(ctx[b])
        if n < 0 or n > PAGE * table.shape[1]:
            bad[b] = 1
            continue
        m = lens[b] = min(n, keep)
        r = min(recent, m)
        for h in range(Hkv):
            with np.errstate(invalid="ignore"):   # signalling NaNs
                w = weights[b, h, :n - r].astype(np.float64)
            order = sorted(range(n - r), key=lambda j: (-w[j] if w[j] == w[j] else np.inf, w[j] != w[j], j))
            stay = sorted(order[:m - r]) + list(range(n - r, n))
            kept[b, h, :m] = stay
            new_w[b, h, :m] = weights[b, h, stay]
            for j, old in enumerate(stay):
                src, dst = table[b, old // PAGE], new_table[b, j // PAGE]
                if not (0 <= src < num_pages and 0 <= dst < num_pages):
                    bad[b] = 1
                    continue
                for pool in (k_pool, v_pool):
                    pool[dst, h, j % PAGE] = pool[src, h, old % PAGE]
    return k_pool, v_pool, kept, new_w, lens, bad
