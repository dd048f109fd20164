"""The MX paged KV cache restated in numpy, in 64 bits: the formats, the pages'
bytes, the writer, the reader and the decode.

No counterpart in the reference, which has no KV cache: a format published by
the Open Compute Project (blocks of 32 values with a power-of-two scale in one
byte; values in E2M1 or E4M3), with this library's rule for the scale
(scale_codes) and its order of a page's bytes (code_offsets, scale_offsets).

Rows of 16-bit values are passed as their bit patterns (uint16) with bf16 to
tell their type: numpy has no bfloat16.
"""
from __future__ import annotations

import numpy as np

PAGE = 16
LIM = {4: 7.0, 8: 464.0}     # half a step past the format's largest, to which values up to there go
TOP = {(4, False): 140, (4, True): 252, (8, False): 134, (8, True): 246}   # largest scale code, by (bits, bf16)


def grid(bits: int) -> np.ndarray:
    """The format's values from 0 up; a value's index is its code."""
    if bits == 4:
        return np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
    v = [m * 2.0 ** -9 for m in range(8)]
    v += [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)]
    return np.array(v[:127])


def code_values(bits: int) -> np.ndarray:
    """Value of every code (E4M3 has a NaN of either sign)."""
    half = 8 if bits == 4 else 128
    g = np.full(half, np.nan)
    g[:len(grid(bits))] = grid(bits)
    return np.concatenate([g, -g])


def to_f64(bits16: np.ndarray, bf16: bool) -> np.ndarray:
    with np.errstate(invalid="ignore"):   # signalling NaNs
        if bf16:
            return (bits16.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
        return bits16.view(np.float16).astype(np.float64)


def from_f64(x: np.ndarray, bf16: bool) -> np.ndarray:
    """Bit patterns of x to nearest even; every NaN as the positive quiet one."""
    with np.errstate(over="ignore", invalid="ignore"):
        if not bf16:
            r = x.astype(np.float16).view(np.uint16)
            return np.where(np.isnan(x), np.uint16(0x7e00), r)
        f = x.astype(np.float32).view(np.uint32).astype(np.uint64)
        r = ((f + 0x7fff + ((f >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7fc0), r)


def scale_codes(amax: np.ndarray, bits: int, bf16: bool) -> np.ndarray:
    """Smallest s in [1, TOP] with amax <= LIM 2^(s - 127), or TOP."""
    edges = LIM[bits] * np.exp2(np.arange(1, TOP[bits, bf16]) - 127.0)
    return 1 + np.searchsorted(edges, amax, side="left")


def quantize(rows16: np.ndarray, bits: int, bf16: bool):
    """(codes uint8 [..., D], scales uint8 [..., D / 32]) of rows [..., D]."""
    x = to_f64(rows16, bf16)
    blocks = x.reshape(*x.shape[:-1], -1, 32)
    finite = np.isfinite(blocks).all(-1)
    blocks = np.where(finite[..., None], blocks, 0.0)
    s = scale_codes(np.abs(blocks).max(-1), bits, bf16)
    y = np.abs(blocks) / np.exp2(s - 127.0)[..., None]
    g = grid(bits)
    mid = (g[1:] + g[:-1]) / 2
    lo, hi = np.searchsorted(mid, y, side="left"), np.searchsorted(mid, y, side="right")
    idx = np.where(lo % 2 == 0, lo, hi)          # they differ on a tie: the even one
    neg = np.signbit(x.reshape(blocks.shape)) & finite[..., None]
    codes = idx + np.where(neg, 8 if bits == 4 else 128, 0)
    scales = np.where(finite, s, 255)
    return codes.reshape(x.shape).astype(np.uint8), scales.astype(np.uint8)


def dequantize(codes: np.ndarray, scales: np.ndarray, bits: int) -> np.ndarray:
    """float64 rows [..., D]."""
    unit = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return code_values(bits)[codes] * np.repeat(unit, 32, axis=-1)


def page_bytes(D: int, bits: int) -> int:
    return PAGE * D * bits // 8 + PAGE * D // 32


def code_offsets(D: int, bits: int, is_v: bool) -> np.ndarray:
    """[16, D bits / 8]: where byte j of row t lies in a page."""
    w = D * bits // 8
    out = np.zeros((PAGE, w), np.int64)
    for t in range(PAGE):
        for j in range(w):
            if not is_v:
                out[t, j] = t * w + j if w < 128 else 1024 * (j % 32 // 16) + 16 * (4 * t + j // 32) + j % 16
            else:
                c, r = divmod(j, w // 16)
                cell = 16 * (t // 4) + c
                out[t, j] = (cell * w // 4 + t % 4 * w // 16 + r if w < 128
                             else 1024 * (t % 4 // 2) + 16 * cell + 8 * (t % 2) + r)
    return out


def scale_offsets(D: int, bits: int, is_v: bool) -> np.ndarray:
    """[16, D / 32]: where the scale of block i of row t lies in a page."""
    t, i = np.arange(PAGE)[:, None], np.arange(D // 32)[None]
    return PAGE * D * bits // 8 + (16 * i + t if is_v else t * (D // 32) + i)


def _pack(codes: np.ndarray, bits: int) -> np.ndarray:
    return codes if bits == 8 else codes[..., 0::2] | (codes[..., 1::2] << 4)


def _unpack(data: np.ndarray, bits: int) -> np.ndarray:
    if bits == 8:
        return data
    return np.stack([data & 15, data >> 4], -1).reshape(*data.shape[:-1], -1)


def pack_pages(codes: np.ndarray, scales: np.ndarray, bits: int, is_v: bool) -> np.ndarray:
    """Codes [..., 16, D] and scales [..., 16, D / 32] as pages [..., page_bytes]."""
    D = codes.shape[-1]
    out = np.zeros((*codes.shape[:-2], page_bytes(D, bits)), np.uint8)
    out[..., code_offsets(D, bits, is_v).ravel()] = _pack(codes, bits).reshape(*codes.shape[:-2], -1)
    out[..., scale_offsets(D, bits, is_v).ravel()] = scales.reshape(*scales.shape[:-2], -1)
    return out


def unpack_pages(pages: np.ndarray, D: int, bits: int, is_v: bool):
    """(codes [..., 16, D], scales [..., 16, D / 32])."""
    lead = pages.shape[:-1]
    data = pages[..., code_offsets(D, bits, is_v).ravel()].reshape(*lead, PAGE, -1)
    scales = pages[..., scale_offsets(D, bits, is_v).ravel()].reshape(*lead, PAGE, D // 32)
    return _unpack(data, bits), scales


def page_values(pages: np.ndarray, D: int, bits: int, is_v: bool) -> np.ndarray:
    """float64 [..., 16, D]."""
    return dequantize(*unpack_pages(pages, D, bits, is_v), bits)


def _place(table, num_pages, b, pos):
    """(page id, slot) of a position, or None."""
    if pos < 0 or pos >= table.shape[1] * PAGE:
        return None
    pid = int(table[b, pos // PAGE])
    return (pid, pos % PAGE) if 0 <= pid < num_pages else None


def append_mx(k_pool, v_pool, table, start, k_new, v_new, k_bits, v_bits, bf16, lens=None):
    """(k_pool, v_pool, bad) after appending k_new, v_new (uint16 [B, H, T, D])."""
    k_pool, v_pool = k_pool.copy(), v_pool.copy()
    B, _, T, D = k_new.shape
    bad = np.zeros(B, np.int32)
    for pool, rows, bits, is_v in ((k_pool, k_new, k_bits, False), (v_pool, v_new, v_bits, True)):
        co, so = code_offsets(D, bits, is_v), scale_offsets(D, bits, is_v)
        codes, scales = quantize(rows, bits, bf16)
        data = _pack(codes, bits)
        for b in range(B):
            n = T if lens is None else min(max(int(lens[b]), 0), T)
            for t in range(n):
                at = _place(table, pool.shape[0], b, int(start[b]) + t)
                if at is None:
                    bad[b] = 1
                    continue
                pool[at[0]][:, co[at[1]]] = data[b, :, t]
                pool[at[0]][:, so[at[1]]] = scales[b, :, t]
    return k_pool, v_pool, bad


def read_mx(k_pool, v_pool, table, start, T, D, k_bits, v_bits, lens=None):
    """(k, v float64 [B, H, T, D], bad)."""
    B, H = table.shape[0], k_pool.shape[1]
    out, bad = [], np.zeros(B, np.int32)
    for pool, bits, is_v in ((k_pool, k_bits, False), (v_pool, v_bits, True)):
        x = np.zeros((B, H, T, D))
        for b in range(B):
            n = T if lens is None else min(max(int(lens[b]), 0), T)
            for t in range(n):
                at = _place(table, pool.shape[0], b, int(start[b]) + t)
                if at is None:
                    x[b, :, t], bad[b] = np.nan, 1
                else:
                    x[b, :, t] = page_values(pool[at[0]], D, bits, is_v)[:, at[1]]
        out.append(x)
    return out[0], out[1], bad


def decode_mx(q16, k_pool, v_pool, table, ctx, k_bits, v_bits, bf16, p_top=2.0 ** 15):
    """(O, L, tol_O, tol_L) in 64 bits, of valid sequences; q16 uint16 [B, H, D].

    tol_O and tol_L bound what a computation with exact 16-bit operands, 32-bit
    sums and P rounded to two terms of fp16 (22 bits) or of bf16 (16) may be off
    by (p_top = 1: to one fp16 term, 11 bits, as the 16-bit decode does), with
    u = 2^-24: the scores by D u sum |q k| / sqrt(D) (their sum)
    and 4 u |s| (scaling, the exponential's argument), which P and so each
    weight take twice (numerator and sum), 16 u of the exponential, and the two
    sums over n tokens by (n / 16 + 64) u each (a lane adds a sixteenth of a
    chunk's tokens, then waves and chunks join). A weight
    exp(s - m) is off by an absolute step besides: fp16 holds p_top (2^15) of it in
    steps of 2^-24, so half a step is 2^-40 of the largest weight (1); in bf16 what
    lies below the smallest normal 32-bit number, 2^-126, may vanish, of the
    weight's first term or of its second, 2^-125 in all. O is rounded once.
    """
    B, H, D = q16.shape
    Hkv = k_pool.shape[1]
    q = to_f64(q16, bf16)
    O, L = np.zeros((B, H, D)), np.full((B, H), -np.inf)
    tO, tL = np.zeros((B, H, D)), np.zeros((B, H))
    u, half = 2.0 ** -24, 2.0 ** -8 if bf16 else 2.0 ** -11
    p_err = 2.0 ** -16 if bf16 else 2.0 ** -11 if p_top == 1 else 2.0 ** -22
    step = 2.0 ** -125 if bf16 else 2.0 ** -25 / p_top
    least = 2.0 ** -134 if bf16 else 2.0 ** -25   # half the type's smallest step
    for b in range(B):
        n = int(ctx[b])
        if n == 0:
            continue
        pages = table[b, :-(-n // PAGE)]
        for hk in range(Hkv):
            k = page_values(k_pool[pages, hk], D, k_bits, False).reshape(-1, D)[:n]
            v = page_values(v_pool[pages, hk], D, v_bits, True).reshape(-1, D)[:n]
            for h in range(hk * (H // Hkv), (hk + 1) * (H // Hkv)):
                s = k @ q[b, h] / np.sqrt(D)
                m = s.max()
                e = np.exp(s - m)
                z = e.sum()
                p = e / z
                O[b, h], L[b, h] = p @ v, m + np.log(z)
                mag = (np.abs(k) @ np.abs(q[b, h])).max() / np.sqrt(D)
                ds = D * u * mag + 4 * u * np.abs(s).max()
                w = 2 * ds + 32 * u + 2 * (n / 16 + 64) * u
                av = p @ np.abs(v)
                tO[b, h] = av * (p_err + w) + step * np.abs(v).sum(0) / z + np.abs(O[b, h]) * half + least
                tL[b, h] = w + 4 * u * abs(L[b, h])
    return O, L, tO, tL
