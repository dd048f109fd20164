"""GPU tier of the MX KV cache (kv_append_mx, kv_read_mx, decode_paged_mx)
against its restatement in 64 bits (oracle/mx.py).

Writer and reader have one rounding each, so the bar is equality: of every byte
of both pools, slots that the call must not touch among them, and of every row
read. The decode is held to a bound that follows from its roundings
(oracle.mx.decode_mx).
"""
import numpy as np
import pytest
import torch

from oracle import mx

pytestmark = pytest.mark.gpu

FORMS = [(64, 4, 4), (64, 8, 8), (64, 8, 4), (64, 4, 8), (128, 4, 4), (128, 8, 8), (128, 8, 4), (128, 4, 8)]
TYPES = {False: torch.float16, True: torch.bfloat16}


def _rows(rng, shape, bf16, spread=1.5):
    """Rows whose blocks and channels differ in size, as bit patterns."""
    x = rng.standard_normal(shape) * np.exp(spread * rng.standard_normal((*shape[:-1], 1)))
    return mx.from_f64(x * np.exp(0.7 * rng.standard_normal(shape[-1])), bf16)


def _pool(rng, pages, H, D, bits, is_v, bf16, spread=1.0):
    codes, scales = mx.quantize(_rows(rng, (pages, H, 16, D), bf16, spread), bits, bf16)
    return mx.pack_pages(codes, scales, bits, is_v)


def _to(dev, *xs):
    return [torch.from_numpy(np.ascontiguousarray(x)).to(dev) for x in xs]


def _rows_to(dev, x16, bf16):
    return torch.from_numpy(np.ascontiguousarray(x16).view(np.int16)).to(dev).view(TYPES[bf16])


def _bits(t):
    return t.cpu().view(torch.int16).numpy().view(np.uint16)


def _append(fa, dev, kp, vp, table, start, k, v, bf16, lens=None):
    tkp, tvp, tt, ts = _to(dev, kp, vp, table, start)
    tl = None if lens is None else _to(dev, lens)[0]
    bad = fa.kv_append_mx(_rows_to(dev, k, bf16), _rows_to(dev, v, bf16), tkp, tvp, tt, ts, tl)
    return tkp.cpu().numpy(), tvp.cpu().numpy(), bad.cpu().numpy()


def _same(got, want, tag):
    for g, w, name in zip(got, want, ("k_pool", "v_pool", "bad")):
        assert np.array_equal(g, w), f"{tag}: {name} differs in {(g != w).sum()} places"


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("D,kb,vb", FORMS)
@pytest.mark.parametrize("B,H,T", [(1, 1, 1), (3, 2, 2), (2, 3, 37), (3, 1, 130)])
def test_append_matches_oracle(fa, dev, B, H, T, D, kb, vb, bf16):
    rng = np.random.default_rng(B * 100 + T + D + kb)
    maxp = (T + 70) // 16 + 2
    P = B * maxp + 3
    table = rng.permutation(P).astype(np.int32)[:B * maxp].reshape(B, maxp)
    kp = rng.integers(0, 256, (P, H, mx.page_bytes(D, kb))).astype(np.uint8)   # slots not covered keep theirs
    vp = rng.integers(0, 256, (P, H, mx.page_bytes(D, vb))).astype(np.uint8)
    k, v = _rows(rng, (B, H, T, D), bf16), _rows(rng, (B, H, T, D), bf16)
    start = rng.integers(0, 60, B).astype(np.int32)
    start[0] = 15   # the first token is a page's last slot
    for lens in (None, rng.integers(-2, T + 3, B).astype(np.int32)):
        want = mx.append_mx(kp, vp, table, start, k, v, kb, vb, bf16, lens)
        _same(_append(fa, dev, kp, vp, table, start, k, v, bf16, lens), want, f"lens {lens}")


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("D,kb,vb", [(64, 4, 8), (128, 8, 4)])
def test_append_of_every_value(fa, dev, D, kb, vb, bf16):
    """All 65536 bit patterns, NaN, infinities, subnormals and both zeros among them, in blocks of
    like size and shuffled, so that every scale and both of its limits come up."""
    x = np.arange(65536, dtype=np.uint32).astype(np.uint16)
    rng = np.random.default_rng(5)
    x = np.concatenate([x, rng.permutation(x), rng.permutation(x[np.isfinite(mx.to_f64(x, bf16))])[:60000 // D * D]])
    x = x.reshape(1, 1, -1, D)
    T = x.shape[2]
    P = -(-T // 16)
    table = rng.permutation(P).astype(np.int32)[None]
    kp, vp = (np.zeros((P, 1, mx.page_bytes(D, b)), np.uint8) for b in (kb, vb))
    start = np.zeros(1, np.int32)
    want = mx.append_mx(kp, vp, table, start, x, x, kb, vb, bf16)
    got = _append(fa, dev, kp, vp, table, start, x, x, bf16)
    _same(got, want, "every value")
    k, v, bad = fa.kv_read_mx(*_to(dev, got[0], got[1], table, start), T, dtype=TYPES[bf16])
    wk, wv, _ = mx.read_mx(want[0], want[1], table, start, T, D, kb, vb)
    for g, w in ((k, wk), (v, wv)):
        g = g.double().cpu().numpy()
        assert ((g == w) | (np.isnan(g) & np.isnan(w))).all()


@pytest.mark.parametrize("D,kb,vb", [(64, 4, 4), (128, 8, 4)])
def test_append_bad_pages_and_positions(fa, dev, D, kb, vb):
    B, H, T, maxp, P = 6, 2, 40, 5, 40
    rng = np.random.default_rng(9)
    table = rng.permutation(P).astype(np.int32)[:B * maxp].reshape(B, maxp).copy()
    kp, vp = (rng.integers(0, 256, (P, H, mx.page_bytes(D, b))).astype(np.uint8) for b in (kb, vb))
    k, v = _rows(rng, (B, H, T, D), False), _rows(rng, (B, H, T, D), False)
    start = np.array([10, 0, maxp * 16 - 7, -2, -100, 2147483640], np.int32)
    table[0, 1], table[1, 0] = -5, P
    want = mx.append_mx(kp, vp, table, start, k, v, kb, vb, False)
    assert want[2].tolist() == [1] * 6
    _same(_append(fa, dev, kp, vp, table, start, k, v, False), want, "invalid")
    tkp, tvp, tt, ts = _to(dev, want[0], want[1], table, start)
    got = fa.kv_read_mx(tkp, tvp, tt, ts, T)
    wk, wv, bad = mx.read_mx(want[0], want[1], table, start, T, D, kb, vb)
    assert np.array_equal(got[2].cpu().numpy(), bad)
    for g, w in zip(got[:2], (wk, wv)):
        g, w = _bits(g), mx.from_f64(w, False)
        ok = (g == w) | (((g & 0x7fff) > 0x7c00) & ((w & 0x7fff) > 0x7c00))   # NaN for NaN
        assert ok.all()


def test_flags_over_stale_memory_and_no_tokens(fa, dev):
    B, H, D, P = 3, 2, 64, 30
    kp, vp = fa.kv_pools_mx(P, H, D, 4, 8, device=dev)
    table = torch.arange(P, dtype=torch.int32, device=dev).reshape(B, -1).contiguous()
    start = torch.tensor([0, 16 * 10, -1], dtype=torch.int32, device=dev)
    for T in (0, 3):
        x = torch.randn(B, H, T, D, device=dev, dtype=torch.half)
        stale = [torch.full((B,), 7, dtype=torch.int32, device=dev) for _ in range(4)]
        del stale   # the caching allocator hands one of these blocks out next
        assert fa.kv_append_mx(x, x, kp, vp, table, start).tolist() == [0, int(T > 0), int(T > 0)]
        k, v, bad = fa.kv_read_mx(kp, vp, table, start, T)
        assert bad.tolist() == [0, int(T > 0), int(T > 0)] and k.shape == v.shape == (B, H, T, D)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("D,kb,vb", FORMS)
def test_read_matches_oracle(fa, dev, D, kb, vb, bf16):
    """Any bytes: every code, and scales from below the type's range to above it (bf16: from 2^-97 up)."""
    B, H, T, maxp, P = 3, 2, 75, 8, 26
    rng = np.random.default_rng(D + kb + vb)
    lo, hi = (30, 256) if bf16 else (80, 160)
    pools = []
    for bits, is_v in ((kb, False), (vb, True)):
        codes = rng.integers(0, 16 if bits == 4 else 256, (P, H, 16, D)).astype(np.uint8)
        scales = rng.integers(lo, hi, (P, H, 16, D // 32)).astype(np.uint8)
        pools.append(mx.pack_pages(codes, scales, bits, is_v))
    table = rng.permutation(P).astype(np.int32)[:B * maxp].reshape(B, maxp)
    start = np.array([0, 13, 31], np.int32)
    for lens in (None, np.array([1, T + 9, 16], np.int32), np.array([0, -4, T], np.int32)):
        tl = None if lens is None else _to(dev, lens)[0]
        k, v, bad = fa.kv_read_mx(*_to(dev, *pools, table, start), T, tl, dtype=TYPES[bf16])
        wk, wv, wb = mx.read_mx(*pools, table, start, T, D, kb, vb, lens)
        assert not bad.any() and not wb.any()
        inf = 0x7f80 if bf16 else 0x7c00
        for g, w, name in ((k, wk, "k"), (v, wv, "v")):
            g, w = _bits(g), mx.from_f64(w, bf16)
            same = (g == w) | (((g & 0x7fff) > inf) & ((w & 0x7fff) > inf))
            assert same.all(), f"{name}: {(~same).sum()} differ"


@pytest.mark.parametrize("D,kb,vb,bf16", [(128, 4, 8, False), (64, 8, 4, True)])
def test_read_of_many_rows(fa, dev, D, kb, vb, bf16):
    """Rows of more than 100 MB, which are written past the caches: equal to the same rows read in
    short runs, ragged lengths, an invalid page and starts inside pages included."""
    B, H, T, P = 3, 5, 14000 * 128 // D, 4000
    g = torch.Generator(device=dev).manual_seed(D)
    kp, vp = (torch.randint(0, 255, (P, H, mx.page_bytes(D, b)), generator=g, device=dev, dtype=torch.uint8)
              for b in (kb, vb))
    table = torch.randint(0, P, (B, T // 16 + 2), generator=g, device=dev, dtype=torch.int32)
    table[1, 9] = -1
    start = torch.tensor([0, 7, 15], dtype=torch.int32, device=dev)
    lens = torch.tensor([T, T - 1, 100], dtype=torch.int32, device=dev)
    k, v, bad = fa.kv_read_mx(kp, vp, table, start, T, lens, dtype=TYPES[bf16])
    assert 2 * k.numel() * 2 >= 100 << 20 and bad.tolist() == [0, 1, 0]
    n = 3001
    for t in range(0, T, n):
        m = min(n, T - t)
        ks, vs, _ = fa.kv_read_mx(kp, vp, table, start + t, m, (lens - t).clamp(min=0), dtype=TYPES[bf16])
        for whole, part in ((k, ks), (v, vs)):
            assert torch.equal(whole[:, :, t:t + m].contiguous().view(torch.int16), part.view(torch.int16))


def _decode_case(seed, ctx, H, Hkv, D, kb, vb, bf16, poison=True, extra=0):
    """Pools, table and queries; slots past the contexts and unused pages hold NaN."""
    rng = np.random.default_rng(seed)
    need = [-(-c // 16) for c in ctx]
    P = sum(need) + 2
    perm = rng.permutation(P).astype(np.int32)
    table = np.full((len(ctx), max(max(need), 1) + extra), -1, np.int32)   # past a context: not looked at
    kp, vp = _pool(rng, P, Hkv, D, kb, False, bf16), _pool(rng, P, Hkv, D, vb, True, bf16)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
        if poison and ctx[b] % 16:
            for pool, bits, is_v in ((kp, kb, False), (vp, vb, True)):
                co, so = mx.code_offsets(D, bits, is_v), mx.scale_offsets(D, bits, is_v)
                for t in range(ctx[b] % 16, 16):
                    pool[table[b, n - 1]][:, co[t]] = 0x7f
                    pool[table[b, n - 1]][:, so[t]] = 255
    if poison:
        kp[perm[at:]] = 255
        vp[perm[at:]] = 255
    q = mx.from_f64(rng.standard_normal((len(ctx), H, D)), bf16)
    return q, kp, vp, table, np.asarray(ctx, np.int32)


def _check_decode(O, L, want, tag):
    Ow, Lw, tO, tL = want
    O, L = O.double().cpu().numpy(), L.double().cpu().numpy()
    empty = np.isneginf(Lw)
    assert np.array_equal(np.isneginf(L), empty) and (O[empty] == 0).all(), tag
    eo = np.abs(O - Ow) / np.maximum(tO, 1e-300)
    assert (np.abs(O - Ow) <= tO).all(), f"{tag}: O off by {np.nanmax(eo):.2f} of its bound"
    el = np.abs(L[~empty] - Lw[~empty])
    assert (el <= tL[~empty]).all(), f"{tag}: L off by {(el / tL[~empty]).max():.2f} of its bound"


def _decode(fa, dev, case, kb, vb, bf16, tag):
    q, kp, vp, table, ctx = case
    print(f"[mx decode] {tag}: q {q.shape} ctx {ctx[:8]} K{kb} V{vb} bf16 {bf16}", flush=True)
    tkp, tvp, tt, tc = _to(dev, kp, vp, table, ctx)
    tq = _rows_to(dev, q, bf16)
    O, L = fa.decode_paged_mx(tq, tkp, tvp, tt, tc)
    _check_decode(O, L, mx.decode_mx(q, kp, vp, table, ctx, kb, vb, bf16), tag)
    O2, L2 = fa.decode_paged_mx(tq, tkp, tvp, tt, tc)
    assert torch.equal(O, O2) and torch.equal(L, L2), f"{tag}: two calls differ"


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("D,kb,vb", FORMS)
@pytest.mark.parametrize("H,Hkv,ctx", [
    (1, 1, [1]),
    (4, 4, [0, 1, 15, 16, 17]),
    (8, 2, [63, 64, 65, 250, 256, 257, 0]),
    (6, 2, [1030]),
])
def test_decode_matches_oracle(fa, dev, H, Hkv, ctx, D, kb, vb, bf16):
    _decode(fa, dev, _decode_case(H + D + kb, ctx, H, Hkv, D, kb, vb, bf16), kb, vb, bf16, f"H{H}/{Hkv}")


@pytest.mark.parametrize("D,kb,vb,bf16,H,Hkv,ctx", [
    (128, 4, 4, False, 32, 1, [9001]),            # two groups of 16 heads, one KV head, many chunks
    (128, 4, 4, True, 40, 2, [3000, 5, 700]),     # groups of 20: 16 and 4
    (64, 8, 8, False, 16, 4, [12000, 1, 0, 33]),  # one long sequence among short ones
    (128, 8, 4, True, 8, 8, [4097, 4095, 16]),
    (64, 4, 4, True, 4, 1, [20000]),
    (64, 4, 4, False, 1, 1, [10350]),             # 647 pages in 40 chunks
    (128, 4, 8, False, 2, 1, [10300, 10000, 9990, 400]),
])
def test_decode_long_and_grouped(fa, dev, D, kb, vb, bf16, H, Hkv, ctx):
    _decode(fa, dev, _decode_case(len(ctx) + H, ctx, H, Hkv, D, kb, vb, bf16), kb, vb, bf16, "long")


@pytest.mark.parametrize("B", [64, 257, 1000])
def test_decode_many_sequences(fa, dev, B):
    """More sequences than a workgroup has threads, most of them short, empty ones among them."""
    rng = np.random.default_rng(B)
    ctx = rng.integers(0, 40, B)
    ctx[rng.integers(0, B, 5)] = rng.integers(600, 2500, 5)
    ctx[-1], ctx[0] = 1777, 0
    _decode(fa, dev, _decode_case(B, ctx.tolist(), 2, 1, 64, 4, 8, False), 4, 8, False, f"B{B}")


@pytest.mark.parametrize("B,long", [(70, [3000, 700]), (256, [9000, 2400, 2304]), (300, [131072, 2500, 4000]),
                                    (2100, [4000, 2400])])
def test_decode_of_planned_batches(fa, dev, B, long):
    """A few long sequences among many short, empty and invalid ones: chunks found by the waves
    (a lane for up to four sequences) and, past 256 sequences, planned by a launch."""
    rng = np.random.default_rng(B)
    ctx = rng.integers(0, 30, B)
    ctx[rng.choice(B, len(long), replace=False)] = long
    case = _decode_case(B, ctx.tolist(), 2, 1, 64, 4, 8, False)
    _decode(fa, dev, case, 4, 8, False, f"B{B}")
    q, kp, vp, table, c = case
    bad = int(np.argmin(c))   # one sequence's length is invalid: the others stay as they are
    O, L = fa.decode_paged_mx(_rows_to(dev, q, False), *_to(dev, kp, vp, table, c))
    c2 = c.copy()
    c2[bad] = -5
    O2, L2 = fa.decode_paged_mx(_rows_to(dev, q, False), *_to(dev, kp, vp, table, c2))
    keep = np.arange(B) != bad
    assert torch.isnan(O2[bad]).all() and torch.isnan(L2[bad]).all()
    assert torch.equal(O2[keep], O[keep]) and torch.equal(L2[keep], L[keep])


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("D,kb,vb", FORMS)
def test_decode_large_pools(fa, dev, D, kb, vb, bf16):
    """Pools of 64 MB and more are read with the non-temporal hint: the same pages spread over such
    pools give the same bits, in cut and uncut batches of four and of eight waves."""
    for H, Hkv, ctx in ((4, 2, [1500, 40, 0]), (2, 2, [300, 511]), (2, 1, [9])):
        q, kp, vp, table, c = _decode_case(D + H, ctx, H, Hkv, D, kb, vb, bf16)
        P = (64 << 20) // (Hkv * (kp.shape[2] + vp.shape[2])) + 100
        tkp, tvp, tt, tc = _to(dev, kp, vp, table, c)
        at = torch.from_numpy(np.random.default_rng(1).choice(P, kp.shape[0], replace=False)).to(dev)
        big = []
        for t in (tkp, tvp):
            x = torch.full((P, Hkv, t.shape[2]), 255, dtype=torch.uint8, device=dev)
            x[at] = t
            big.append(x)
        moved = torch.where(tt >= 0, at[tt.clamp(min=0).long()].int(), tt)
        tq = _rows_to(dev, q, bf16)
        O, L = fa.decode_paged_mx(tq, *big, moved, tc)
        Ow, Lw = fa.decode_paged_mx(tq, tkp, tvp, tt, tc)
        assert torch.equal(O, Ow) and torch.equal(L, Lw)
        _check_decode(O, L, mx.decode_mx(q, kp, vp, table, c, kb, vb, bf16), f"{ctx}")


@pytest.mark.parametrize("H,Hkv,B,pages", [
    (2, 2, 3, [32, 31, 1]), (2, 2, 3, [33, 24, 23]),          # the widest table of one launch, and the next
    (64, 64, 4, [143, 1, 90, 0]), (64, 64, 4, [144, 143, 1, 8]),   # and where the sequences fill the chip
])
def test_decode_at_the_limits_of_one_launch(fa, dev, H, Hkv, B, pages):
    ctx = [16 * p - (p > 1) * 3 for p in pages]
    _decode(fa, dev, _decode_case(H, ctx, H, Hkv, 64, 4, 4, False), 4, 4, False, f"{pages}")


def test_decode_wide_table(fa, dev):
    """A table far wider than the contexts: entries past them are not looked at."""
    _decode(fa, dev, _decode_case(3, [5, 70, 16], 4, 2, 128, 4, 4, False, extra=3000), 4, 4, False, "wide")


def test_decode_large_scores(fa, dev):
    """One token far above the rest, and scores so large that all others vanish."""
    D, n = 128, 500
    q, kp, vp, table, ctx = _decode_case(2, [n, n], 2, 1, D, 8, 8, False)
    for b, gain in ((0, 30.0), (1, 400.0)):
        rows = np.zeros((1, 1, 1, D))
        rows[..., :] = mx.to_f64(q[b, 0], False) * gain / np.sqrt(D)
        k16 = mx.from_f64(rows, False)
        kp, _, _ = mx.append_mx(kp, vp, table[b:b + 1], np.array([n // 3], np.int32), k16, k16, 8, 8, False)
    _decode(fa, dev, (q, kp, vp, table, ctx), 8, 8, False, "large scores")


def test_decode_bad_sequences_are_nan(fa, dev):
    D, H = 64, 4
    q, kp, vp, table, ctx = _decode_case(8, [40, 700, 100, 33, 16], H, 2, D, 4, 4, False)
    want = mx.decode_mx(q, kp, vp, table, ctx, 4, 4, False)
    table[0, 1] = kp.shape[0]
    table[1, 17] = -1
    ctx[2], ctx[3] = -1, table.shape[1] * 16 + 1
    O, L = fa.decode_paged_mx(_rows_to(dev, q, False), *_to(dev, kp, vp, table, ctx))
    assert torch.isnan(O[:4]).all() and torch.isnan(L[:4]).all()
    _check_decode(O[4:], L[4:], [x[4:] for x in want], "the sequence that is valid")


def test_decode_nan_block_reaches_its_heads_only(fa, dev):
    D = 128
    q, kp, vp, table, ctx = _decode_case(4, [50], 8, 4, D, 4, 4, True)
    want = mx.decode_mx(q, kp, vp, table, ctx, 4, 4, True)
    kp[table[0, 1], 2, mx.scale_offsets(D, 4, False)[3, 1]] = 255   # KV head 2: query heads 4 and 5
    O, L = fa.decode_paged_mx(_rows_to(dev, q, True), *_to(dev, kp, vp, table, ctx))
    assert torch.isnan(O[0, 4:6]).all() and torch.isnan(L[0, 4:6]).all()
    keep = [0, 1, 2, 3, 6, 7]
    _check_decode(O[:, keep], L[:, keep], [x[:, keep] for x in want], "other heads")


def _serve(fa, dev, tk, tv, tq, kp, vp, table, prompt, steps):
    """A prompt appended, then steps of append and decode: [O], [L]."""
    ctx = prompt.clone()
    bad = fa.kv_append_mx(tk[:, :, :int(prompt.max())].contiguous(), tv[:, :, :int(prompt.max())].contiguous(),
                          kp, vp, table, torch.zeros_like(prompt), prompt)
    assert not bad.any()
    out = []
    for i in range(steps):
        sel = ctx.long()[:, None, None, None].expand(-1, tk.shape[1], 1, tk.shape[3])
        fa.kv_append_mx(tk.gather(2, sel), tv.gather(2, sel), kp, vp, table, ctx)
        ctx = ctx + 1
        out.append(fa.decode_paged_mx(tq[i], kp, vp, table, ctx))
    return out


@pytest.mark.parametrize("D,kb,vb,bf16", [(128, 4, 4, True), (64, 8, 4, False)])
def test_serving_run(fa, dev, D, kb, vb, bf16):
    """Prompt, then 40 generated tokens, across page borders: every step against the oracle over the
    cache as the oracle's writer fills it; at the end the cache read back equals it."""
    B, H, Hkv, N = 3, 8, 2, 120
    rng = np.random.default_rng(D)
    k, v = _rows(rng, (B, Hkv, N, D), bf16, 0.5), _rows(rng, (B, Hkv, N, D), bf16, 0.5)
    steps, prompt = 40, np.array([1, 47, 80], np.int32)
    q = mx.from_f64(rng.standard_normal((steps, B, H, D)), bf16)
    maxp, P = 8, 30
    table = rng.permutation(P).astype(np.int32)[:B * maxp].reshape(B, maxp)
    kp, vp = fa.kv_pools_mx(P, Hkv, D, kb, vb, device=dev)
    tt, tp = _to(dev, table, prompt)
    out = _serve(fa, dev, _rows_to(dev, k, bf16), _rows_to(dev, v, bf16), _rows_to(dev, q, bf16), kp, vp, tt, tp, steps)
    wkp, wvp = np.zeros(tuple(kp.shape), np.uint8), np.zeros(tuple(vp.shape), np.uint8)
    wkp, wvp, _ = mx.append_mx(wkp, wvp, table, np.zeros(B, np.int32), k, v, kb, vb, bf16, prompt + steps)
    assert np.array_equal(kp.cpu().numpy(), wkp) and np.array_equal(vp.cpu().numpy(), wvp)
    for i in range(0, steps, 3):
        _check_decode(*out[i], mx.decode_mx(q[i], wkp, wvp, table, prompt + i + 1, kb, vb, bf16), f"step {i}")
    rk, rv, bad = fa.kv_read_mx(kp, vp, tt, torch.zeros_like(tp), N, tp + steps, dtype=TYPES[bf16])
    wk, wv, _ = mx.read_mx(wkp, wvp, table, np.zeros(B, np.int32), N, D, kb, vb, prompt + steps)
    assert not bad.any()
    assert np.array_equal(rk.double().cpu().numpy(), wk) and np.array_equal(rv.double().cpu().numpy(), wv)


def test_captured_step_replays(fa, dev):
    """Append and decode in one graph, replayed with new rows, lengths and eager calls of another
    batch in between; two graphs of different shapes replayed in turn."""
    rng = np.random.default_rng(11)
    B, H, Hkv, D = 4, 8, 2, 128
    graphs = []
    for ctx in ([300, 17, 900, 64], [2000, 3, 16, 129]):
        q, kp, vp, table, c = _decode_case(len(graphs), [n + 8 for n in ctx], H, Hkv, D, 4, 8, False, poison=False)
        k, v = _rows(rng, (8, B, Hkv, 1, D), False, 0.5), _rows(rng, (8, B, Hkv, 1, D), False, 0.5)
        st = dict(q=_rows_to(dev, q, False), table=table, host=(q, kp, vp), k=k, v=v, ctx=np.asarray(ctx, np.int32))
        st["kp"], st["vp"], st["tt"], st["tc"] = _to(dev, kp, vp, table, st["ctx"])
        st["tk"], st["tv"] = _rows_to(dev, k[0], False), _rows_to(dev, v[0], False)
        graphs.append(st)

    def step(s):
        bad = fa.kv_append_mx(s["tk"], s["tv"], s["kp"], s["vp"], s["tt"], s["tc"])
        s["tc"] += 1
        return (*fa.decode_paged_mx(s["q"], s["kp"], s["vp"], s["tt"], s["tc"]), bad)

    for s in graphs:   # first calls outside the capture; they take token 0
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(s)
        torch.cuda.current_stream().wait_stream(side)
        s["graph"] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(s["graph"]):
            s["out"] = step(s)
    for i in range(1, 6):
        for s in graphs:
            s["tk"].copy_(_rows_to(dev, s["k"][i], False))
            s["tv"].copy_(_rows_to(dev, s["v"][i], False))
            s["graph"].replay()
        e = graphs[i % 2]   # an eager call over the same memory between the replays
        eo, el = fa.decode_paged_mx(e["q"], e["kp"], e["vp"], e["tt"], e["tc"])
        torch.cuda.synchronize()
        assert torch.equal(eo, e["out"][0]) and torch.equal(el, e["out"][1])
        for s in graphs:
            q, kp, vp = s["host"]
            if i == 1:
                kp, vp, _ = mx.append_mx(kp, vp, s["table"], s["ctx"], s["k"][0], s["v"][0], 4, 8, False)
            kp, vp, _ = mx.append_mx(kp, vp, s["table"], s["ctx"] + i, s["k"][i], s["v"][i], 4, 8, False)
            s["host"] = (q, kp, vp)
            want = mx.decode_mx(q, kp, vp, s["table"], s["ctx"] + i + 1, 4, 8, False)
            _check_decode(s["out"][0], s["out"][1], want, f"replay {i}")
            assert not s["out"][2].any()


def test_other_streams(fa, dev):
    """Calls on two streams at once, each over its own batch, and the eager result of each."""
    cases = [_decode_case(20 + i, [1500 + 700 * i, 40], 8, 2, 64, 4, 4, False) for i in range(2)]
    args = [[_rows_to(dev, c[0], False), *_to(dev, *c[1:])] for c in cases]
    want = [fa.decode_paged_mx(*a) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(fa.decode_paged_mx(*args[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for O, L in got[i]:
            assert torch.equal(O, want[i][0]) and torch.equal(L, want[i][1])


def test_pool_beyond_4_gib(fa, dev):
    """Pages whose byte offsets pass 2^32, written, read and attended."""
    D, H, kb, vb, bf16 = 128, 8, 8, 4, False
    P = (1 << 32) // (H * mx.page_bytes(D, kb)) + 3000
    kp = torch.empty(P, H, mx.page_bytes(D, kb), dtype=torch.uint8, device=dev)
    vp = torch.empty(P, H, mx.page_bytes(D, vb), dtype=torch.uint8, device=dev)
    assert kp.numel() > 1 << 32
    rng = np.random.default_rng(6)
    n = 700
    table = (P - 1 - rng.permutation(2000)[:-(-n // 16)]).astype(np.int32)[None]
    k, v = _rows(rng, (1, H, n, D), bf16, 0.5), _rows(rng, (1, H, n, D), bf16, 0.5)
    tt, ts, tc = _to(dev, table, np.zeros(1, np.int32), np.array([n], np.int32))
    assert not fa.kv_append_mx(_rows_to(dev, k, bf16), _rows_to(dev, v, bf16), kp, vp, tt, ts).any()
    used = table[0]
    small = [mx.pack_pages(np.zeros((len(used), H, 16, D), np.uint8), np.zeros((len(used), H, 16, D // 32), np.uint8), b, z)
             for b, z in ((kb, False), (vb, True))]
    local = np.arange(len(used), dtype=np.int32)[None]
    wk, wv, _ = mx.append_mx(*small, local, np.zeros(1, np.int32), k, v, kb, vb, bf16)
    rk, rv, bad = fa.kv_read_mx(kp, vp, tt, ts, n)
    ok, ov, _ = mx.read_mx(wk, wv, local, np.zeros(1, np.int32), n, D, kb, vb)
    assert not bad.any() and np.array_equal(rk.double().cpu().numpy(), ok) and np.array_equal(rv.double().cpu().numpy(), ov)
    q = mx.from_f64(rng.standard_normal((1, 16, D)), bf16)
    O, L = fa.decode_paged_mx(_rows_to(dev, q, bf16), kp, vp, tt, tc)
    _check_decode(O, L, mx.decode_mx(q, wk, wv, local, np.array([n]), kb, vb, bf16), "beyond 4 GiB")


def test_agrees_with_16_bit_decode(fa, dev):
    """The 16-bit decode over the rows that kv_read_mx returns is the same attention."""
    B, H, Hkv, D, n = 2, 8, 2, 128, 1000
    q, kp, vp, table, ctx = _decode_case(31, [n, 333], H, Hkv, D, 4, 4, False)
    tq, (tkp, tvp, tt, tc) = _rows_to(dev, q, False), _to(dev, kp, vp, table, ctx)
    k, v, _ = fa.kv_read_mx(tkp, tvp, tt, torch.zeros_like(tc), n, tc)
    P = B * (-(-n // 16))
    kp16 = torch.zeros(P, Hkv, 16, D, dtype=torch.half, device=dev)
    vp16 = torch.zeros_like(kp16)
    t16 = torch.arange(P, dtype=torch.int32, device=dev).reshape(B, -1)
    fa.kv_append(k, v, kp16, vp16, t16, torch.zeros_like(tc))
    O, L = fa.decode_paged_mx(tq, tkp, tvp, tt, tc)
    O16, L16 = fa.decode_paged(tq, kp16, vp16, t16, tc)
    _check_decode(O, L, mx.decode_mx(q, kp, vp, table, ctx, 4, 4, False), "MX")
    # the 16-bit decode holds weights of at most 1 in fp16, in steps of 2^-24
    _check_decode(O16, L16, mx.decode_mx(q, kp, vp, table, ctx, 4, 4, False, p_top=1.0), "16 bits")


def test_rejects_bad_arguments(fa, dev):
    kp, vp = fa.kv_pools_mx(4, 2, 64, 4, 8, device=dev)
    x = torch.zeros(1, 2, 3, 64, dtype=torch.half, device=dev)
    t = torch.zeros(1, 2, dtype=torch.int32, device=dev)
    s = torch.zeros(1, dtype=torch.int32, device=dev)
    q = torch.zeros(1, 4, 64, dtype=torch.half, device=dev)
    k128, _ = fa.kv_pools_mx(4, 2, 128, 4, 4, device=dev)
    for call, match in [
        (lambda: fa.kv_append_mx(x.float(), x.float(), kp, vp, t, s), "float16"),
        (lambda: fa.kv_append_mx(x, x.bfloat16(), kp, vp, t, s), "float16"),
        (lambda: fa.kv_append_mx(x, x[:, :, :2], kp, vp, t, s), "same shape"),
        (lambda: fa.kv_append_mx(x.transpose(1, 2), x.transpose(1, 2), kp, vp, t, s), "contiguous"),
        (lambda: fa.kv_append_mx(x, x, kp.half(), vp, t, s), "uint8"),
        (lambda: fa.kv_append_mx(x, x, k128, vp, t, s), "same D"),
        (lambda: fa.kv_append_mx(x, x, kp[:, :, :500].contiguous(), vp, t, s), "page_bytes"),
        (lambda: fa.kv_append_mx(x, x, kp[:2], vp, t, s), "num_pages"),
        (lambda: fa.kv_append_mx(x, x, kp[:, :1], vp[:, :1], t, s), "contiguous"),
        (lambda: fa.kv_append_mx(x[:, :1].contiguous(), x[:, :1].contiguous(), kp, vp, t, s), "H and D"),
        (lambda: fa.kv_append_mx(x, x, kp, vp, t.long(), s), "int32"),
        (lambda: fa.kv_append_mx(x, x, kp, vp, t, s.long()), "int32"),
        (lambda: fa.kv_append_mx(x, x, kp, vp, t, s, s.long()), "int32"),
        (lambda: fa.kv_append_mx(x, x, kp, vp, t.cpu(), s), "CUDA"),
        (lambda: fa.kv_read_mx(kp, vp, t, s, -1), "num_tokens"),
        (lambda: fa.kv_read_mx(kp, vp, t, s.cpu(), 1), "CUDA"),
        (lambda: fa.kv_read_mx(kp, vp, t, torch.zeros(2, dtype=torch.int32, device=dev), 1), "start_pos"),
        (lambda: fa.decode_paged_mx(q.float(), kp, vp, t, s), "float16 or bfloat16"),
        (lambda: fa.decode_paged_mx(q[:, :3].contiguous(), kp, vp, t, s), "multiple"),
        (lambda: fa.decode_paged_mx(q[:, :, :32].contiguous(), kp, vp, t, s), "q's D"),
        (lambda: fa.decode_paged_mx(q.transpose(1, 2).contiguous().transpose(1, 2), kp, vp, t, s), "contiguous"),
        (lambda: fa.decode_paged_mx(q, kp, vp, t[:0], s), "batch size"),
        (lambda: fa.decode_paged_mx(q[:0], kp, vp, t[:0], s[:0]), "NULL"),
        (lambda: fa.decode_paged_mx(q, kp, vp, t[:, :0], s), "max_pages"),
        (lambda: fa.decode_paged_mx(q, kp[:0], vp[:0], t, s), "NULL|num_pages"),
    ]:
        with pytest.raises(RuntimeError, match=match):
            call()


def _huge_score_case(seed, ctx, D, kb, vb, bf16, b, qs):
    """Scores far beyond 2^24, as rows of one KV head per b and query heads per (b, a): every value of
    a K row is b but the first, b f with f of _STEPS; every value of a query is a but the first, which
    makes the products a b (D - 1) +- 8 f g with g the last place of the product in 32 bits, so that
    each is a number of 24 bits and any order of its sum is exact. Every seventh column of V is zero."""
    q, kp, vp, table, ctx = _decode_case(seed, ctx, len(qs) * len(b), len(b), D, kb, vb, bf16)
    rng = np.random.default_rng(seed)
    B, n = len(ctx), int(ctx.max())
    f = rng.choice(_STEPS, (B, 1, n))
    k = np.broadcast_to(np.asarray(b)[None, :, None, None], (B, len(b), n, D)).copy()
    k[..., 0] *= f
    v = mx.to_f64(_rows(rng, (B, len(b), n, D), bf16, 0.5), bf16)
    v[..., ::7] = 0
    k16, v16 = mx.from_f64(k, bf16), mx.from_f64(v, bf16)
    kp, vp, _ = mx.append_mx(kp, vp, table, np.zeros(B, np.int32), k16, v16, kb, vb, bf16, ctx)
    q = np.zeros((B, len(b) * len(qs), D))
    units = np.zeros(q.shape[1])   # of a head: its products are base + units f
    base = np.zeros(q.shape[1])
    for h in range(q.shape[1]):
        bh, a = b[h // len(qs)], qs[h % len(qs)]
        g = 2.0 ** (np.floor(np.log2(D * abs(a) * bh)) - 23)
        q[:, h], q[:, h, 0] = a, 8 * g / bh * (1 if h % 2 else -1)
        units[h], base[h] = q[0, h, 0] * bh, a * bh * (D - 1)
    s = base[None, :, None] + units[None, :, None] * f
    assert np.array_equal(s.astype(np.float32), s) and np.array_equal(mx.to_f64(mx.from_f64(q, bf16), bf16), q)
    return (mx.from_f64(q, bf16), kp, vp, table, ctx), s


_STEPS = np.array([0, 1, 2, 3, 4, 6, 8, 12]) / 8   # of b: values that both formats hold beside b


def _exact_score_result(s, case, kb, vb, bf16):
    """(O, L, tol_O, tol_L) where the products s are exact. With x_t = (s_t - max) / sqrt(D) log 2
    exponents, u = 2^-24: a weight 2^x is off by the scale's and the product's rounding (4 u |x|, of
    log 2), the argument's with the shift of 15 (u (15 + |x|)), and by 2 u of each exponential and u of
    each product where it is taken in parts (in its wave, up to eight new maxima, waves, chunks):
    u (4 |x| + 64) in all. Sums and roundings as in oracle.mx.decode_mx; L's scale, logarithm and
    products are 8 u of it."""
    q16, kp, vp, table, ctx = case
    B, H, D = q16.shape
    Hkv = kp.shape[1]
    u, half, least = 2.0 ** -24, 2.0 ** -8 if bf16 else 2.0 ** -11, 2.0 ** -134 if bf16 else 2.0 ** -25
    p_err, step = (2.0 ** -16, 2.0 ** -125) if bf16 else (2.0 ** -11, 2.0 ** -40)
    O, L = np.zeros((B, H, D)), np.full((B, H), -np.inf)
    tO, tL = np.zeros((B, H, D)), np.zeros((B, H))
    for b in range(B):
        n = int(ctx[b])
        if n == 0:
            continue
        for h in range(H):
            v = mx.page_values(vp[table[b, :-(-n // 16)], h // (H // Hkv)], D, vb, True).reshape(-1, D)[:n]
            sh = s[b, h, :n] if s.shape[0] > 1 else s[0, h, :n]
            m = sh.max()
            x = (sh - m) / np.sqrt(D) / np.log(2)
            e = np.exp2(x)
            p = e / e.sum()
            rel = p * u * (4 * np.abs(np.maximum(x, -200)) + 64)
            w = rel.sum() + (n / 16 + 64) * u
            O[b, h], L[b, h] = p @ v, m / np.sqrt(D) + np.log(e.sum())
            av = p @ np.abs(v)
            tO[b, h] = (rel @ np.abs(v) + w * np.abs(O[b, h]) + (n / 16 + 64) * u * av + p_err * av +
                        step * np.abs(v).sum(0) / e.sum() + half * np.abs(O[b, h]) + least)
            tL[b, h] = w + 8 * u * abs(L[b, h])
    return O, L, tO, tL


@pytest.mark.parametrize("ctx", [[1], [2, 17, 16, 500], [3000, 33, 1100], [20000]])
@pytest.mark.parametrize("D,kb,vb,bf16", [(128, 4, 8, False), (64, 8, 4, False), (128, 8, 4, True), (64, 4, 8, True)])
def test_decode_huge_scores(fa, dev, D, kb, vb, bf16, ctx):
    """Scores (in units of log 2) of 2^22 to 2^32 in fp16 and 2^14 to 2^90 in bf16, of both signs: the
    weights follow from the scores' differences, whatever the scores."""
    b = [1024.0, 2.0 ** 45 if bf16 else 16384.0]
    qs = [512.0, 1020.0, -2040.0, -2.0 ** 41, 1.5] if bf16 else [512.0, 1023.0, -2047.0, -1024.0, 16384.0]
    case, s = _huge_score_case(len(ctx) + D, ctx, D, kb, vb, bf16, b, qs)
    O, L = fa.decode_paged_mx(_rows_to(dev, case[0], bf16), *_to(dev, *case[1:]))
    _check_decode(O, L, _exact_score_result(s, case, kb, vb, bf16), f"{ctx}")
    assert (O.view(len(ctx), len(b) * len(qs), D)[..., ::7] == 0).all()


@pytest.mark.parametrize("D,vb,ctx", [(64, 4, 1), (64, 8, 2), (128, 8, 3), (128, 4, 40), (64, 8, 1500)])
def test_decode_weights_keep_32_bits_in_fp16(fa, dev, D, vb, ctx):
    """V of 1 and -1 in nearly equal weights: O is the small rest of a difference, which half a place
    of an 11-bit weight would show. With the scores' exponents below 2 (|q k| / sqrt(D) log 2), P's two
    terms (2^-22), 16 u of an exponential, D u of a score and the sums' (n / 16 + 64) u, twice each,
    O is off by that and by its own rounding (2^-11)."""
    rng = np.random.default_rng(D + ctx)
    H, n = 8, -(-ctx // 16) * 16
    kc, ks = rng.integers(0, 16, (n // 16, 1, 16, D)).astype(np.uint8), np.full((n // 16, 1, 16, D // 32), 127, np.uint8)
    vc = np.zeros((n // 16, 1, 16, D), np.uint8)
    one = 2 if vb == 4 else 0x38
    vc[:] = np.where(np.arange(n).reshape(-1, 1, 16, 1) % 2, one, one | (8 if vb == 4 else 128))
    kp, vp = mx.pack_pages(kc, ks, 4, False), mx.pack_pages(vc, ks, vb, True)
    q = mx.from_f64(rng.standard_normal((1, H, D)) * 0.1, False)
    table, c = np.arange(n // 16, dtype=np.int32)[None], np.array([ctx], np.int32)
    O, L = fa.decode_paged_mx(_rows_to(dev, q, False), *_to(dev, kp, vp, table, c))
    k = mx.page_values(kp[:, 0], D, 4, False).reshape(-1, D)[:ctx]
    s = k @ mx.to_f64(q[0], False).T / np.sqrt(D)
    mag = (np.abs(k) @ np.abs(mx.to_f64(q[0], False)).T).max() / np.sqrt(D)
    e = np.exp(s - s.max(0))
    v = mx.page_values(vp[:, 0], D, vb, True).reshape(-1, D)[:ctx, :1]
    want = (e * v).sum(0) / e.sum(0)
    u = 2.0 ** -24
    tol = 2.0 ** -22 + 2 * (16 + D * mag + 4 * np.abs(s).max() + n / 16 + 64) * u + 2.0 ** -11 * np.abs(want) + 2.0 ** -25
    err = np.abs(O[0].double().cpu().numpy() - want[:, None])
    assert (err <= tol[:, None]).all(), f"off by {(err / tol[:, None]).max():.2f} of the bound"


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bf16", [False, True])
def test_read_of_every_code_and_scale(fa, dev, bf16, D):
    """Every code under every scale, 0 and 255 among them: exact where the type has the value, to
    nearest even where it lies between two of the type's subnormals, infinite past its range."""
    rng = np.random.default_rng(D)
    blocks = {4: np.tile(np.arange(32) % 16, (256 * 8, 1)), 8: np.tile(np.arange(256).reshape(8, 32), (256, 1))}
    order = rng.permutation(256 * 8)   # neighbouring scales differ
    scales = np.repeat(np.arange(256), 8)[order].reshape(-1, 1, 16, D // 32).astype(np.uint8)
    P = len(scales)
    table = np.arange(P, dtype=np.int32)[None]
    for kb, vb in ((4, 8), (8, 4)):
        codes = {n: blocks[n][order].reshape(P, 1, 16, D).astype(np.uint8) for n in (4, 8)}
        kp, vp = mx.pack_pages(codes[kb], scales, kb, False), mx.pack_pages(codes[vb], scales, vb, True)
        k, v, bad = fa.kv_read_mx(*_to(dev, kp, vp, table, np.zeros(1, np.int32)), 16 * P, dtype=TYPES[bf16])
        assert not bad.any()
        inf = 0x7f80 if bf16 else 0x7c00
        for got, bits in ((k, kb), (v, vb)):
            w = mx.from_f64(mx.dequantize(codes[bits], scales, bits).reshape(1, 1, -1, D), bf16)
            g = _bits(got)
            same = (g == w) | (((g & 0x7fff) > inf) & ((w & 0x7fff) > inf))
            assert same.all(), f"{bits} bits: {(~same).sum()} differ"


@pytest.mark.parametrize("vb", [4, 8])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bf16", [False, True])
def test_decode_of_every_value_code_and_scale(fa, dev, bf16, D, vb):
    """One token of a page has all the weight, at each of a lane's four places; the other 15 hold zeros
    under other scales. O is that token's V row: every code under every scale whose values the type
    has, and scale 255. The weight is one up to 2^-22, the values have four bits: O is the value."""
    rng = np.random.default_rng(D + vb)
    per = 1 if vb == 4 else 8
    codes = np.tile((np.arange(32) % 16)[None] if vb == 4 else np.arange(256).reshape(8, 32), (256, 1))
    scales = np.repeat(np.arange(256), per)
    val = mx.dequantize(codes.astype(np.uint8), scales[:, None].astype(np.uint8), vb)
    back = mx.to_f64(mx.from_f64(val, bf16), bf16)
    has = np.where(scales == 255, True, ((back == val) | np.isnan(val)).all(1))
    codes, scales = codes[has], scales[has]
    nb = D // 32
    n = -(-len(scales) // nb) * nb
    pick = np.concatenate([rng.permutation(len(scales)), np.arange(n - len(scales))])
    rows, rs = codes[pick].reshape(-1, D), scales[pick].reshape(-1, nb)
    rows, rs = np.tile(rows, (4, 1)), np.tile(rs, (4, 1))
    B = len(rows)
    slot = 4 * rng.integers(0, 4, B) + np.repeat(np.arange(4), B // 4)
    vc, vs = np.zeros((B, 1, 16, D), np.uint8), rng.integers(0, 255, (B, 1, 16, nb)).astype(np.uint8)
    vc[np.arange(B), 0, slot], vs[np.arange(B), 0, slot] = rows, rs
    kc, ks = np.zeros((B, 1, 16, D), np.uint8), np.full((B, 1, 16, nb), 127, np.uint8)
    kc[np.arange(B), 0, slot, 0] = 7   # 6: its score is 6000 / sqrt(D) above the others'
    q = np.zeros((B, 1, D))
    q[..., 0] = 1000
    kp, vp = mx.pack_pages(kc, ks, 4, False), mx.pack_pages(vc, vs, vb, True)
    O, _ = fa.decode_paged_mx(_rows_to(dev, mx.from_f64(q, bf16), bf16),
                              *_to(dev, kp, vp, np.arange(B, dtype=np.int32)[:, None].copy(), np.full(B, 16, np.int32)))
    w = mx.dequantize(rows.astype(np.uint8), rs.astype(np.uint8), vb)
    g = mx.to_f64(_bits(O)[:, 0], bf16)
    same = (g == w) | (np.isnan(g) & np.isnan(w))
    i = np.argwhere(~same)
    assert same.all(), f"{len(i)} differ, of scales {sorted(set(rs[i[:, 0], i[:, 1] // 32]))[:9]}, {g[~same][:4]} {w[~same][:4]}"


@pytest.mark.parametrize("top", [118, -118])
@pytest.mark.parametrize("H,Hkv,ctx", [(4, 1, [20000]), (8, 8, [3000, 700, 40])])
def test_decode_joins_the_range_of_bf16(fa, dev, H, Hkv, ctx, top):
    """V of 2^118 and of 2^-118 in equal weights over many chunks: a chunk's sums stay in range, and so
    must the joined ones, which are as many times larger as there are tokens. O is V, of one bit, with
    equal weights that the sums leave (n / 16 + 64) u off, twice, below half a place of O."""
    D, kb, vb = 64, 4, 8
    q, kp, vp, table, c = _decode_case(3, ctx, H, Hkv, D, kb, vb, True)
    B, n = len(ctx), max(ctx)
    k = np.zeros((B, Hkv, n, D))
    v = np.broadcast_to(2.0 ** top * np.where(np.arange(D) % 3 == 0, -1, 1), k.shape)
    kp, vp, _ = mx.append_mx(kp, vp, table, np.zeros(B, np.int32), mx.from_f64(k, True), mx.from_f64(v, True), kb, vb, True, c)
    O, L = fa.decode_paged_mx(_rows_to(dev, q, True), *_to(dev, kp, vp, table, c))
    assert np.array_equal(mx.to_f64(_bits(O), True), np.broadcast_to(v[:1, :1, 0], O.shape))
    want = np.log(c.astype(np.float64))[:, None]
    assert (np.abs(L.double().cpu().numpy() - want) <= (n / 16 + 64) * 2.0 ** -24 + 2.0 ** -21 * want).all()
