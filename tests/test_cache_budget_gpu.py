"""GPU tier of the attention weights of cached tokens (decode_paged_weights) and of
the eviction by them (kv_evict) against their restatement in 64 bits
(oracle/cache.py, which derives the bounds). The eviction computes nothing but an
order, so its bar is equality."""
import math

import numpy as np
import pytest
import torch

from oracle import cache, rotary
from test_shared_gpu import (HALF, HUGE, TYPES, _case, _check, _climbing_scores, _coherent_roundings, _huge_scores, _i32, _one_term,
                             _want_exact)

pytestmark = pytest.mark.gpu


def _paged(dev, seed, B, H, Hkv, D, ctx, dtype, **kw):
    q, kp, vp, _, _, table, c = _case(dev, seed, B, H, Hkv, D, 0, ctx, dtype, **kw)
    g = torch.Generator(device=dev)
    g.manual_seed(seed + 1)
    w = torch.rand((B, Hkv, 16 * table.shape[1]), generator=g, device=dev) * 3
    return q, kp, vp, table, c, w


def _f64(t):
    return t.cpu().double().numpy()


def _check_weights(got, case, dtype, tag=""):
    q, kp, vp, table, ctx, w = case
    o, l, want, to, tl, tw = cache.decode_weights(_f64(q), _f64(kp), _f64(vp), table.cpu().numpy(), ctx.tolist(),
                                                  w.cpu().numpy(), HALF[dtype])
    _check(got[:2], (o, l, to, tl), dtype, tag)
    W = got[2]
    assert W.dtype == torch.float32 and W.shape == w.shape
    err = np.abs(_f64(W) - want)
    assert (err <= tw).all(), f"{tag} W: worst {np.nanmax(err / np.maximum(tw, 1e-300)):.2f} of the bound, {np.isnan(err).sum()} NaN"


CASES = [(1, 1, 1, 64, [1]), (2, 8, 2, 64, [0, 5]), (3, 4, 4, 128, [1, 16, 17]), (4, 8, 8, 64, [300, 0, 2, 64]),
         (2, 32, 8, 128, [33, 1700]), (3, 40, 2, 64, [100, 2500, 17]), (1, 128, 1, 128, [800]), (2, 36, 2, 128, [1023, 1025]),
         (20, 4, 2, 64, [13 * i for i in range(20)]), (1, 300, 1, 64, [1100]), (300, 4, 2, 64, [7 * i % 90 for i in range(300)]),
         (1500, 2, 1, 64, [i % 5 for i in range(1500)]), (1, 8, 1, 128, [9000]), (65, 2, 2, 128, [40] * 64 + [3000]),
         (3, 36, 4, 128, [512, 0, 497]), (2, 16, 1, 64, [255, 256]), (256, 2, 2, 128, [i % 300 for i in range(256)])]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("wide", [0, 40])   # short tables are walked in one launch, wide ones in chunks
@pytest.mark.parametrize("i", range(len(CASES)))
def test_weights_match_oracle(fa, dev, i, wide, dtype):
    B, H, Hkv, D, ctx = CASES[i]
    case = _paged(dev, i, B, H, Hkv, D, ctx, dtype, extra=i % 3 + wide)
    before = case[5].clone()
    got = fa.decode_paged_weights(*case)
    _check_weights(got, case, dtype, f"{CASES[i]}")
    assert torch.equal(case[5], before)
    again = fa.decode_paged_weights(*case)
    assert all(torch.equal(x, y) for x, y in zip(got, again))
    w = before.clone()
    inplace = fa.decode_paged_weights(*case[:5], w, inplace=True)
    assert inplace[2].data_ptr() == w.data_ptr() and all(torch.equal(x, y) for x, y in zip(got, inplace))


def test_weights_of_a_step_sum_to_the_heads(fa, dev):
    """From zeros every KV head's weights sum to the query heads that share it: each head's weights are off by the
    factor of oracle.cache.attend, here below 2e-4."""
    case = _paged(dev, 3, 3, 24, 4, 128, [500, 1, 3333], "bf16", poison=False)
    W = fa.decode_paged_weights(*case[:5], torch.zeros_like(case[5]))[2]
    assert (W.double().sum(-1) - 6).abs().max() < 6 * 2e-4
    assert (W[0, :, 500:] == 0).all() and (W[1, :, 1:] == 0).all()


def test_weights_large_scores(fa, dev):
    for amp in (8.0, 60.0):
        case = _paged(dev, 4, 3, 8, 2, 64, [700, 3, 1200], "fp16", amp=amp)
        _check_weights(fa.decode_paged_weights(*case), case, "fp16", f"amp {amp}")


@pytest.mark.parametrize("wide", [0, 40])
@pytest.mark.parametrize("D", [64, 128])
def test_weights_invalid(fa, dev, D, wide):
    """An invalid page or length: O, L and the weights up to the context, cut to the table, are NaN; the rest is kept."""
    ctx = [40, 300, 40, 64, 0]
    q, kp, vp, table, c, w = _paged(dev, 5, 5, 8, 2, D, ctx, "fp16", extra=wide)
    good = fa.decode_paged_weights(q, kp, vp, table, c, w)
    t, n = table.clone(), c.clone()
    t[0, 2], t[1, 9] = -1, kp.shape[0]
    n[2], n[3] = 16 * table.shape[1] + 7, -4
    O, L, W = fa.decode_paged_weights(q, kp, vp, t, n, w)
    for b in range(4):
        assert torch.isnan(O[b]).all() and torch.isnan(L[b]).all()
    assert torch.isnan(W[0, :, :40]).all() and torch.equal(W[0, :, 40:], w[0, :, 40:])
    assert torch.isnan(W[1, :, :300]).all() and torch.isnan(W[2]).all()
    assert torch.equal(W[3], w[3]) and torch.equal(W[4], w[4])
    assert (O[4] == 0).all() and torch.isneginf(L[4]).all()
    t[0, 3:] = -1   # entries past a context are not looked at
    t[0, 2] = table[0, 2]
    O, L, W = fa.decode_paged_weights(q, kp, vp, t, c.index_fill(0, torch.tensor([1], device=dev), 16), w)
    assert torch.equal(O[0], good[0][0]) and torch.equal(W[0], good[2][0])


@pytest.mark.parametrize("wide", [0, 40])
def test_weights_graph(fa, dev, wide):
    """The weights added up in place by a captured step, replayed, against eager steps."""
    q, kp, vp, table, c, w = _paged(dev, 6, 4, 16, 4, 64, [90, 0, 17, 200], "bf16", poison=False, extra=wide)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fa.decode_paged_weights(q, kp, vp, table, c, w.clone(), inplace=True)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fa.decode_paged_weights(q, kp, vp, table, c, w, inplace=True)
    mine = w.clone()
    for i in range(4):
        q.copy_(torch.randn_like(q))
        c[3] = 200 - 3 * i
        graph.replay()
        want = fa.decode_paged_weights(q, kp, vp, table, c, mine, inplace=True)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, want)), i


@pytest.mark.parametrize("wide", [0, 40])
def test_weights_two_streams(fa, dev, wide):
    cases = [_paged(dev, 30 + i, 4, 16, 4, 128, [90 + i, 0, 300, 5], "fp16", extra=wide) for i in range(2)]
    want = [fa.decode_paged_weights(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(fa.decode_paged_weights(*cases[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, y) for out in got[i] for x, y in zip(out, want[i]))


# ---------------------------------------------------------------------------
# kv_evict
# ---------------------------------------------------------------------------
def _evict_case(dev, seed, Hkv, D, ctx, keep, dtype="fp16", ties=True, wide=0):
    B = len(ctx)
    rng = np.random.default_rng(seed)
    old = [-(-n // 16) for n in ctx]
    new = [-(-min(n, keep) // 16) for n in ctx]
    pages = sum(old) + sum(new) + 2
    perm = rng.permutation(pages).astype(np.int32)
    table = np.full((B, max(1, max(old)) + wide), -1, np.int32)
    new_table = np.full((B, -(-keep // 16) + wide), -1, np.int32)
    at = 0
    for t, need in ((table, old), (new_table, new)):
        for b, n in enumerate(need):
            t[b, :n] = perm[at:at + n]
            at += n
    pools = [torch.from_numpy(rng.integers(-2 ** 15, 2 ** 15, (pages, Hkv, 16, D)).astype(np.int16)).view(TYPES[dtype]) for _ in range(2)]
    w = np.exp(2 * rng.standard_normal((B, Hkv, 16 * table.shape[1]))).astype(np.float32)
    if ties:
        w = np.floor(w * 4) / np.float32(4)
    return pools, table, np.array(ctx, np.int32), w, new_table


def _run_evict(fa, dev, pools, table, ctx, w, new_table, keep, recent):
    p = [x.to(dev) for x in pools]
    t = lambda x: torch.from_numpy(x).to(dev)
    out = fa.kv_evict(*p, t(table), t(ctx), t(w), t(new_table), keep, recent)
    return [x.cpu().view(torch.int16).numpy() for x in p] + [x.cpu().numpy() for x in out]


def _check_evict(fa, dev, pools, table, ctx, w, new_table, keep, recent, tag=""):
    got = _run_evict(fa, dev, pools, table, ctx, w, new_table, keep, recent)
    want = cache.evict(*[x.view(torch.int16).numpy() for x in pools], table, ctx, w, new_table, keep, recent)
    for g, x, name in zip(got, want, ("k_pool", "v_pool", "kept", "new_weights", "new_lens", "bad")):
        assert g.shape == x.shape and np.array_equal(g, x, equal_nan=name == "new_weights"), \
            f"{tag}: {name} differs in {(g != x).sum()} places"


EVICT = [([1], 1, 0), ([2], 1, 0), ([2], 1, 1), ([5, 0, 9], 4, 2), ([16, 17, 33], 16, 0), ([100, 31, 64], 33, 33),
         ([300, 20], 64, 7), ([70, 1030, 2100, 513], 200, 16), ([5000], 1000, 100), ([40, 41], 50, 10), ([1025, 1024], 1023, 1),
         ([3000, 64], 2999, 0)]


@pytest.mark.parametrize("D,Hkv,dtype", [(64, 3, "fp16"), (128, 2, "bf16")])
@pytest.mark.parametrize("ties", [True, False])
@pytest.mark.parametrize("i", range(len(EVICT)))
def test_evict_matches_oracle(fa, dev, i, ties, D, Hkv, dtype):
    ctx, keep, recent = EVICT[i]
    case = _evict_case(dev, i, Hkv, D, ctx, keep, dtype, ties, wide=i % 3)
    _check_evict(fa, dev, *case, keep, recent, f"{EVICT[i]}")


@pytest.mark.parametrize("kind", ["zeros", "one value", "nan", "negative", "infinite", "steps", "bits"])
def test_evict_odd_weights(fa, dev, kind):
    """Equal weights stay from the lowest slot on; -0 is 0; NaN goes first; every digit of the order is used."""
    ctx, keep, recent = [700, 90], 100, 9
    pools, table, c, w, new_table = _evict_case(dev, 20, 2, 64, ctx, keep)
    rng = np.random.default_rng(5)
    if kind == "zeros":
        w[:] = np.where(rng.random(w.shape) < 0.5, 0.0, -0.0)
    elif kind == "one value":
        w[:] = 0.25
    elif kind == "nan":
        w[rng.random(w.shape) < 0.95] = np.nan
    elif kind == "negative":
        w[:] = rng.standard_normal(w.shape)
    elif kind == "infinite":
        w[rng.random(w.shape) < 0.3] = np.inf
        w[rng.random(w.shape) < 0.3] = -np.inf
    elif kind == "steps":
        w[:] = np.float32(1) + rng.integers(0, 40, w.shape).astype(np.float32) * np.float32(2.0 ** -23)
    else:
        w[:] = rng.integers(0, 2 ** 32, w.shape, dtype=np.uint32).view(np.float32)
    _check_evict(fa, dev, pools, table, c, w, new_table, keep, recent, kind)


def test_evict_invalid(fa, dev):
    """Rows without an old or a new page are flagged and left out; lengths out of range leave nothing."""
    ctx, keep, recent = [100, 100, 100, 100, 30, 100], 40, 8
    pools, table, c, w, new_table = _evict_case(dev, 21, 2, 64, ctx, keep)
    pages = pools[0].shape[0]
    table[0, 6] = pages      # of the newest
    new_table[1, 1] = -7
    c[2], c[3] = -1, 16 * table.shape[1] + 1
    new_table[4, 0] = pages
    _check_evict(fa, dev, pools, table, c, w, new_table, keep, recent)
    got = _run_evict(fa, dev, pools, table, c, w, new_table, keep, recent)
    assert got[5].tolist() == [1, 1, 1, 1, 1, 0] and got[4].tolist() == [40, 40, 0, 0, 30, 40]


def test_evict_far_pages(fa, dev):
    """Pages past 2^31 values of a pool."""
    Hkv, D, ctx, keep = 8, 128, [90, 33], 32
    pools, table, c, w, new_table = _evict_case(dev, 22, Hkv, D, ctx, keep)
    n = pools[0].shape[0]
    pages = (1 << 31) // (Hkv * 16 * D) + n + 1
    far = [torch.empty(pages, Hkv, 16, D, dtype=x.dtype, device=dev) for x in pools]
    for f, x in zip(far, pools):
        f[pages - n:] = x.to(dev)
    t = lambda x: torch.from_numpy(x).to(dev)
    shift = lambda x: np.where(x >= 0, x + pages - n, x).astype(np.int32)
    out = fa.kv_evict(*far, t(shift(table)), t(c), t(w), t(shift(new_table)), keep, 5)
    want = _run_evict(fa, dev, pools, table, c, w, new_table, keep, 5)
    for f, x in zip(far, want[:2]):
        assert np.array_equal(f[pages - n:].cpu().view(torch.int16).numpy(), x)
    assert all(np.array_equal(a.cpu().numpy(), b) for a, b in zip(out, want[2:]))


def test_evict_many_tokens(fa, dev):
    """130000 slots of one head, of which half stay: counted by torch's stable sort."""
    n, keep, recent = 130000, 65000, 100
    g = torch.Generator(device=dev)
    g.manual_seed(3)
    w = torch.floor(torch.rand((1, 1, -(-n // 16) * 16), generator=g, device=dev) * 5000) / 5000
    pages = -(-n // 16) + -(-keep // 16)
    pools = [torch.randn((pages, 1, 16, 64), generator=g, device=dev, dtype=torch.bfloat16) for _ in range(2)]
    table = torch.arange(-(-n // 16), dtype=torch.int32, device=dev)[None]
    new_table = torch.arange(-(-n // 16), pages, dtype=torch.int32, device=dev)[None]
    rows = [p.reshape(-1, 64)[:n].clone() for p in pools]
    kept, new_w, lens, bad = fa.kv_evict(*pools, table, _i32(dev, [n]), w, new_table, keep, recent)
    order = torch.sort(w[0, 0, :n - recent], descending=True, stable=True).indices[:keep - recent]
    want = torch.cat((torch.sort(order).values, torch.arange(n - recent, n, device=dev)))
    assert torch.equal(kept[0, 0].long(), want) and lens.tolist() == [keep] and bad.tolist() == [0]
    assert torch.equal(new_w[0, 0, :keep], w[0, 0, want])
    for p, r in zip(pools, rows):
        assert torch.equal(p[table.shape[1]:].reshape(-1, 64)[:keep], r[want])


def test_evict_graph(fa, dev):
    pools, table, c, w, new_table = _evict_case(dev, 23, 2, 64, [300, 80, 500], 64)
    t = lambda x: torch.from_numpy(x).to(dev)
    p, tw, tc = [x.to(dev) for x in pools], t(w), t(c)
    tables = t(table), t(new_table)

    def call(p):
        return fa.kv_evict(*p, tables[0], tc, tw, tables[1], 64, 10)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(p)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(p)
    for i in range(4):
        tw.copy_(torch.rand_like(tw))
        tc[2] = 500 - 100 * i
        mine = [x.clone() for x in p]
        graph.replay()
        want = call(mine)
        torch.cuda.synchronize()
        assert all(torch.equal(x.view(torch.int16) if x.dtype == torch.float16 else x, y.view(torch.int16) if y.dtype == torch.float16 else y)
                   for x, y in zip([*out, *p], [*want, *mine])), i


def test_a_budget_as_used(fa, dev):
    """A small server: prompts behind a shared instruction, tokens generated with weights added up, the cache cut to its
    budget, tokens generated on. Every step's attention is that of the rows that should be in the cache, rotated by the
    positions at which they came."""
    B, H, Hkv, D, P, T, keep, recent = 3, 8, 2, 64, 37, 60, 40, 12
    rng = np.random.default_rng(1)
    freqs, _ = fa.rope_frequencies(D, device=dev)
    f = _f64(freqs)
    g = torch.Generator(device=dev)
    g.manual_seed(5)
    rnd = lambda *s: torch.randn(s, generator=g, device=dev, dtype=torch.float16)
    pages = rng.permutation(80).astype(np.int32)
    take = lambda n, at=[0]: (pages[at[0]:at[0] + n], at.__setitem__(0, at[0] + n))[0]
    pools = [torch.zeros(80, Hkv, 16, D, dtype=torch.float16, device=dev) for _ in range(2)]
    prefix = torch.from_numpy(take(3)).to(dev)
    old = torch.from_numpy(np.stack([take(6) for _ in range(B)])).to(dev)
    new = torch.from_numpy(np.stack([take(4) for _ in range(B)])).to(dev)
    # the instruction, once; then each prompt from position P on
    k0, v0, q0 = rnd(1, Hkv, P, D), rnd(1, Hkv, P, D), rnd(1, H, P, D)
    _, bad = fa.kv_append_rope(q0, k0, v0, *pools, prefix[None].contiguous(), _i32(dev, [0]), freqs)
    lens = [60, 33, 51]
    kt, vt, qt = rnd(B, Hkv, T, D), rnd(B, Hkv, T, D), rnd(B, H, T, D)
    zero, at = _i32(dev, [0] * B), _i32(dev, [P] * B)
    fa.kv_append_rope(qt, kt, vt, *pools, old, zero, freqs, at, _i32(dev, lens))
    ks = [[rotary.rotate(_f64(kt[b, :, :n]), np.arange(P, P + n), f), _f64(vt[b, :, :n])] for b, n in enumerate(lens)]
    shared = [rotary.rotate(_f64(k0[0]), np.arange(P), f), _f64(v0[0])]
    table, slots, pos = old, _i32(dev, lens), _i32(dev, [P + n for n in lens])
    weights = torch.zeros(B, Hkv, 16 * old.shape[1], device=dev)
    plain = np.zeros((B, Hkv, 16 * old.shape[1]))

    def attend(b, q, with_prefix):
        """Per head (o, weights of the own rows), and how far they may be off: q and k are rounded once each."""
        k, v = ks[b]
        if with_prefix:
            k, v = np.concatenate([shared[0], k], 1), np.concatenate([shared[1], v], 1)
        out = []
        for h in range(H):
            kk, vv = k[h // (H // Hkv)], v[h // (H // Hkv)]
            s = kk @ q[h] / 8
            e = np.exp(s - s.max())
            p = e / e.sum()
            ds = 2.0 ** -10 * (np.abs(kk) @ np.abs(q[h])).max() / 8 + 1e-5
            out.append((p @ vv, p, (2 * ds + 2.0 ** -10) * (p @ np.abs(vv)) + 2.0 ** -11 * np.abs(p @ vv) + 1e-5, p * (2.1 * ds)))
        return out

    for step in range(12):
        if step == 6:
            kept, weights, slots, bad = fa.kv_evict(*pools, table, slots, weights, new, keep, recent)
            table = new
            assert not bad.any() and slots.tolist() == [min(n + 6, keep) for n in lens]
            plain = np.zeros((B, Hkv, 16 * new.shape[1]))
            for b in range(B):
                n = int(slots[b])
                idx = kept[b, :, :n].cpu().numpy()
                assert (np.diff(idx, axis=1) > 0).all() and (idx[:, n - min(recent, n):] >= lens[b] + 6 - recent).all()
                ks[b] = [np.take_along_axis(x, idx[:, :, None], 1) for x in ks[b]]
            plain[:] = _f64(weights)
        q, k, v = rnd(B, H, 1, D), rnd(B, Hkv, 1, D), rnd(B, Hkv, 1, D)
        qr, bad = fa.kv_append_rope(q, k, v, *pools, table, slots, freqs, pos)
        assert not bad.any()
        slots, qr = slots + 1, qr[:, :, 0].contiguous()
        O, L = fa.decode_shared(qr, *pools, prefix, _i32(dev, [P]), table, slots)
        O2, L2, weights = fa.decode_paged_weights(qr, *pools, table, slots, weights)
        for b in range(B):
            p = int(pos[b])
            ks[b] = [np.concatenate([x, y], 1) for x, y in zip(ks[b], (rotary.rotate(_f64(k[b]), [p], f), _f64(v[b])))]
            qa = rotary.rotate(_f64(q[b]), [p], f)[:, 0]
            assert ks[b][0].shape[1] == int(slots[b])
            for got, with_prefix in ((O, True), (O2, False)):
                for h, (o, w, tol, tw) in enumerate(attend(b, qa, with_prefix)):
                    assert (np.abs(_f64(got[b, h]) - o) <= tol).all(), (step, b, h)
                    if not with_prefix:
                        n = len(w)
                        plain[b, h // (H // Hkv), :n] += w
        pos = pos + 1
    # twelve steps' weights, each off by less than 2.1 times a score's error (above, 0.05 here) of itself
    err = np.abs(_f64(weights) - plain)
    assert (err <= 0.1 * np.maximum(plain, 1e-6) + 1e-6).all()


@pytest.mark.parametrize("ctx,wide", [([1], 0), ([2, 17, 0, 500], 0), ([3000, 33, 1100], 0), ([333, 5], 40), ([20000], 0)])
@pytest.mark.parametrize("D,dtype", [(64, "fp16"), (128, "fp16"), (64, "bf16"), (128, "bf16")])
def test_weights_huge_scores(fa, dev, D, dtype, ctx, wide):
    """Scores (in units of log 2) of 2^17 to 2^33 in fp16 and to 2^90 in bf16, of both signs: O, L and the weights follow from the
    scores' differences."""
    b, qs = HUGE[dtype]
    B = len(ctx)
    q, kp, vp, _, _, table, c = _huge_scores(_case(dev, B, B, 16, 2, D, 0, ctx, dtype, extra=wide), b, qs)
    w = torch.rand((B, 2, 16 * table.shape[1]), device=dev)
    got = fa.decode_paged_weights(q, kp, vp, table, c, w)
    qf, kf, vf, tf, want = [_f64(x) for x in (q, kp, vp, table, w)]
    res = [np.zeros((B, 16, D)), np.full((B, 16), -np.inf), np.zeros((B, 16, D)), np.zeros((B, 16))]
    tw = np.zeros(want.shape)
    for i, n in enumerate(ctx):
        for h in range(2 if n else 0):
            g = slice(8 * h, 8 * h + 8)
            k, v = (cache.rows(x, tf[i, :-(-n // 16)], n, h) for x in (kf, vf))
            s = qf[i, g] @ k.T
            assert np.array_equal(s.astype(np.float32), s)
            o, l, p, to, tl, tp = cache.attend_exact(s, v, HALF[dtype], HALF[dtype] ** 2)
            for x, y in zip(res, (o, l, to, tl)):
                x[i, g] = y
            want[i, h, :n] += p.sum(0)
            tw[i, h, :n] = tp.sum(0) + 9 * 2.0 ** -24 * want[i, h, :n]   # the sum's roundings
    _check(got[:2], res, dtype, f"{ctx}")
    err = np.abs(_f64(got[2]) - want)
    assert (err <= tw).all(), f"{ctx} W: worst {np.nanmax(err / np.maximum(tw, 1e-300)):.2f} of the bound, {np.isnan(err).sum()} NaN"


@pytest.mark.parametrize("top", [118, -118])
@pytest.mark.parametrize("H,Hkv,ctx", [(4, 1, [500]), (4, 1, [20000]), (8, 8, [3000, 700, 40]), (1, 1, [131072])])
@pytest.mark.parametrize("D", [64, 128])
def test_weights_range_of_bf16(fa, dev, D, H, Hkv, ctx, top):
    """V of 2^118 and of 2^-118 in equal weights: what up to 131072 of them add up to is past the range, O is V. Equal weights' sums
    are (n / 16 + 64) 2^-24 off, twice: 2^-10, below half a place of O."""
    q, kp, vp, table, c, w = _paged(dev, 3, len(ctx), H, Hkv, D, ctx, "bf16", poison=False)
    kp.zero_()
    sign = torch.where(torch.arange(D, device=dev) % 3 == 0, -1.0, 1.0)
    vp.copy_((sign * 2.0 ** top).expand_as(vp))
    O, L, W = fa.decode_paged_weights(q, kp, vp, table, c, w)
    assert torch.equal(O, (sign * 2.0 ** top).to(O.dtype).expand_as(O))
    for b, n in enumerate(ctx):
        off = (n / 16 + 64) * 2.0 ** -24 + 2.0 ** -21
        assert (L[b].double() - math.log(n)).abs().max() <= off + 2.0 ** -21 * math.log(n)
        add = (W[b, :, :n].double() - w[b, :, :n].double()) * n * Hkv / H
        assert (add - 1).abs().max() <= off + 2.0 ** -24 * 4 * n * Hkv / H   # and the sum with weights of up to 3


@pytest.mark.parametrize("wide", [0, 40])
@pytest.mark.parametrize("D,dtype", [(64, "fp16"), (128, "bf16")])
def test_weights_masked_by_minus_infinity(fa, dev, D, dtype, wide):
    """Keys whose scores are -inf get no weight; where all of a head are, O is 0, L -inf and the weights stay as they were."""
    q, kp, vp, table, c, w = _paged(dev, 8, 3, 8, 2, D, [300, 33, 16], dtype, extra=wide)
    q[..., 0] = q[..., 0].abs() + 0.5
    k = kp.clone()
    for b, n in ((0, 300), (1, 33)):
        k[table[b, :-(-n // 16)].long(), 0, :, 0] = -math.inf      # KV head 0: all
    k[table[0, :10].long(), 1, :, 0] = -math.inf                   # and of head 1 the first 160 keys
    O, L, W = fa.decode_paged_weights(q, k, vp, table, c, w)
    assert (O[:2, :4] == 0).all() and torch.isneginf(L[:2, :4]).all() and torch.equal(W[:2, 0], w[:2, 0])
    assert torch.equal(W[0, 1, :160], w[0, 1, :160])
    for b, h, skip in ((0, 1, 160), (1, 1, 0), (2, 0, 0), (2, 1, 0)):
        n, g = int(c[b]), slice(4 * h, 4 * h + 4)
        kk, vv = (cache.rows(_f64(x), table[b, :-(-n // 16)].cpu().numpy(), n, h)[skip:] for x in (kp, vp))
        o, l, p, to, tl, tp = cache.attend(_f64(q[b, g]), kk, vv, HALF[dtype])
        assert (np.abs(_f64(O[b, g]) - o) <= to).all() and (np.abs(_f64(L[b, g]) - l) <= tl).all()
        want = _f64(w[b, h, skip:n]) + p.sum(0)
        assert (np.abs(_f64(W[b, h, skip:n]) - want) <= tp.sum(0) + 5 * 2.0 ** -24 * want).all()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("B,H,Hkv,D,ctx", [(8, 32, 8, 128, [200, 0, 777, 4, 1025, 16, 90, 3]), (3, 16, 8, 64, [2000, 33, 515])])
def test_weights_of_a_large_pool(fa, dev, B, H, Hkv, D, ctx, dtype):
    """Pools from 64 MiB on: pages are read past the caches."""
    pages = (64 << 20) // (Hkv * 16 * D * 4)
    case = _paged(dev, 11, B, H, Hkv, D, ctx, dtype, spare=pages, extra=40)
    got = fa.decode_paged_weights(*case)
    _check_weights(got, case, dtype)
    again = fa.decode_paged_weights(*case)
    assert all(torch.equal(x, y) for x, y in zip(got, again))


@pytest.mark.parametrize("wide", [0, 40])
def test_weights_far_pages(fa, dev, wide):
    """Pages past 2^31 values of a pool, in one launch and in chunks; the same call on a small pool gives its bits."""
    Hkv, D = 8, 128
    pages = (1 << 31) // (Hkv * 16 * D) + 100
    q, kp, vp, table, c, w = _paged(dev, 12, 3, 16, Hkv, D, [150, 0, 33], "bf16", spare=0, extra=wide)
    n = kp.shape[0]
    far = []
    for x in (kp, vp):
        y = torch.empty(pages, Hkv, 16, D, dtype=x.dtype, device=dev)
        y[pages - n:] = x
        far.append(y)
    got = fa.decode_paged_weights(q, *far, torch.where(table >= 0, table + (pages - n), table), c, w)
    want = fa.decode_paged_weights(q, kp, vp, table, c, w)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    _check_weights(got, (q, kp, vp, table, c, w), "bf16")


@pytest.mark.parametrize("ctx,wide", [([400, 9], 0), ([2500, 77, 0], 0), ([300, 5], 40)])
@pytest.mark.parametrize("D,dtype", [(64, "fp16"), (128, "bf16")])
def test_weights_climbing_scores(fa, dev, D, dtype, ctx, wide):
    """The maximum moves along the keys, by little and by far."""
    B = len(ctx)
    q, kp, vp, prefix, plen, table, c = _climbing_scores(_case(dev, 5, B, 16, 2, D, 0, ctx, dtype, extra=wide))
    w = torch.rand((B, 2, 16 * table.shape[1]), device=dev)
    O, L, W = fa.decode_paged_weights(q, kp, vp, table, c, w)
    want, tol = _f64(w), np.zeros(w.shape)
    for b, n in enumerate(ctx):
        for h in range(2 if n else 0):
            g = slice(8 * h, 8 * h + 8)
            k, v = (cache.rows(_f64(x), table[b, :-(-n // 16)].cpu().numpy(), n, h) for x in (kp, vp))
            o, l, p, to, tl, tp = cache.attend_exact(_f64(q[b, g]) @ k.T, v, HALF[dtype], HALF[dtype] ** 2)
            assert (np.abs(_f64(O[b, g]) - o) <= to).all() and (np.abs(_f64(L[b, g]) - l) <= tl).all()
            want[b, h, :n] += p.sum(0)
            tol[b, h, :n] = tp.sum(0) + 9 * 2.0 ** -24 * want[b, h, :n]
    assert (np.abs(_f64(W) - want) <= tol).all()


# Tables of the eviction: up to 256 pages the selection lists what stays, beyond a launch of its own does; up to 1024, to 2048 and
# more pages it has 16, 32 and no keys of a thread in registers.
WIDE = [300, 1100, 2100]


@pytest.mark.parametrize("wide", WIDE)
@pytest.mark.parametrize("kind", ["zeros", "one value", "nan", "negative", "infinite", "steps", "bits"])
def test_evict_odd_weights_of_wide_tables(fa, dev, kind, wide):
    """As test_evict_odd_weights."""
    ctx, keep, recent = [700, 90, 2500], 100, 9
    pools, table, c, w, new_table = _evict_case(dev, 20, 2, 64, ctx, keep, wide=wide)
    rng = np.random.default_rng(5)
    if kind == "zeros":
        w[:] = np.where(rng.random(w.shape) < 0.5, 0.0, -0.0)
    elif kind == "one value":
        w[:] = 0.25
    elif kind == "nan":
        w[rng.random(w.shape) < 0.97] = np.nan
    elif kind == "negative":
        w[:] = rng.standard_normal(w.shape)
    elif kind == "infinite":
        w[rng.random(w.shape) < 0.3] = np.inf
        w[rng.random(w.shape) < 0.3] = -np.inf
    elif kind == "steps":
        w[:] = np.float32(1) + rng.integers(0, 40, w.shape).astype(np.float32) * np.float32(2.0 ** -23)
    else:
        w[:] = rng.integers(0, 2 ** 32, w.shape, dtype=np.uint32).view(np.float32)
    _check_evict(fa, dev, pools, table, c, w, new_table, keep, recent, kind)


@pytest.mark.parametrize("wide", WIDE)
def test_evict_invalid_of_wide_tables(fa, dev, wide):
    """As test_evict_invalid."""
    ctx, keep, recent = [100, 100, 100, 100, 30, 100], 40, 8
    pools, table, c, w, new_table = _evict_case(dev, 21, 2, 64, ctx, keep, wide=wide)
    pages = pools[0].shape[0]
    table[0, 6] = pages
    new_table[1, 1] = -7
    c[2], c[3] = -1, 16 * table.shape[1] + 1
    new_table[4, 0] = pages
    _check_evict(fa, dev, pools, table, c, w, new_table, keep, recent)
    got = _run_evict(fa, dev, pools, table, c, w, new_table, keep, recent)
    assert got[5].tolist() == [1, 1, 1, 1, 1, 0] and got[4].tolist() == [40, 40, 0, 0, 30, 40]


@pytest.mark.parametrize("wide", [0, *WIDE])
@pytest.mark.parametrize("keep,recent", [(64, 0), (64, 1), (64, 63), (64, 64), (1500, 1500), (1500, 20), (1, 0), (1, 1)])
def test_evict_mixed_batches(fa, dev, keep, recent, wide):
    """Caches above, at and below the budget, empty ones and an invalid length side by side; nothing but the newest, and nothing of them."""
    ctx = [1, 64, 65, 0, 4000, 63, 1500, 1501, 17]
    case = _evict_case(dev, 24, 2, 64, ctx, keep, "bf16", wide=wide)
    case[2][8] = -3
    _check_evict(fa, dev, *case, keep, recent, f"{keep} {recent}")


@pytest.mark.parametrize("ctx,keep,recent", [([20000], 4096, 256), ([17000, 300, 32768, 16385], 1000, 0), ([33000], 4096, 4096)])
def test_evict_long(fa, dev, ctx, keep, recent):
    """Lengths that fill tables of 1025 pages and more."""
    _check_evict(fa, dev, *_evict_case(dev, 25, 2, 64, ctx, keep, "bf16"), keep, recent)


def test_graphs_of_one_pool(fa, dev):
    """A decode with weights and an eviction, captured with one memory pool, so that their workspaces share memory, replayed in
    turn with new queries and lengths, eager calls between."""
    q, kp, vp, table, c, w = _paged(dev, 26, 3, 16, 2, 64, [600, 90, 300], "fp16", poison=False, extra=300, spare=60)
    t, n = table.clone().clamp_(min=0), kp.shape[0]
    used = set(table[table >= 0].tolist())
    new = torch.tensor([i for i in range(n) if i not in used][:24], dtype=torch.int32, device=dev).reshape(3, 8)

    def decode(w):
        return fa.decode_paged_weights(q, kp, vp, t, c, w)

    def evict(k, v):
        return fa.kv_evict(k, v, t, c, w, new, 100, 10)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        decode(w), evict(kp.clone(), vp.clone())
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs, pool = [], [], None
    for call in (lambda: decode(w), lambda: evict(kp, vp)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            outs.append(call())
        pool = graph.pool()
        graphs.append(graph)
    for i in range(4):
        q.copy_(torch.randn_like(q))
        w.copy_(torch.rand_like(w))
        c[0] = 600 - 100 * i
        pools = kp.clone(), vp.clone()
        for graph in graphs:
            graph.replay()
        want = [*decode(w), *evict(*pools)]
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip([*outs[0], *outs[1], kp, vp], [*want, *pools])), i


@pytest.mark.parametrize("ctx,wide", [([320, 16], 0), ([320, 16], 40), ([4000, 0], 0)])
@pytest.mark.parametrize("D,dtype", [(64, "fp16"), (128, "fp16"), (64, "bf16"), (128, "bf16")])
def test_weighted_values_keep_two_terms(fa, dev, D, dtype, ctx, wide):
    """P has two terms of the type, 22 bits in fp16 and 16 in bf16, in one launch and in chunks."""
    case = _coherent_roundings(_case(dev, 3, 2, 8, 2, D, 0, ctx, dtype, poison=False, extra=wide))
    want = _want_exact(case, HALF[dtype], HALF[dtype] ** 2)
    assert not _one_term(case, want, 0, ctx[0])
    q, kp, vp, _, _, table, c = case
    _check(fa.decode_paged_weights(q, kp, vp, table, c, torch.zeros(2, 2, 16 * table.shape[1], device=dev))[:2], want, dtype)
