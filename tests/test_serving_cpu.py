"""CPU tier of the rotary positions, the shared prefix and the cache budget: arguments are refused before any HIP call, by
the C ABI and by the torch binding; rope_frequencies; the oracles against each other."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from oracle import cache, rotary

A = 0x10000   # a fake, 16-byte aligned address: never dereferenced by validation


def _st(*x):
    return C.cast((C.c_int64 * 3)(*x), C.c_void_p)


def _rope(**kw):
    a = dict(q=A, qs=_st(8 * 64 * 128, 64 * 128, 128), k=A, ks=_st(8 * 64 * 128, 64 * 128, 128), f=A, p=A, ps=64, qo=A, ko=A, B=2, H=8,
             Hkv=8, N=64, D=128, R=128, it=0, ot=0)
    a.update(kw)
    return [a[x] for x in ("q", "qs", "k", "ks", "f", "p", "ps", "qo", "ko", "B", "H", "Hkv", "N", "D", "R", "it", "ot")]


ROPE = [
    (dict(), "FA_OK"), (dict(q=0), "FA_ERR_NULL_POINTER"), (dict(qs=None), "FA_ERR_NULL_POINTER"), (dict(f=0), "FA_ERR_NULL_POINTER"),
    (dict(k=0), "FA_ERR_NULL_POINTER"), (dict(ko=0), "FA_ERR_NULL_POINTER"), (dict(k=0, ko=0, ks=None, Hkv=0), "FA_OK"),
    (dict(p=0), "FA_OK"), (dict(D=96, R=96), "FA_ERR_HEAD_DIM"), (dict(N=0), "FA_ERR_SEQ_LEN"), (dict(B=0), "FA_ERR_BATCH_HEADS"),
    (dict(Hkv=-1), "FA_ERR_KV_HEADS"), (dict(R=0), "FA_ERR_ROT_DIM"), (dict(R=24), "FA_ERR_ROT_DIM"), (dict(R=144), "FA_ERR_ROT_DIM"),
    (dict(R=16), "FA_OK"), (dict(it=2, ot=0), "FA_OK"), (dict(it=2, ot=1), "FA_OK"), (dict(it=2, ot=2), "FA_OK"),
    (dict(it=0, ot=1), "FA_ERR_TYPE"), (dict(it=1, ot=2), "FA_ERR_TYPE"), (dict(it=3, ot=3), "FA_ERR_TYPE"), (dict(it=-1, ot=-1), "FA_ERR_TYPE"),
    (dict(q=A + 2), "FA_ERR_ALIGNMENT"), (dict(ko=A + 8), "FA_ERR_ALIGNMENT"), (dict(f=A + 4), "FA_ERR_ALIGNMENT"),
    (dict(p=A + 2), "FA_ERR_ALIGNMENT"), (dict(qs=_st(4, 64 * 128, 128)), "FA_ERR_STRIDE"), (dict(ks=_st(8, 16, 129)), "FA_ERR_STRIDE"),
    (dict(ks=_st(8, 16, -128)), "FA_ERR_STRIDE"), (dict(qs=_st(3, 0, 128), B=1), "FA_OK"), (dict(qs=_st(4, 4, 4), it=2, ot=2), "FA_OK"),
    (dict(ps=-1), "FA_ERR_STRIDE"), (dict(B=70000), "FA_ERR_TOO_LARGE"), (dict(H=65530), "FA_ERR_TOO_LARGE"), (dict(N=1 << 29), "FA_ERR_TOO_LARGE"),
]


@pytest.mark.parametrize("i", range(len(ROPE)))
def test_validate_rope(capi, i):
    kw, code = ROPE[i]
    lib, a = capi.load(), _rope(**kw)
    assert lib.fa_validate_rope(*a) == capi.STATUS[code]
    if code != "FA_OK":
        assert lib.fa_rope(*a[:15], 1.0, 0, 0, *a[15:], None) == capi.STATUS[code]


def _append(**kw):
    st = _st(8 * 5 * 128, 5 * 128, 128)
    a = dict(q=A, qs=st, k=A, ks=st, v=A, vs=st, f=A, t=A, s=A, p=0, n=0, kp=A, vp=A, qo=A, ko=0, bad=A, B=2, H=8, Hkv=8, T=5, D=128, R=64,
             size=16, mp=10, pages=100)
    a.update(kw)
    return list(a.values())


APPEND = [
    (dict(), "FA_OK"), (dict(bad=0), "FA_ERR_NULL_POINTER"), (dict(q=0), "FA_ERR_NULL_POINTER"), (dict(v=0), "FA_ERR_NULL_POINTER"),
    (dict(vs=None), "FA_ERR_NULL_POINTER"), (dict(qo=0), "FA_ERR_NULL_POINTER"), (dict(t=0), "FA_ERR_NULL_POINTER"),
    (dict(f=0), "FA_ERR_NULL_POINTER"), (dict(T=0, q=0, k=0, v=0, qo=0, qs=None, ks=None, vs=None), "FA_OK"), (dict(T=-1), "FA_ERR_SEQ_LEN"),
    (dict(H=9), "FA_ERR_KV_HEADS"), (dict(H=0), "FA_ERR_KV_HEADS"), (dict(Hkv=0), "FA_ERR_BATCH_HEADS"), (dict(D=32, R=32), "FA_ERR_HEAD_DIM"),
    (dict(R=8), "FA_ERR_ROT_DIM"), (dict(size=32), "FA_ERR_PAGE_SIZE"), (dict(mp=0), "FA_ERR_MAX_PAGES"), (dict(pages=0), "FA_ERR_NUM_PAGES"),
    (dict(qs=_st(8, 8, 4)), "FA_ERR_STRIDE"), (dict(vs=_st(8, 8, -8)), "FA_ERR_STRIDE"), (dict(ko=A + 4), "FA_ERR_ALIGNMENT"),
    (dict(p=A + 1), "FA_ERR_ALIGNMENT"), (dict(k=A + 2), "FA_ERR_ALIGNMENT"), (dict(H=64000, Hkv=1000), "FA_ERR_TOO_LARGE"),
    (dict(T=(1 << 28) + 1), "FA_ERR_TOO_LARGE"),
]


@pytest.mark.parametrize("i", range(len(APPEND)))
def test_validate_append(capi, i):
    kw, code = APPEND[i]
    lib, a = capi.load(), _append(**kw)
    assert lib.fa_validate_kv_append_rope(*a) == capi.STATUS[code]
    if code != "FA_OK":
        assert lib.fa_kv_append_rope(*a[:22], 1.0, 0, *a[22:], 0, None) == capi.STATUS[code]


def _shared(**kw):
    a = dict(q=A, kp=A, vp=A, pt=A, pl=A, t=A, c=A, B=4, H=32, Hkv=8, D=128, size=16, pp=100, mp=20, pages=500, ws=A, o=A, l=A)
    a.update(kw)
    return list(a.values())


SHARED = [
    (dict(), "FA_OK"), (dict(q=0), "FA_ERR_NULL_POINTER"), (dict(pt=0), "FA_ERR_NULL_POINTER"), (dict(pl=0), "FA_ERR_NULL_POINTER"),
    (dict(ws=0), "FA_ERR_NULL_POINTER"), (dict(ws=0, pp=16, mp=20), "FA_OK"), (dict(ws=0, pp=17, mp=20), "FA_ERR_NULL_POINTER"),
    (dict(o=0), "FA_ERR_NULL_POINTER"), (dict(l=0), "FA_ERR_NULL_POINTER"), (dict(H=30), "FA_ERR_KV_HEADS"),
    (dict(Hkv=0), "FA_ERR_KV_HEADS"), (dict(D=96), "FA_ERR_HEAD_DIM"), (dict(B=0), "FA_ERR_BATCH_HEADS"), (dict(size=8), "FA_ERR_PAGE_SIZE"),
    (dict(pp=0), "FA_ERR_MAX_PAGES"), (dict(mp=0), "FA_ERR_MAX_PAGES"), (dict(pages=0), "FA_ERR_NUM_PAGES"), (dict(ws=A + 4), "FA_ERR_ALIGNMENT"),
    (dict(pl=A + 2), "FA_ERR_ALIGNMENT"), (dict(o=A + 2), "FA_ERR_ALIGNMENT"), (dict(pp=1 << 27), "FA_ERR_TOO_LARGE"),
    (dict(B=40000, H=1000, Hkv=1), "FA_ERR_TOO_LARGE"), (dict(B=70000), "FA_ERR_TOO_LARGE"),
    (dict(B=65535, H=128), "FA_OK"), (dict(B=65535, H=136), "FA_ERR_TOO_LARGE"),
]


@pytest.mark.parametrize("i", range(len(SHARED)))
def test_validate_shared(capi, i):
    kw, code = SHARED[i]
    lib, a = capi.load(), _shared(**kw)
    assert lib.fa_validate_decode_shared(*a) == capi.STATUS[code]
    if code != "FA_OK":
        assert lib.fa_decode_shared(*a, 0, None) == capi.STATUS[code]


def _weights(**kw):
    a = dict(q=A, kp=A, vp=A, t=A, c=A, w=A, B=4, H=32, Hkv=8, D=128, size=16, mp=20, pages=500, ws=A, o=A, l=A, wo=A)
    a.update(kw)
    return list(a.values())


WEIGHTS = [
    (dict(), "FA_OK"), (dict(w=0), "FA_ERR_NULL_POINTER"), (dict(wo=0), "FA_ERR_NULL_POINTER"), (dict(ws=0, mp=33), "FA_ERR_NULL_POINTER"),
    (dict(ws=0, mp=32), "FA_OK"), (dict(ws=0, H=136), "FA_ERR_NULL_POINTER"),
    (dict(l=0), "FA_ERR_NULL_POINTER"), (dict(H=30), "FA_ERR_KV_HEADS"),
    (dict(D=32), "FA_ERR_HEAD_DIM"), (dict(w=A + 4), "FA_ERR_ALIGNMENT"), (dict(wo=A + 8), "FA_ERR_ALIGNMENT"), (dict(l=A + 1), "FA_ERR_ALIGNMENT"),
    (dict(mp=1 << 17, B=2000, Hkv=2), "FA_OK"), (dict(mp=1 << 17, B=2100, Hkv=2), "FA_ERR_TOO_LARGE"), (dict(B=40000, H=1000, Hkv=1), "FA_ERR_TOO_LARGE"),
    (dict(B=65535, H=128), "FA_OK"), (dict(B=65535, H=136), "FA_ERR_TOO_LARGE"),
]


@pytest.mark.parametrize("i", range(len(WEIGHTS)))
def test_validate_weights(capi, i):
    kw, code = WEIGHTS[i]
    lib, a = capi.load(), _weights(**kw)
    assert lib.fa_validate_decode_weights(*a) == capi.STATUS[code]
    if code != "FA_OK":
        assert lib.fa_decode_paged_weights(*a, 0, None) == capi.STATUS[code]


def _evict(**kw):
    a = dict(kp=A, vp=A, t=A, c=A, w=A, nt=A, kept=A, nw=A, nl=A, bad=A, ws=A, B=4, Hkv=8, D=128, keep=100, recent=10, size=16, mp=20, nmp=7, pages=500)
    a.update(kw)
    return list(a.values())


EVICT = [
    (dict(), "FA_OK"), *((({x: 0}), "FA_ERR_NULL_POINTER") for x in ("kp", "vp", "t", "c", "w", "nt", "kept", "nw", "nl", "bad")),
    (dict(ws=0), "FA_OK"), (dict(ws=0, mp=256), "FA_OK"), (dict(ws=0, mp=257), "FA_ERR_NULL_POINTER"),
    (dict(D=96), "FA_ERR_HEAD_DIM"), (dict(B=0), "FA_ERR_BATCH_HEADS"), (dict(size=4), "FA_ERR_PAGE_SIZE"), (dict(mp=0), "FA_ERR_MAX_PAGES"),
    (dict(nmp=0), "FA_ERR_MAX_PAGES"), (dict(pages=-1), "FA_ERR_NUM_PAGES"), (dict(kp=A + 8), "FA_ERR_ALIGNMENT"), (dict(kept=A + 2), "FA_ERR_ALIGNMENT"),
    (dict(keep=0), "FA_ERR_BUDGET"), (dict(keep=113), "FA_ERR_BUDGET"), (dict(keep=112), "FA_OK"), (dict(recent=-1), "FA_ERR_BUDGET"),
    (dict(recent=101), "FA_ERR_BUDGET"), (dict(recent=100), "FA_OK"), (dict(mp=1 << 27), "FA_ERR_TOO_LARGE"), (dict(nmp=1 << 24), "FA_ERR_TOO_LARGE"),
    (dict(nmp=(1 << 24) - 128, keep=(1 << 28) - 2048), "FA_OK"), (dict(Hkv=70000), "FA_ERR_TOO_LARGE"),
]


@pytest.mark.parametrize("i", range(len(EVICT)))
def test_validate_evict(capi, i):
    kw, code = EVICT[i]
    lib, a = capi.load(), _evict(**kw)
    assert lib.fa_validate_kv_evict(*a) == capi.STATUS[code]
    if code != "FA_OK":
        assert lib.fa_kv_evict(*a, None) == capi.STATUS[code]


def test_status_strings(capi):
    lib = capi.load()
    for name, word in (("FA_ERR_ROT_DIM", b"rot_dim"), ("FA_ERR_STRIDE", b"stride"), ("FA_ERR_TYPE", b"type"), ("FA_ERR_BUDGET", b"recent")):
        assert word in lib.fa_status_str(capi.STATUS[name])


@pytest.mark.parametrize("B,H,Hkv,D,pp,mp", [(1, 1, 1, 64, 1, 1), (32, 32, 8, 128, 500, 94), (64, 32, 8, 128, 2048, 63), (1, 32, 1, 128, 8192, 1),
                                             (300, 32, 32, 64, 625, 1), (1, 128, 1, 128, 50, 2), (2000, 8, 8, 64, 10, 4000), (65535, 1, 1, 64, 4, 8)])
def test_workspaces(capi, B, H, Hkv, D, pp, mp):
    """Room for a part of the prefix and a chunk a sequence at least, at most 256 parts and 4096 workgroups' chunks or a
    chunk for 8 pages beside one a sequence; none for calls of one launch and for sizes that are refused."""
    lib = capi.load()
    part = B * H * (D + 2)
    chunk = H * (D + 2)
    groups = Hkv * -(-H // Hkv // 16)
    most = min(B * mp // 8, -(-4096 // groups)) + B
    small = 3 + 2 * B + (4 * (1 + most) if B > 256 else 0)
    n = lib.fa_decode_shared_workspace_floats(B, H, Hkv, D, pp, mp)
    blocks = B * Hkv * -(-H // Hkv // 16)
    if blocks <= 256 and (pp + mp) * D <= 4608 or blocks <= 512 and (pp + mp) * D <= 2304:
        assert n == 0
    else:
        assert part + B * chunk <= n <= min(256, -(-pp // 4)) * part + most * chunk + small
    w = lib.fa_decode_weights_workspace_floats(B, H, Hkv, D, mp)
    scores = B * H * 16 * mp
    if mp <= 32 and H // Hkv <= 16 and B * Hkv <= 512:
        assert w == 0
    else:
        assert scores + B * chunk <= w <= scores + most * chunk + small
    for bad in ((0, H, Hkv, D, pp, mp), (B, H, H + 1, D, pp, mp), (B, H, Hkv, 96, pp, mp), (B, H, Hkv, D, 0, mp), (B, H, Hkv, D, pp, -1),
                (B, 70000, 1, D, pp, mp), (B, H, Hkv, D, 1 << 27, mp), (65535, H, Hkv, D, pp, 1 << 16)):
        assert lib.fa_decode_shared_workspace_floats(*bad) == 0
        if bad[0] == 0 or bad[1] == 70000:
            assert lib.fa_kv_evict_workspace_words(bad[0], bad[1], 300) == 0
        if bad[4] not in (0, 1 << 27):
            assert lib.fa_decode_weights_workspace_floats(*bad[:4], bad[5]) == 0


@pytest.mark.parametrize("B,H,Hkv,D,pp,mp", [(257, 1, 1, 64, 20, 80), (301, 3, 1, 128, 9, 40), (257, 1, 1, 64, 24, 80), (1001, 5, 5, 64, 30, 9)])
def test_workspace_table_is_aligned(capi, B, H, Hkv, D, pp, mp):
    """Above 256 sequences the chunks' table, entries of 16 bytes, and then two words a sequence and one more end the
    workspace: the table lies on 16 bytes where what comes before it, and it, are multiples of four words."""
    lib = capi.load()
    assert (lib.fa_decode_shared_workspace_floats(B, H, Hkv, D, pp, mp) - 2 * B - 1) % 4 == 0
    assert (lib.fa_decode_weights_workspace_floats(B, H, Hkv, D, mp) - 2 * B) % 4 == 0


def test_binding_refuses_host_tensors(fa):
    x = torch.zeros(1, 2, 3, 64)
    i = torch.zeros(1, dtype=torch.int32)
    t = i[:, None]
    f, _ = fa.rope_frequencies(64, device="cpu")
    pool = torch.zeros(2, 2, 16, 64, dtype=torch.half)
    w = torch.zeros(1, 2, 16)
    for call in (lambda: fa.rope(x, x, f), lambda: fa.rope_backward(x, None, f),
                 lambda: fa.kv_append_rope(x, x, x, pool, pool, t, i, f),
                 lambda: fa.decode_shared(x[:, :, 0].half(), pool, pool, i, i, t, i),
                 lambda: fa.decode_paged_weights(x[:, :, 0].half(), pool, pool, t, i, w),
                 lambda: fa.kv_evict(pool, pool, t, i, w, t, 4, 1)):
        with pytest.raises(RuntimeError, match="must be CUDA tensors"):
            call()
    with pytest.raises(RuntimeError, match="dtype must be"):
        fa.rope_backward(x, None, f, dtype=torch.float64)


# ---------------------------------------------------------------------------
# rope_frequencies
# ---------------------------------------------------------------------------
def test_frequencies(fa):
    for R, base in ((64, 10000.0), (16, 500000.0), (128, 1e6)):
        f, scale = fa.rope_frequencies(R, base, device="cpu")
        assert f.dtype == torch.float64 and scale == 1.0
        assert np.allclose(f.numpy(), [base ** (-2 * i / R) for i in range(R // 2)], rtol=1e-14)
        lin, scale = fa.rope_frequencies(R, base, "linear", 4.0, device="cpu")
        assert torch.equal(lin, f / 4) and scale == 1.0
        ntk, scale = fa.rope_frequencies(R, base, "ntk", 8.0, device="cpu")
        assert scale == 1.0 and ntk[0] == 1 and float(f[-1] / ntk[-1]) == pytest.approx(8.0, rel=1e-12)
        assert (ntk[1:] < f[1:]).all()
        n = 4096
        parts, scale = fa.rope_frequencies(R, base, "by_parts", 16.0, n, device="cpu")
        assert scale == pytest.approx(0.1 * math.log(16) + 1)
        turns = n * f / (2 * math.pi)
        assert torch.equal(parts[turns > 32 * base ** (2 / R)], f[turns > 32 * base ** (2 / R)])
        slow = turns < base ** (-2 / R)
        assert torch.allclose(parts[slow], f[slow] / 16, rtol=1e-12)
        ratio = (parts / f).numpy()
        assert (np.diff(ratio) <= 1e-15).all() and ratio.max() <= 1 and ratio.min() >= 1 / 16 - 1e-15
        same, scale = fa.rope_frequencies(R, base, "by_parts", 1.0, n, device="cpu")
        assert torch.allclose(same, f, rtol=1e-14) and scale == 1.0


@pytest.mark.parametrize("R,base,n,slow,fast", [(128, 1e4, 131072, 1, 32), (128, 1e4, 65536, 1, 32), (16, 1e4, 65536, 1, 32), (64, 1e4, 1 << 20, 2, 20),
                                                (64, 5e5, 1 << 22, 1, 4), (128, 1e4, 150, 1, 32), (32, 1e4, 5, 1, 32), (64, 100.0, 4096, 1, 32),
                                                (16, 1e4, 4096, 1, 32), (8, 1e4, 40, 0.5, 1000)])
def test_frequencies_by_parts_ramp(fa, R, base, n, slow, fast):
    """The ramp's ends lie where the number of turns within the trained length is fast_turns and slow_turns, out of
    the frequencies there are too (a trained length above 2 pi base, or below 2 pi fast_turns): each frequency's share
    of the division is read off the line between the places, rounded outwards, found here by bisection over a real index."""
    def place(turns):
        lo, hi = -4.0 * R, 5.0 * R
        for _ in range(200):
            mid = (lo + hi) / 2
            lo, hi = (mid, hi) if n / (2 * math.pi) * base ** (-2 * mid / R) > turns else (lo, mid)
        return (lo + hi) / 2

    a, b = math.floor(place(fast)), math.ceil(place(slow))
    want = [min(max((i - a) / (b - a), 0.0), 1.0) for i in range(R // 2)]
    f = fa.rope_frequencies(R, base, device="cpu")[0].numpy()
    got, scale = fa.rope_frequencies(R, base, "by_parts", 8.0, n, slow_turns=slow, fast_turns=fast, device="cpu")
    assert scale == pytest.approx(0.1 * math.log(8) + 1)
    # five roundings of 2^-53 each in the ramp, its complement, the two products and the sum
    assert np.allclose(got.numpy(), [x * (1 - r) + x / 8 * r for x, r in zip(f, want)], rtol=2e-15, atol=0)
    turns = n * f / (2 * math.pi)
    step = base ** (2 / R)   # from one frequency to the next; beyond a place rounded outwards the ends are reached
    assert (got.numpy()[turns >= fast * step] == f[turns >= fast * step]).all()
    assert np.allclose(got.numpy()[turns <= slow / step], f[turns <= slow / step] / 8, rtol=2e-15, atol=0)


def test_frequencies_by_parts_by_hand(fa):
    """128 dims, base 10000, trained on 131072 positions, 8 times as long: fast_turns 32 at index 64 log(131072 / (64 pi)) / log
    10000 = 45.03, slow_turns 1 at 64 log(131072 / (2 pi)) / log 10000 = 69.11, past the last of the 64 frequencies. The ramp goes
    from 45 to 70: the last, of 2.4 turns, has 18 / 25 of the division, the one of index 50 a fifth of it."""
    f, _ = fa.rope_frequencies(128, 10000.0, device="cpu")
    g, _ = fa.rope_frequencies(128, 10000.0, "by_parts", 8.0, 131072, device="cpu")
    r = (g / f).numpy()
    assert np.allclose(r[[45, 50, 63]], [1, 1 - 0.2 * 7 / 8, 1 - 0.72 * 7 / 8], rtol=1e-14) and (r[:46] == 1).all()


def test_frequencies_by_parts_one_place(fa):
    """Numbers of turns so near to each other that both places are one index: kept up to it, divided from the next on."""
    R, base, n = 16, 1e4, 4096
    f, _ = fa.rope_frequencies(R, base, device="cpu")
    for k in (5, 7):
        slow = n / (2 * math.pi) * base ** (-2 * k / R)
        g, _ = fa.rope_frequencies(R, base, "by_parts", 8.0, n, slow_turns=slow, fast_turns=math.nextafter(slow, math.inf), device="cpu")
        assert torch.equal(g[:k + 1], f[:k + 1]) and torch.allclose(g[k + 1:], f[k + 1:] / 8, rtol=2e-15, atol=0)


def test_frequencies_refuse(fa):
    for kw, word in ((dict(rot_dim=0), "rot_dim"), (dict(rot_dim=15), "rot_dim"), (dict(rot_dim=16, base=1.0), "base"),
                     (dict(rot_dim=16, factor=0.5), "factor"), (dict(rot_dim=16, scaling="ramp"), "scaling"),
                     (dict(rot_dim=2, scaling="ntk"), "ntk"), (dict(rot_dim=16, scaling="by_parts"), "original_len"),
                     (dict(rot_dim=16, scaling="by_parts", original_len=10, slow_turns=5.0, fast_turns=5.0), "slow_turns"),
                     (dict(rot_dim=16, base=math.nan), "base")):
        with pytest.raises(RuntimeError, match=word):
            fa.rope_frequencies(**kw, device="cpu")


# ---------------------------------------------------------------------------
# The oracles
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("inter", [False, True])
def test_rotation_oracle(inter):
    """By hand for one pair; scores of rotated rows depend on the positions' difference alone; back is the transpose."""
    f = np.array([0.5, 0.01])
    x = np.array([[1.0, 2.0, 3.0, 4.0, 9.0]])
    y = rotary.rotate(x, [3], f, inter, 2.0)
    i, j = ((0, 1) if inter else (0, 2))
    a = 1.5
    assert np.allclose([y[0, i], y[0, j]], [2 * (x[0, i] * math.cos(a) - x[0, j] * math.sin(a)),
                                            2 * (x[0, j] * math.cos(a) + x[0, i] * math.sin(a))])
    assert y[0, 4] == 9.0
    rng = np.random.default_rng(0)
    q, k, g = rng.standard_normal((3, 6, 4))
    at = lambda p: (rotary.rotate(q, p + 5, f, inter) * rotary.rotate(k, p, f, inter)).sum(-1)
    assert np.allclose(at(np.arange(6)), at(np.arange(6) + 1000))
    p = np.arange(6) * 11
    assert np.allclose((g * rotary.rotate(q, p, f, inter, 1.5)).sum(), (rotary.rotate(g, p, f, inter, 1.5, True) * q).sum())


def test_cache_oracles():
    """A shared prefix is the same keys in every sequence; a head's weights sum to its query heads; eviction keeps what
    a sort by hand keeps."""
    rng = np.random.default_rng(0)
    kp, vp = rng.standard_normal((2, 9, 2, 16, 8))
    q = rng.standard_normal((2, 4, 8))
    prefix, table = np.array([3, 0]), np.array([[5, 6], [7, 8]])
    o, l, _, _ = cache.decode_shared(q, kp, vp, prefix, 32, table, [20, 3], 0.0)
    joined = np.concatenate([np.tile(prefix, (2, 1)), table], 1)
    o2, l2, w, _, _, _ = cache.decode_weights(q, kp, vp, joined, [52, 35], np.zeros((2, 2, 64)), 0.0)
    assert np.allclose(o, o2) and np.allclose(l, l2) and np.allclose(w.sum(-1), 2.0) and not w[1, :, 35:].any()
    w = np.array([[[5, 1, 5, 2, 5, 9, 0, 0, 1, 3] + [0] * 6]], np.float32)
    k, v = rng.standard_normal((2, 4, 1, 16, 8))
    k2, v2, kept, nw, n, bad = cache.evict(k, v, np.array([[2]]), [10], w, np.array([[1]]), 5, 2)
    assert kept.tolist() == [[[0, 2, 5, 8, 9]]] and nw[0, 0, :6].tolist() == [5, 5, 9, 1, 3, 0] and n == [5] and bad == [0]
    assert np.array_equal(k2[1, 0, :5], k[2, 0, [0, 2, 5, 8, 9]]) and np.array_equal(k2[1, 0, 5:], k[1, 0, 5:])
