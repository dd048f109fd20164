"""GPU tier of the decode over a shared prefix (decode_shared) against its
restatement in 64 bits (oracle/cache.py, which derives the bounds)."""
import math

import numpy as np
import pytest
import torch

from oracle import cache

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
HALF = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8}


def _i32(dev, x):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _case(dev, seed, B, H, Hkv, D, P, ctx, dtype, poison=True, spare=3, extra=0, amp=1.0):
    """Pools, tables and lengths; slots that no sequence has hold NaN, spare table entries an invalid page."""
    rng = np.random.default_rng(seed)
    need = [-(-n // 16) for n in [P, *ctx]]
    pages = sum(need) + spare
    perm = rng.permutation(pages).astype(np.int32)
    prefix = np.full(max(1, need[0] + extra), -1 if extra else 0, np.int32)
    table = np.full((B, max(1, max(need[1:], default=0) + extra)), -1 if extra else 0, np.int32)
    prefix[:need[0]] = perm[:need[0]]
    at = need[0]
    for b, n in enumerate(need[1:]):
        table[b, :n] = perm[at:at + n]
        at += n
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    pools = []
    for _ in range(2):
        x = torch.randn((pages, Hkv, 16, D), generator=g, device=dev, dtype=TYPES[dtype])
        if poison:
            keep = torch.zeros(pages, 16, dtype=torch.bool)
            for n, ids in zip([P, *ctx], [prefix, *table]):
                for j in range(-(-n // 16)):
                    keep[int(ids[j]), :min(16, n - 16 * j)] = True
            x = torch.where(keep.to(dev)[:, None, :, None], x, torch.full_like(x, math.nan))
        pools.append(x)
    q = (torch.randn((B, H, D), generator=g, device=dev) * amp).to(TYPES[dtype])
    return q, *pools, torch.from_numpy(prefix).to(dev), _i32(dev, [P]), torch.from_numpy(table).to(dev), _i32(dev, ctx)


def _want(case, dtype):
    q, kp, vp, prefix, plen, table, ctx = case
    f = lambda t: t.cpu().double().numpy()
    return cache.decode_shared(f(q), f(kp), f(vp), prefix.cpu().numpy(), int(plen), table.cpu().numpy(),
                               ctx.tolist(), HALF[dtype])


def _check(got, want, dtype, tag=""):
    O, L = got
    o, l, to, tl = want
    assert O.dtype == TYPES[dtype] and L.dtype == torch.float32 and O.shape == o.shape and L.shape == l.shape
    eo = np.abs(O.cpu().double().numpy() - o)
    assert (eo <= to).all(), f"{tag} O: worst {np.nanmax(eo / to):.2f} of the bound, {np.isnan(eo).sum()} NaN"
    lg = L.cpu().double().numpy()
    empty = np.isneginf(l)
    assert np.array_equal(np.isneginf(lg), empty), tag
    el = np.abs(lg[~empty] - l[~empty])
    assert (el <= tl[~empty]).all(), f"{tag} L: worst {(el / tl[~empty]).max():.2f} of the bound"


CASES = [
    # B, H, Hkv, D, P, own lengths
    (1, 1, 1, 64, 1, [0]), (1, 1, 1, 128, 16, [1]), (2, 8, 2, 64, 63, [0, 5]), (3, 4, 4, 128, 64, [1, 16, 17]),
    (4, 8, 8, 64, 65, [300, 0, 2, 64]), (2, 32, 8, 128, 500, [33, 700]), (5, 6, 2, 128, 129, [1, 2, 3, 4, 5]),
    (9, 16, 4, 64, 1000, [40] * 9), (16, 32, 8, 128, 700, list(range(0, 160, 10))), (33, 4, 1, 64, 257, [7] * 33),
    (31, 36, 4, 128, 300, [9 * i % 50 for i in range(31)]), (70, 8, 2, 64, 333, [3 * i for i in range(70)]),
    (1, 128, 1, 128, 800, [20]), (3, 40, 2, 64, 2100, [100, 0, 17]), (2, 2, 1, 128, 0, [70, 0]), (2, 4, 2, 64, 15, [0, 0]),
    (40, 32, 8, 128, 70, [2] * 40), (300, 2, 1, 64, 90, [5 * i % 70 for i in range(300)]), (600, 4, 4, 128, 40, [i % 3 for i in range(600)]),
    (16, 2, 1, 64, 1500, [3] * 16), (17, 2, 1, 64, 1500, [40] * 16 + [2000]),
    (3, 40, 2, 128, 160, [333, 0, 17]), (64, 4, 4, 64, 515, [i % 33 for i in range(64)]), (128, 4, 4, 64, 300, [i % 120 for i in range(128)]),
    (1, 8, 8, 128, 0, [575]), (2, 3, 1, 64, 1151, [1, 0]), (512, 1, 1, 128, 17, [i % 160 for i in range(512)]),
]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("wide", [0, 80])   # short tables are walked in one launch, wide ones in chunks
@pytest.mark.parametrize("i", range(len(CASES)))
def test_matches_oracle(fa, dev, i, wide, dtype):
    B, H, Hkv, D, P, ctx = CASES[i]
    case = _case(dev, i, B, H, Hkv, D, P, ctx, dtype, extra=i % 3 + wide)
    got = fa.decode_shared(*case)
    _check(got, _want(case, dtype), dtype, f"case {CASES[i][:5]}")
    again = fa.decode_shared(*case)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


@pytest.mark.parametrize("P", [1, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 127, 128, 129, 191, 193, 255, 256, 257])
@pytest.mark.parametrize("wide", [0, 80])
@pytest.mark.parametrize("D,dtype", [(64, "bf16"), (128, "fp16")])
def test_prefix_lengths(fa, dev, P, D, dtype, wide):
    """The prefix ends at every place of a page, a tile and the ring of tiles."""
    case = _case(dev, P, 3, 8, 2, D, P, [5, 0, 31], dtype, extra=wide)
    _check(fa.decode_shared(*case), _want(case, dtype), dtype)


@pytest.mark.parametrize("B,H,Hkv,D,dtype", [(8, 32, 8, 128, "fp16"), (40, 32, 8, 128, "bf16"), (33, 8, 8, 64, "fp16"), (20, 32, 2, 64, "bf16")])
def test_long_prefix(fa, dev, B, H, Hkv, D, dtype):
    """Long enough for more than 64 tiles a workgroup in a table far wider than the prefix, and for splits of a few."""
    for P, extra in ((20000, 0), (9001, 700)):
        case = _case(dev, P, B, H, Hkv, D, P, [11 * b for b in range(B)], dtype, poison=False, extra=extra)
        q, kp, vp, prefix, plen, table, ctx = case
        some = [0, B // 2, B - 1]   # the oracle's time: some sequences
        got = fa.decode_shared(*case)
        sub = (q[some], kp, vp, prefix, plen, table[some], ctx[some])
        _check([x[some] for x in got], _want(sub, dtype), dtype, f"P {P}")


def test_many_tiles_a_workgroup(fa, dev):
    """32 KV heads and 300 query rows of each: one run of over 64 tiles, three row blocks."""
    case = _case(dev, 3, 300, 32, 32, 64, 10000, [b % 3 for b in range(300)], "fp16", poison=False)
    q, kp, vp, prefix, plen, table, ctx = case
    some = [0, 127, 128, 299]
    got = fa.decode_shared(*case)
    _check([x[some] for x in got], _want((q[some], kp, vp, prefix, plen, table[some], ctx[some]), "fp16"), "fp16")


@pytest.mark.parametrize("wide", [0, 80])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
def test_invalid_pages_and_lengths(fa, dev, D, dtype, wide):
    """An invalid own page or length makes its sequence NaN, an invalid prefix all of them."""
    ctx = [40, 40, 40, 0, 16]
    case = list(_case(dev, 4, 5, 8, 2, D, 200, ctx, dtype, spare=1, extra=wide))
    good = fa.decode_shared(*case)
    pages = case[1].shape[0]
    t = case[5].clone()
    t[0, 1], t[1, 2] = -1, pages
    c = case[6].clone()
    c[2] = 16 * t.shape[1] + 1
    c[4] = -1
    O, L = fa.decode_shared(*case[:5], t, c)
    for b in (0, 1, 2, 4):
        assert torch.isnan(O[b]).all() and torch.isnan(L[b]).all(), b
    assert torch.equal(O[3], good[0][3]) and torch.equal(L[3], good[1][3])
    for at, page in ((0, -5), (12, pages), (5, 2 ** 31 - 1)):
        p = case[3].clone()
        p[at] = page
        O, L = fa.decode_shared(*case[:3], p, *case[4:])
        assert torch.isnan(O).all() and torch.isnan(L).all(), (at, page)
    for n in (-1, 16 * case[3].numel() + 1, 2 ** 31 - 1):
        O, L = fa.decode_shared(*case[:4], _i32(dev, [n]), *case[5:])
        assert torch.isnan(O).all() and torch.isnan(L).all(), n
    p = case[3].clone()   # entries past the prefix are not looked at
    p[4:] = -1
    O, L = fa.decode_shared(*case[:3], p, _i32(dev, [64]), *case[5:])
    assert torch.isfinite(O).all() and torch.isfinite(L).all()


def test_no_prefix_is_the_paged_decode(fa, dev):
    """Of an empty prefix O and L are decode_paged's, within both bounds."""
    case = _case(dev, 5, 4, 8, 2, 128, 0, [100, 1, 0, 777], "fp16")
    got = fa.decode_shared(*case)
    _check(got, _want(case, "fp16"), "fp16")
    assert (got[0][2] == 0).all() and torch.isneginf(got[1][2]).all()


def test_prefix_in_the_own_pages(fa, dev):
    """The same keys shared, and as the start of every sequence's own pages: one result within the bounds."""
    case = _case(dev, 6, 6, 16, 4, 64, 160, [30, 1, 0, 64, 15, 16], "bf16")
    q, kp, vp, prefix, plen, table, ctx = case
    joined = torch.cat((prefix[:10].expand(6, 10), table), 1).contiguous()
    _check(fa.decode_shared(q, kp, vp, prefix, plen * 0, joined, ctx + 160), _want(case, "bf16"), "bf16")
    _check(fa.decode_shared(*case), _want(case, "bf16"), "bf16")


def test_sharp_and_large_scores(fa, dev):
    """Scores of hundreds: a few keys carry the weight, and the maximum moves along the keys."""
    for amp in (8.0, 60.0):
        case = _case(dev, 7, 4, 8, 2, 64, 700, [50, 0, 3, 100], "fp16", amp=amp)
        _check(fa.decode_shared(*case), _want(case, "fp16"), "fp16", f"amp {amp}")


def test_masked_by_minus_infinity(fa, dev):
    """Keys whose scores are -inf (their K holds infinities) have no weight, a whole tile of them included."""
    D, P = 64, 256
    q, kp, vp, prefix, plen, table, ctx = _case(dev, 8, 2, 4, 2, D, P, [16, 3], "fp16")
    q[..., 0] = q[..., 0].abs() + 0.5
    kp[prefix[:8].long(), :, :, 0] = -math.inf   # the first 128 keys
    kp[prefix[12].long(), :, 3:9, 0] = -math.inf
    O, L = fa.decode_shared(q, kp, vp, prefix, plen, table, ctx)
    f = lambda t: t.cpu().double().numpy()
    live = np.ones(P, bool)
    live[:128] = False
    live[12 * 16 + 3:12 * 16 + 9] = False
    for b in range(2):
        for h in range(4):
            k, v = (np.concatenate([cache.rows(f(x), prefix.cpu().numpy(), P, h // 2)[live],
                                    cache.rows(f(x), table[b].cpu().numpy(), int(ctx[b]), h // 2)]) for x in (kp, vp))
            o, l, _, to, tl, _ = cache.attend(f(q[b, h:h + 1]), k, v, HALF["fp16"])
            assert (np.abs(f(O[b, h]) - o[0]) <= to[0]).all() and abs(float(L[b, h]) - l[0]) <= tl[0]


def test_nan_stays_in_its_head(fa, dev):
    """A NaN in a key of the prefix, or in an own value, reaches every query that sees it and no other."""
    case = _case(dev, 9, 3, 8, 4, 64, 100, [20, 20, 20], "fp16")
    q, kp, vp, prefix, plen, table, ctx = case
    good = fa.decode_shared(*case)
    kp[int(prefix[2]), 1, 5, 7] = math.nan
    vp[int(table[2, 0]), 3, 4, 9] = math.nan
    O, L = fa.decode_shared(*case)
    hit = torch.zeros(3, 8, dtype=torch.bool, device=dev)
    hit[:, 2:4] = True
    assert torch.isnan(O[hit]).all() and torch.isnan(L[hit]).all()
    hit[2, 6:8] = True
    assert torch.isnan(O[2, 6:8, 9]).all()
    assert torch.equal(O[~hit], good[0][~hit]) and torch.equal(L[~hit], good[1][~hit])


def test_far_pages(fa, dev):
    """Pages past 2^31 values of a pool."""
    Hkv, D = 8, 128
    pages = (1 << 31) // (Hkv * 16 * D) + 40
    case = _case(dev, 10, 2, 16, Hkv, D, 150, [40, 9], "bf16", spare=0)
    q, kp, vp, prefix, plen, table, ctx = case
    n = kp.shape[0]
    far = []
    for x in (kp, vp):
        y = torch.empty(pages, Hkv, 16, D, dtype=x.dtype, device=dev)
        y[pages - n:] = x
        far.append(y)
    got = fa.decode_shared(q, *far, prefix + (pages - n), plen, table + (pages - n), ctx)
    want = fa.decode_shared(*case)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_graphs_replayed_in_turn(fa, dev):
    """Two captured calls that may share a workspace's memory, replayed with new lengths and queries, eager calls between."""
    side = torch.cuda.Stream()
    runs = []
    for seed, shape in ((11, (3, 8, 2, 64, 300, [50, 3, 0])), (12, (17, 32, 8, 128, 900, [5 * i for i in range(17)]))):
        case = _case(dev, seed, *shape, "fp16", poison=False)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            fa.decode_shared(*case)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = fa.decode_shared(*case)
        runs.append((case, graph, out))
    for i in range(4):
        for case, graph, out in runs:
            case[0].copy_(torch.randn_like(case[0]))
            case[4].fill_(17 * i + 1)
            case[6].clamp_(max=40 - 9 * i)
            graph.replay()
        for case, graph, out in runs:
            want = fa.decode_shared(*case)
            torch.cuda.synchronize()
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]), i
            _check(out, _want(case, "fp16"), "fp16")


def test_two_streams(fa, dev):
    cases = [_case(dev, 13 + i, 6, 16, 4, 128, 600 + 100 * i, [40, 0, 9, 100, 1, 64], "bf16") for i in range(2)]
    want = [fa.decode_shared(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(fa.decode_shared(*cases[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, want[i][0]) and torch.equal(b, want[i][1]) for a, b in got[i])


@pytest.mark.parametrize("B,H,Hkv,D,P", [(257, 1, 1, 64, 300), (301, 3, 1, 128, 130)])
def test_odd_batch_planned_on_the_device(fa, dev, B, H, Hkv, D, P):
    """More sequences than a wave plans, with an odd number of the prefix's parts: the chunks' table behind them lies on 16 bytes."""
    case = _case(dev, B, B, H, Hkv, D, P, [7 * i % 90 for i in range(B)], "bf16", extra=80)
    _check(fa.decode_shared(*case), _want(case, "bf16"), "bf16")


STEPS = np.array([0, 1, 2, 3, 4, 6, 8, 12]) / 8   # numbers that both types hold beside a power of two


def _huge_scores(case, b, qs):
    """The case with products of q and k far beyond 2^24, as rows of one KV head per b and query heads per (b, a): every value
    of a K row is b but the first, b f with f of STEPS; every value of a query is a but the first, which makes the products
    a b (D - 1) +- 8 f g with g the last place of the product in 32 bits, so that each is a number of 24 bits and any
    order of its sum is exact. Slots that no sequence has keep their NaN."""
    q, kp, vp = case[:3]
    D, dt = q.shape[-1], q.dtype
    rng = np.random.default_rng(3)
    f = torch.from_numpy(rng.choice(STEPS, (kp.shape[0], 16))).to(kp.device)
    k = torch.tensor(b, dtype=torch.float64, device=kp.device)[None, :, None, None].expand(kp.shape[0], -1, 16, D).clone()
    k[..., 0] *= f[:, None]
    kp.copy_(torch.where(torch.isnan(kp), kp.double(), k))
    for h in range(q.shape[1]):
        bh, a = b[h // len(qs)], qs[h % len(qs)]
        g = 2.0 ** (math.floor(math.log2(D * abs(a) * bh)) - 23)
        q[:, h] = a
        q[:, h, 0] = 8 * g / bh * (1 if h % 2 else -1)
        assert float(q[0, h, 1]) == a and abs(float(q[0, h, 0])) == 8 * g / bh
    return case


HUGE = {"fp16": ([1024.0, 16384.0], [512.0, 1023.0, -2047.0, -1024.0, 16384.0, 4096.0, -640.0, 8192.0]),
        "bf16": ([1024.0, 2.0 ** 45], [512.0, 1020.0, -2040.0, -2.0 ** 41, 1.5, 2.0 ** 20, -96.0, 2.0 ** 30])}


@pytest.mark.parametrize("B,P,ctx,wide", [(2, 200, [9, 0], 0), (2, 700, [50, 333], 80), (6, 700, [50, 0, 333, 5, 1, 17], 80),
                                          (17, 3000, [7 * i for i in range(17)], 80), (40, 257, [i % 30 for i in range(40)], 80)])
@pytest.mark.parametrize("D,dtype", [(64, "fp16"), (128, "fp16"), (64, "bf16"), (128, "bf16")])
def test_huge_scores(fa, dev, D, dtype, B, P, ctx, wide):
    """Scores (in units of log 2) of 2^17 to 2^33 in fp16 and to 2^90 in bf16, of both signs: the weights follow from the scores'
    differences. 16 to 320 query rows of a KV head: one launch, chunks, and tiles."""
    b, qs = HUGE[dtype]
    case = _huge_scores(_case(dev, B + P, B, 16, 2, D, P, ctx, dtype, extra=wide), b, qs)
    O, L = fa.decode_shared(*case)
    # weights of a prefix in tiles have the type's bits; the others' two terms keep more, within the same bound
    _check((O, L), _want_exact(case, HALF[dtype], HALF[dtype]), dtype, f"B {B}")


def _want_exact(case, half, p_half):
    """_want() of a case whose products of q and k the kernels have exactly."""
    q, kp, vp, prefix, plen, table, ctx = [x.cpu().double().numpy() for x in case]
    B, H, D = q.shape
    Hkv = kp.shape[1]
    G = H // Hkv
    want = [np.zeros((B, H, D)), np.zeros((B, H)), np.zeros((B, H, D)), np.zeros((B, H))]
    for b in range(B):
        P, n = int(plen[0]), int(ctx[b])
        for h in range(Hkv):
            g = slice(G * h, G * h + G)
            k, v = (np.concatenate([cache.rows(x, prefix, P, h), cache.rows(x, table[b, :-(-n // 16)], n, h)]) for x in (kp, vp))
            s = q[b, g] @ k.T
            assert np.array_equal(s.astype(np.float32), s)
            o, l, _, to, tl, _ = cache.attend_exact(s, v, half, p_half)
            for x, y in zip(want, (o, l, to, tl)):
                x[b, g] = y
    return want


def _climbing_scores(case):
    """Products of q and k that rise along a sequence's keys, prefix and then own, from below -A 256 to A 256, A from 1/16 to 512 and of
    both signs, with up to 16 beside that: multiples of 1/16 below 2^18, so each is a number of 24 bits and exact."""
    q, kp, vp, prefix, plen, table, ctx = case
    P, H, dev = int(plen), q.shape[1], q.device
    total = P + int(ctx.max())
    rng = np.random.default_rng(5)
    k0 = lambda at: torch.from_numpy(np.floor(at / total * 512) - 256).to(dev, kp.dtype)
    for ids, first, n in [(prefix, 0, P)] + [(t, P, int(n)) for t, n in zip(table, ctx)]:
        for j in range(-(-n // 16)):
            m = min(16, n - 16 * j)
            page = int(ids[j])
            kp[page, :, :m, 0] = k0(first + 16 * j + np.arange(m))
            kp[page, :, :m, 1] = torch.from_numpy(rng.integers(0, 256, (kp.shape[1], m))).to(dev, kp.dtype)
    q.zero_()
    scale = torch.tensor([64, -64, 1, -1 / 16, 512, -512, 0.25, 16], device=dev, dtype=q.dtype)
    q[..., 0] = scale[torch.arange(H, device=dev) % 8]
    q[..., 1] = 1 / 16
    return case


@pytest.mark.parametrize("B,H,Hkv,P,ctx,wide", [(2, 8, 1, 300, [20, 9], 0), (3, 8, 1, 2500, [300, 0, 77], 80), (40, 8, 2, 2500, [3 * i for i in range(40)], 80),
                                                (40, 8, 1, 9000, [i % 7 for i in range(40)], 0), (9, 32, 4, 700, [600 - i for i in range(9)], 80)])
@pytest.mark.parametrize("D,dtype", [(64, "fp16"), (128, "fp16"), (64, "bf16"), (128, "bf16")])
def test_climbing_scores(fa, dev, D, dtype, B, H, Hkv, P, ctx, wide):
    """The maximum moves along the keys, by less and by more than the weights' slack, from far scores over near ones to far ones,
    in rows side by side: one launch, chunks, and tiles."""
    case = _climbing_scores(_case(dev, P, B, H, Hkv, D, P, ctx, dtype, extra=wide))
    _check(fa.decode_shared(*case), _want_exact(case, HALF[dtype], HALF[dtype]), dtype, f"B {B}")


@pytest.mark.parametrize("top", [118, -110])
@pytest.mark.parametrize("B,H,Hkv,P,ctx,wide", [(2, 8, 2, 250, [200, 0], 0), (2, 8, 2, 20000, [3000, 70], 0), (40, 32, 8, 20000, [9 * i for i in range(40)], 80),
                                                (17, 4, 2, 130000, [5] * 17, 0), (1, 2, 1, 0, [131072], 0)])
@pytest.mark.parametrize("D", [64, 128])
def test_range_of_bf16(fa, dev, D, B, H, Hkv, P, ctx, wide, top):
    """V of 2^118 and 2^-110 in equal weights, in one launch, over chunks and over tiles: what up to 131072 of them add up to is past
    the range, O is V. Equal weights' sums are (n / 16 + 64) 2^-24 off, twice: 2^-10, below half a place of O."""
    q, kp, vp, prefix, plen, table, c = _case(dev, 3, B, H, Hkv, D, P, ctx, "bf16", poison=False, extra=wide)
    kp.zero_()
    sign = torch.where(torch.arange(D, device=dev) % 3 == 0, -1.0, 1.0)
    vp.copy_((sign * 2.0 ** top).expand_as(vp))
    O, L = fa.decode_shared(q, kp, vp, prefix, plen, table, c)
    assert torch.equal(O, (sign * 2.0 ** top).to(O.dtype).expand_as(O))
    n = (c + plen).double().cpu().numpy()
    want = np.log(n)[:, None]
    assert (np.abs(L.double().cpu().numpy() - want) <= (n[:, None] / 16 + 64) * 2.0 ** -24 + 2.0 ** -21 * want).all()


# ---------------------------------------------------------------------------
# The prefix in tiles: more than 32 query rows a KV head, tables too wide for one launch
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("P", [0, 1, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 127, 128, 129, 191, 193, 255, 256, 257, 319, 321])
@pytest.mark.parametrize("D,dtype", [(64, "bf16"), (128, "fp16")])
def test_tiles_prefix_lengths(fa, dev, P, D, dtype):
    """The prefix ends at every place of a page, a tile and the ring of tiles; an empty one too."""
    case = _case(dev, P, 12, 8, 2, D, P, [5, 0, 31] * 4, dtype, extra=80)
    got = fa.decode_shared(*case)
    _check(got, _want(case, dtype), dtype)
    again = fa.decode_shared(*case)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
def test_tiles_invalid_pages_and_lengths(fa, dev, D, dtype):
    """An invalid own page or length makes its sequence NaN, an invalid prefix all of them."""
    B, ctx = 40, [40, 40, 40, 0, 16] + [7] * 35
    case = list(_case(dev, 4, B, 8, 2, D, 200, ctx, dtype, spare=1, extra=80))
    good = fa.decode_shared(*case)
    pages = case[1].shape[0]
    t = case[5].clone()
    t[0, 1], t[1, 2] = -1, pages
    c = case[6].clone()
    c[2] = 16 * t.shape[1] + 1
    c[4] = -1
    O, L = fa.decode_shared(*case[:5], t, c)
    for b in (0, 1, 2, 4):
        assert torch.isnan(O[b]).all() and torch.isnan(L[b]).all(), b
    assert torch.isfinite(O[3]).all() and torch.isfinite(O[5:]).all() and torch.isfinite(L[5:]).all()
    t = case[5].clone()
    t[0, 1], t[1, 2] = -1, pages   # the lengths as they were: the rest keep their bits
    O, L = fa.decode_shared(*case[:5], t, case[6])
    assert torch.isnan(O[:2]).all() and torch.equal(O[2:], good[0][2:]) and torch.equal(L[2:], good[1][2:])
    for at, page in ((0, -5), (12, pages), (5, 2 ** 31 - 1)):
        p = case[3].clone()
        p[at] = page
        O, L = fa.decode_shared(*case[:3], p, *case[4:])
        assert torch.isnan(O).all() and torch.isnan(L).all(), (at, page)
    for n in (-1, 16 * case[3].numel() + 1, 2 ** 31 - 1):
        O, L = fa.decode_shared(*case[:4], _i32(dev, [n]), *case[5:])
        assert torch.isnan(O).all() and torch.isnan(L).all(), n
    p = case[3].clone()   # entries past the prefix are not looked at
    p[4:] = -1
    O, L = fa.decode_shared(*case[:3], p, _i32(dev, [64]), *case[5:])
    assert torch.isfinite(O).all() and torch.isfinite(L).all()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_tiles_no_keys(fa, dev, dtype):
    """Neither a prefix nor own tokens: O 0 and L -inf, beside sequences that have some."""
    case = _case(dev, 5, 40, 8, 2, 128, 0, [0, 100, 1, 0, 777] * 8, dtype, extra=80)
    got = fa.decode_shared(*case)
    _check(got, _want(case, dtype), dtype)
    assert (got[0][3] == 0).all() and torch.isneginf(got[1][3]).all()


def test_tiles_prefix_in_the_own_pages(fa, dev):
    """The same keys shared, and as the start of every sequence's own pages: one result within the bounds."""
    ctx = [30, 1, 0, 64, 15, 16] * 4
    case = _case(dev, 6, 24, 16, 4, 64, 160, ctx, "bf16", extra=80)
    q, kp, vp, prefix, plen, table, c = case
    joined = torch.cat((prefix[:10].expand(24, 10), table), 1).contiguous()
    _check(fa.decode_shared(q, kp, vp, prefix, plen * 0, joined, c + 160), _want(case, "bf16"), "bf16")
    _check(fa.decode_shared(*case), _want(case, "bf16"), "bf16")


@pytest.mark.parametrize("D,dtype", [(64, "fp16"), (128, "bf16")])
@pytest.mark.parametrize("amp", [8.0, 60.0])
def test_tiles_sharp_and_large_scores(fa, dev, amp, D, dtype):
    """Scores of hundreds: a few keys carry the weight, and the maximum moves along the keys by more than the weights' slack."""
    case = _case(dev, 7, 40, 8, 2, D, 1700, [50, 0, 3, 100] * 10, dtype, amp=amp, extra=80)
    _check(fa.decode_shared(*case), _want(case, dtype), dtype, f"amp {amp}")


@pytest.mark.parametrize("D,dtype", [(64, "fp16"), (128, "bf16")])
def test_tiles_masked_by_minus_infinity(fa, dev, D, dtype):
    """Keys whose scores are -inf have no weight: the first tiles, a page's part, the whole prefix of a KV head, every key of a row."""
    B, P = 40, 256
    q, kp, vp, prefix, plen, table, ctx = _case(dev, 8, B, 4, 2, D, P, [16, 3] * 20, dtype, extra=80)
    q[..., 0] = q[..., 0].abs() + 0.5
    live = np.ones((2, P), bool)
    live[0, :128] = live[0, 195:201] = False
    live[1] = False
    for h in range(2):
        for j in range(P):
            if not live[h, j]:
                kp[prefix[j // 16].long(), h, j % 16, 0] = -math.inf
    kp[table[2, 0].long(), 1, :, 0] = -math.inf   # sequence 2, KV head 1: all
    O, L = fa.decode_shared(q, kp, vp, prefix, plen, table, ctx)
    f = lambda t: t.cpu().double().numpy()
    for b in (0, 1, 2, 39):
        for h in range(4):
            if b == 2 and h >= 2:
                assert (O[b, h] == 0).all() and torch.isneginf(L[b, h])
                continue
            k, v = (np.concatenate([cache.rows(f(x), prefix.cpu().numpy(), P, h // 2)[live[h // 2]],
                                    cache.rows(f(x), table[b].cpu().numpy(), int(ctx[b]), h // 2)]) for x in (kp, vp))
            o, l, _, to, tl, _ = cache.attend(f(q[b, h:h + 1]), k, v, HALF[dtype])
            assert (np.abs(f(O[b, h]) - o[0]) <= to[0]).all() and abs(float(L[b, h]) - l[0]) <= tl[0]


@pytest.mark.parametrize("D,dtype", [(64, "fp16"), (128, "bf16")])
def test_tiles_nan_stays_in_its_head(fa, dev, D, dtype):
    """A NaN in a key or a value of the prefix, or in an own value, reaches every query that sees it and no other."""
    case = _case(dev, 9, 24, 8, 4, D, 100, [20] * 24, dtype, extra=80)
    q, kp, vp, prefix, plen, table, ctx = case
    good = fa.decode_shared(*case)
    kp[int(prefix[2]), 1, 5, 7] = math.nan
    vp[int(prefix[6]), 0, 3, 11] = math.nan
    vp[int(table[2, 0]), 3, 4, 9] = math.nan
    O, L = fa.decode_shared(*case)
    assert torch.isnan(O[:, 2:4]).all() and torch.isnan(L[:, 2:4]).all()
    assert torch.isnan(O[:, :2, 11]).all() and torch.isnan(O[2, 6:8, 9]).all()
    same = torch.ones(24, 8, D, dtype=torch.bool, device=dev)
    same[:, 2:4] = False
    same[:, :2, 11] = False
    same[2, 6:8, 9] = False
    assert torch.equal(O[same], good[0][same])
    keep = torch.tensor([0, 1, 4, 5, 6, 7], device=dev)
    assert torch.equal(L[:, keep], good[1][:, keep])


@pytest.mark.parametrize("few", [True, False])
def test_far_pages_of_chunks_and_tiles(fa, dev, few):
    """Pages past 2^31 values of a pool, in chunks and in tiles that pass the caches; the same call on a small pool gives its bits."""
    Hkv, D = 8, 128
    pages = (1 << 31) // (Hkv * 16 * D) + 200
    B = 2 if few else 20
    case = _case(dev, 10, B, 16, Hkv, D, 350, [40, 9] * (B // 2), "bf16", spare=0, extra=80)
    q, kp, vp, prefix, plen, table, ctx = case
    n = kp.shape[0]
    far = []
    for x in (kp, vp):
        y = torch.empty(pages, Hkv, 16, D, dtype=x.dtype, device=dev)
        y[pages - n:] = x
        far.append(y)
    shift = lambda t: torch.where(t >= 0, t + (pages - n), t)
    got = fa.decode_shared(q, *far, shift(prefix), plen, shift(table), ctx)
    want = fa.decode_shared(*case)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    _check(got, _want(case, "bf16"), "bf16")


def test_tiles_two_streams(fa, dev):
    cases = [_case(dev, 13 + i, 24, 16, 4, 128, 600 + 100 * i, [40, 0, 9, 100, 1, 64] * 4, "bf16", extra=80) for i in range(2)]
    want = [fa.decode_shared(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(fa.decode_shared(*cases[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, want[i][0]) and torch.equal(b, want[i][1]) for a, b in got[i])


def test_graphs_of_one_pool(fa, dev):
    """Captured calls, in tiles and in chunks, of one memory pool, so that their workspaces share memory, replayed in turn with new
    lengths and queries, eager calls between."""
    side = torch.cuda.Stream()
    runs, pool = [], None
    for seed, shape in ((11, (40, 8, 2, 64, 300, [50, 3, 0, 7] * 10)), (12, (3, 8, 2, 128, 900, [5, 80, 0])), (13, (24, 32, 8, 128, 900, [5 * i for i in range(24)]))):
        case = _case(dev, seed, *shape, "fp16", poison=False, extra=80)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            fa.decode_shared(*case)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            out = fa.decode_shared(*case)
        pool = graph.pool()
        runs.append((case, graph, out))
    for i in range(4):
        for case, graph, out in runs:
            case[0].copy_(torch.randn_like(case[0]))
            case[4].fill_(17 * i + 1)
            case[6].clamp_(max=40 - 9 * i)
            graph.replay()
        for case, graph, out in runs:
            want = fa.decode_shared(*case)
            torch.cuda.synchronize()
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]), i
            _check(out, _want(case, "fp16"), "fp16")


def _coherent_roundings(case):
    """Keys of two weights, e^(-a / sqrt(D)) and e^(-b / sqrt(D)) of the largest, one that the type rounds up by nearly half a step and
    one that it rounds down, with values that cancel: what P's rounding does to O adds up, and O's own does not hide it. The first
    slot of each page has the largest weight, which is 1 in every part, and no value."""
    q, kp, vp = case[:3]
    D, dt, dev = q.shape[-1], q.dtype, q.device
    steps = torch.arange(1, 128, dtype=torch.float64) / 32
    p = torch.exp(-steps / math.sqrt(D))
    off = (p.to(dt).double() - p) / p
    a, b = int(off.argmax()), int(off.argmin())
    kp.zero_(), vp.zero_(), q.zero_()
    q[..., 0] = 1
    kp[:, :, 1::2, 0], kp[:, :, 2::2, 0] = -float(steps[a]), -float(steps[b])
    sign = torch.where(torch.arange(D, device=dev) % 3 == 0, -1.0, 1.0).to(dt)
    vp[:, :, 1::2] = sign
    vp[:, :, 2::2] = sign * -float(8 * p[a] / (7 * p[b]))
    return case


def _one_term(case, want, b, n):
    """Whether O of sequence b, of n keys of page 0's kind, would pass the bounds if P were rounded to the type once."""
    q, kp, vp = case[:3]
    k, v = (x[0, 0].cpu().double().repeat(-(-n // 16), 1)[:n] for x in (kp, vp))
    s = k @ q[b, 0].cpu().double() / math.sqrt(q.shape[-1])
    e = torch.exp(s - s.max())
    o = (e.to(q.dtype).double() @ v / e.sum()).numpy()
    return (np.abs(o - want[0][b, 0]) <= 4 * want[2][b, 0]).any()


@pytest.mark.parametrize("B,P,ctx,wide", [(2, 160, [160, 0], 0), (2, 160, [160, 0], 80), (3, 4000, [320, 16, 0], 0), (40, 0, [320] * 40, 80)])
@pytest.mark.parametrize("D,dtype", [(64, "fp16"), (128, "fp16"), (64, "bf16"), (128, "bf16")])
def test_weights_keep_two_terms(fa, dev, D, dtype, B, P, ctx, wide):
    """P has two terms of the type, 22 bits in fp16 and 16 in bf16, in one launch, in chunks of a prefix, and in own pages."""
    case = _coherent_roundings(_case(dev, 3, B, 8, 2, D, P, ctx, dtype, poison=False, extra=wide))
    want = _want_exact(case, HALF[dtype], HALF[dtype] ** 2)
    assert not _one_term(case, want, 0, P + ctx[0])
    _check(fa.decode_shared(*case), want, dtype)
