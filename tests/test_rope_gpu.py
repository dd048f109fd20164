"""GPU tier of the rotary positions (rope, rope_backward, kv_append_rope) against
their restatement in 64 bits (oracle/rotary.py).

A value is off by
  - its factors cos and sin: the angle in turns is rounded to 32 bits once (at most
    2 pi 2^-26), the functions are within 2.2 units of 2^-24 and the scale's product
    rounds once more: 5 units of 2^-24 in all, of |x1| + |x2|; 7 are allowed;
  - a product and a fused product: 2 more of the same units;
  - the rounding to its type: half a step, or half of the smallest step.
"""
import math

import numpy as np
import pytest
import torch

from oracle import rotary

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
HALF = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8, "fp32": 2.0 ** -24}
LEAST = {"fp16": 2.0 ** -25, "bf16": 2.0 ** -134, "fp32": 2.0 ** -150}


def _f64(t):
    return t.detach().cpu().double().numpy()


def _check(y, x, positions, freqs, inter, scale, dtype, back=False, tag=""):
    """y, x tensors [B, h, N, D]; positions [B, N] or [N] in numpy."""
    f = _f64(freqs)
    p = np.asarray(positions)
    p = p[:, None, :] if p.ndim == 2 else p
    want = rotary.rotate(_f64(x), p, f, inter, scale, back)
    size = rotary.pair_size(_f64(x), f, inter)
    tol = 9 * 2.0 ** -24 * abs(scale) * size + HALF[dtype] * np.abs(want) * (1 + 2.0 ** -20) + LEAST[dtype]
    assert y.dtype == TYPES[dtype] and tuple(y.shape) == tuple(x.shape)
    err = np.abs(_f64(y) - want)
    assert (err <= tol).all(), f"{tag}: {(err > tol).sum()} off, worst {np.nanmax(err / tol):.2f} of the bound"
    if 2 * len(f) < x.shape[-1] and y.dtype == x.dtype:
        assert torch.equal(y[..., 2 * len(f):], x[..., 2 * len(f):])


def _rows(dev, seed, shape, dtype):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return torch.randn(shape, generator=g, device=dev, dtype=TYPES[dtype])


SHAPES = [(1, 1, 1, 1, 64), (1, 8, 8, 1, 128), (2, 4, 2, 3, 64), (3, 6, 1, 37, 128), (1, 32, 8, 65, 128),
          (2, 3, 3, 200, 64), (5, 5, 5, 33, 64), (1, 16, 16, 1030, 64)]


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("B,H,Hkv,N,D", SHAPES)
def test_rope(fa, dev, B, H, Hkv, N, D, inter, dtype):
    for R in (D, D // 2, 16):
        freqs, _ = fa.rope_frequencies(R, device=dev)
        Q, K = _rows(dev, N + R, (B, H, N, D), dtype), _rows(dev, N + R + 1, (B, Hkv, N, D), dtype)
        q, k = fa.rope(Q, K, freqs, interleaved=inter)
        assert q.is_contiguous() and k.is_contiguous()
        for y, x in ((q, Q), (k, K)):
            _check(y, x, np.arange(N), freqs, inter, 1.0, dtype, tag=f"R{R}")
        only, = fa.rope(Q, None, freqs, interleaved=inter)
        assert torch.equal(only, q)


@pytest.mark.parametrize("dtype,first", [("fp32", 0), ("fp32", 131072), ("fp32", 2 ** 31 - 40), ("fp32", -2 ** 31),
                                         ("fp16", 100000), ("bf16", 1000003)])
@pytest.mark.parametrize("inter", [False, True])
def test_far_positions(fa, dev, dtype, first, inter):
    """Angles keep their precision whatever the position, one row of positions a sequence."""
    B, H, N, D = 2, 3, 40, 64
    freqs, scale = fa.rope_frequencies(D, scaling="by_parts", factor=16.0, original_len=4096, device=dev)
    assert scale == pytest.approx(0.1 * math.log(16) + 1)
    pos = np.stack([first + np.arange(N), np.arange(N)[::-1] * 7 - 100]).astype(np.int32)
    Q, K = _rows(dev, 1, (B, H, N, D), dtype), _rows(dev, 2, (B, 1, N, D), dtype)
    tp = torch.from_numpy(pos).to(dev)
    for p, t in ((pos, tp), (pos[0], tp[0])):
        q, k = fa.rope(Q, K, freqs, t, interleaved=inter, scale=scale)
        _check(q, Q, p, freqs, inter, scale, dtype)
        _check(k, K, p, freqs, inter, scale, dtype)
    wide = torch.zeros(B, 2 * N, dtype=torch.int32, device=dev)   # positions by strides
    wide[:, ::2] = tp
    assert torch.equal(fa.rope(Q, None, freqs, wide[:, ::2], inter, scale)[0], fa.rope(Q, None, freqs, tp, inter, scale)[0])
    wide[:, :N] = tp
    assert torch.equal(fa.rope(Q, None, freqs, wide[:, :N], inter, scale)[0], fa.rope(Q, None, freqs, tp, inter, scale)[0])
    assert torch.equal(fa.rope(Q, None, freqs, tp[:1].expand(B, N), inter, scale)[0],
                       fa.rope(Q, None, freqs, tp[0], inter, scale)[0])


@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
@pytest.mark.parametrize("inter", [False, True])
def test_views(fa, dev, dtype, inter):
    """Views in any layout give what their contiguous copies give, bit for bit; outputs are contiguous."""
    B, H, Hkv, N, D = 2, 6, 2, 45, 64
    freqs, _ = fa.rope_frequencies(48, device=dev)
    qkv = _rows(dev, 3, (B, N, H + 2 * Hkv, D), dtype)
    flat = _rows(dev, 4, (B * N * H * D + 8 * D,), dtype)
    whole = _rows(dev, 5, (B, H, N, 2 * D), dtype)
    views = {
        "projection": qkv[:, :, :H].transpose(1, 2),
        "heads last": _rows(dev, 6, (N, B, H, D), dtype).permute(1, 2, 0, 3),
        "every other token": _rows(dev, 7, (B, H, 2 * N, D), dtype)[:, :, ::2],
        "one head for all": _rows(dev, 8, (B, 1, N, D), dtype).expand(B, H, N, D),
        "off by one value": flat[1:1 + B * H * N * D].view(B, H, N, D),
        "odd row stride": _rows(dev, 9, (B, H, N, D + 1), dtype)[..., :D],
        "every other value": whole[..., ::2],
        "a slice of wider rows": whole[..., D:],
    }
    K = qkv[:, :, H:H + Hkv].transpose(1, 2)
    for name, x in views.items():
        q, k = fa.rope(x, K, freqs, interleaved=inter)
        q2, k2 = fa.rope(x.contiguous(), K.contiguous(), freqs, interleaved=inter)
        assert q.is_contiguous() and torch.equal(q, q2) and torch.equal(k, k2), name
    assert torch.equal(fa.rope(qkv[:, :, :1].transpose(1, 2)[:, :, :1], None, freqs)[0],
                       fa.rope(qkv[:, :1, :1].transpose(1, 2).contiguous(), None, freqs)[0])


def test_packed(fa, dev):
    """Packed rows [H, total, D], positions that start anew at each sequence."""
    H, Hkv, D = 4, 2, 128
    lens = [1, 17, 0, 100, 64]
    total = sum(lens) + 5
    pos = np.concatenate([np.arange(n) for n in lens] + [np.zeros(5, np.int64)]).astype(np.int32)
    freqs, _ = fa.rope_frequencies(D, device=dev)
    q, k = _rows(dev, 1, (H, total, D), "bf16"), _rows(dev, 2, (Hkv, total, D), "bf16")
    a, b = fa.rope(q, k, freqs, torch.from_numpy(pos).to(dev))
    assert a.shape == q.shape and b.shape == k.shape
    _check(a[None], q[None], pos, freqs, False, 1.0, "bf16")
    _check(b[None], k[None], pos, freqs, False, 1.0, "bf16")
    g = fa.rope_backward(a, b, freqs, torch.from_numpy(pos).to(dev))
    _check(g[0][None], a[None], pos, freqs, False, 1.0, "bf16", back=True)


@pytest.mark.parametrize("d_in,d_out", [("fp32", "fp32"), ("fp32", "bf16"), ("fp32", "fp16"), ("fp16", "fp16"),
                                        ("bf16", "bf16")])
@pytest.mark.parametrize("inter", [False, True])
def test_backward(fa, dev, d_in, d_out, inter):
    """Gradients against the formula."""
    B, H, Hkv, N, D, scale = 2, 4, 2, 77, 128, 1.2
    freqs, _ = fa.rope_frequencies(96, base=500.0, device=dev)
    pos = np.random.default_rng(0).integers(-50, 4000, (B, N)).astype(np.int32)
    gq, gk = _rows(dev, 1, (B, N, H, D), d_in).transpose(1, 2), _rows(dev, 2, (B, Hkv, N, D), d_in)
    dq, dk = fa.rope_backward(gq, gk, freqs, torch.from_numpy(pos).to(dev), inter, scale, TYPES[d_out])
    _check(dq, gq, pos, freqs, inter, scale, d_out, back=True)
    _check(dk, gk, pos, freqs, inter, scale, d_out, back=True)
    same = fa.rope_backward(gq, gk, freqs, torch.from_numpy(pos).to(dev), inter, scale)
    assert same[0].dtype == gq.dtype


@pytest.mark.parametrize("inter", [False, True])
def test_backward_by_differences(fa, dev, inter):
    """<g, rope(x + e) - rope(x - e)> / 2 = <rope_backward(g), e> for the linear map rope, in 32 bits: a value
    of either side is off by 10 units of 2^-24 of its pair (the header's 9 and its rounding), so the sums over
    n values differ by no more than the sums of |g| and |e| times that; the step e is a power of two times a
    unit value, so that x + e and x - e are exact."""
    B, H, N, D, scale = 1, 2, 9, 64, 1.25
    freqs, _ = fa.rope_frequencies(32, device=dev)
    rng = np.random.default_rng(1)
    x = torch.from_numpy(rng.integers(-64, 64, (B, H, N, D)).astype(np.float32) / 16).to(dev)
    e = torch.from_numpy(rng.integers(-8, 9, (B, H, N, D)).astype(np.float32) / 16).to(dev)
    g = _rows(dev, 4, (B, H, N, D), "fp32")
    up, = fa.rope(x + e, None, freqs, None, inter, scale)
    down, = fa.rope(x - e, None, freqs, None, inter, scale)
    back, = fa.rope_backward(g, None, freqs, None, inter, scale)
    left = (_f64(g) * (_f64(up) - _f64(down)) / 2).sum()
    right = (_f64(back) * _f64(e)).sum()
    unit = 10 * 2.0 ** -24 * scale
    f = _f64(freqs)
    tol = unit * ((np.abs(_f64(g)) * (rotary.pair_size(_f64(x + e), f, inter) + rotary.pair_size(_f64(x - e), f, inter)) / 2).sum()
                  + (np.abs(_f64(e)) * rotary.pair_size(_f64(g), f, inter)).sum())
    assert abs(left - right) <= tol
    # one value at a time
    for at in [(0, 0, 0, 0), (0, 1, 8, 17), (0, 1, 5, 31), (0, 0, 3, 63)]:
        one = torch.zeros_like(x)
        one[at] = 0.5
        d = fa.rope(x + one, None, freqs, None, inter, scale)[0] - fa.rope(x - one, None, freqs, None, inter, scale)[0]
        tol = unit * (np.abs(_f64(g)) * (rotary.pair_size(_f64(x + one), f, inter) +
                                         rotary.pair_size(_f64(x - one), f, inter))).sum() + unit * np.abs(_f64(g)).sum()
        assert abs((_f64(g) * _f64(d)).sum() - _f64(back)[at]) <= tol


def test_special_values(fa, dev):
    """NaN and infinities stay in their pair; a NaN in dims past R stays where it is; fp16 overflows to infinity."""
    freqs, _ = fa.rope_frequencies(32, device=dev)
    x = torch.ones(1, 1, 4, 64, device=dev, dtype=torch.float16)
    x[0, 0, 1, 3] = math.nan
    x[0, 0, 2, 40] = math.nan
    x[0, 0, 3, 5] = math.inf
    y, = fa.rope(x, None, freqs)
    bad = ~torch.isfinite(y[0, 0])
    want = torch.zeros_like(bad)
    want[1, 3] = want[1, 19] = want[2, 40] = want[3, 5] = want[3, 21] = True
    assert torch.equal(bad, want)
    z, = fa.rope(torch.full_like(x, 60000.0), None, freqs, torch.zeros(4, dtype=torch.int32, device=dev), scale=2.0)
    assert torch.isinf(z[..., :32]).all() and (z[..., 32:] == 60000.0).all()


def test_many_sequences_and_heads(fa, dev):
    """More rows than a grid has blocks of a kind: 3000 sequences of one token, 300 heads."""
    freqs, _ = fa.rope_frequencies(64, device=dev)
    pos = torch.arange(3000, dtype=torch.int32, device=dev)[:, None]
    for B, H, N in ((3000, 3, 1), (1, 300, 2)):
        x = _rows(dev, B, (B, H, N, 64), "fp16")
        p = pos[:B] + torch.arange(N, dtype=torch.int32, device=dev)
        y, = fa.rope(x, None, freqs, p)
        _check(y, x, p.cpu().numpy(), freqs, False, 1.0, "fp16")


def test_offsets_past_32_bits(fa, dev):
    """Tokens more than 2^31 values apart."""
    freqs, _ = fa.rope_frequencies(128, device=dev)
    stride = (1 << 30) + 64
    big = torch.zeros(2 * stride + 128, dtype=torch.bfloat16, device=dev)
    x = big.as_strided((1, 1, 3, 128), (0, 0, stride, 1))
    x.copy_(_rows(dev, 1, (1, 1, 3, 128), "bf16"))
    y, = fa.rope(x, None, freqs)
    _check(y, x, np.arange(3), freqs, False, 1.0, "bf16")


# ---------------------------------------------------------------------------
# kv_append_rope
# ---------------------------------------------------------------------------
def _append_case(dev, seed, B, H, Hkv, T, D, dtype, start, slack=2):
    need = [-(-(s + T) // 16) + 1 for s in start]
    pages = sum(need) + slack
    perm = np.random.default_rng(seed).permutation(pages).astype(np.int32)
    table = np.zeros((B, max(need)), np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    pools = [_rows(dev, seed + i, (pages, Hkv, 16, D), dtype) for i in range(2)]
    qkv = _rows(dev, seed + 2, (B, T, H + 2 * Hkv, D), dtype)
    q, k, v = (x.transpose(1, 2) for x in qkv.split([H, Hkv, Hkv], 2))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    return q, k, v, pools, torch.from_numpy(table).to(dev), i32(start), i32


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("B,H,Hkv,T,D,start", [(1, 1, 1, 1, 64, [0]), (3, 8, 2, 1, 128, [0, 15, 333]), (2, 32, 8, 1, 128, [16, 4000]),
                                               (2, 4, 4, 37, 64, [3, 0]), (3, 6, 3, 130, 128, [0, 17, 31]), (4, 5, 1, 16, 64, [0, 8, 16, 1])])
def test_append_equals_rope_and_append(fa, dev, B, H, Hkv, T, D, start, inter, dtype):
    """One launch gives what rope and kv_append give, bit for bit, in the pools too."""
    q, k, v, pools, table, tstart, i32 = _append_case(dev, T + D, B, H, Hkv, T, D, dtype, start)
    freqs, _ = fa.rope_frequencies(D // 2, device=dev)
    rng = np.random.default_rng(T)
    for lens in (None, [int(x) for x in rng.integers(0, T + 1, B)], [T + 3] + [-2] * (B - 1)):
        for own_pos in (False, True):
            p0 = [s + (1000 * b + 7 if own_pos else 0) for b, s in enumerate(start)]
            pos = i32(p0)[:, None] + torch.arange(T, dtype=torch.int32, device=dev)
            n = [T] * B if lens is None else [min(max(x, 0), T) for x in lens]
            live = (torch.arange(T, device=dev) < i32(n)[:, None])[:, None, :, None]
            want_q, want_k = fa.rope(q, k, freqs, pos, inter, 1.5)
            want_q, want_k = want_q * live, want_k * live
            a, b = ([x.clone() for x in pools] for _ in range(2))
            tl = None if lens is None else i32(lens)
            want_bad = fa.kv_append(want_k.contiguous(), v.contiguous(), *a, table, tstart, tl)
            got = fa.kv_append_rope(q, k, v, *b, table, tstart, freqs, i32(p0) if own_pos else None, tl, inter, 1.5, want_k=True)
            assert torch.equal(got[0], want_q) and torch.equal(got[1], want_k) and torch.equal(got[2], want_bad)
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
            c = [x.clone() for x in pools]
            got = fa.kv_append_rope(q, k, v, *c, table, tstart, freqs, i32(p0) if own_pos else None, tl, inter, 1.5)
            assert len(got) == 2 and torch.equal(got[0], want_q) and torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])


def test_append_invalid_pages(fa, dev):
    """Tokens without a valid page are rotated and flagged; nothing else is written."""
    B, H, Hkv, T, D = 6, 4, 2, 20, 64
    q, k, v, pools, table, _, i32 = _append_case(dev, 5, B, H, Hkv, T, D, "fp16", [0] * B)
    start = i32([0, 0, -3, 16 * table.shape[1] - 5, 2 ** 31 - 8, 4])
    table[0, 1] = -1
    table[1, 0] = pools[0].shape[0]
    freqs, _ = fa.rope_frequencies(D, device=dev)
    pos = start.long()[:, None] + torch.arange(T, device=dev)
    want_q, _ = fa.rope(q, k, freqs, pos.clamp(max=2 ** 31 - 1).to(torch.int32))
    _, want_k = fa.rope(q, k, freqs, pos.clamp(max=2 ** 31 - 1).to(torch.int32))
    a, b = ([x.clone() for x in pools] for _ in range(2))
    want_bad = fa.kv_append(want_k, v.contiguous(), *a, table, start)
    got_q, got_k, bad = fa.kv_append_rope(q, k, v, *b, table, start, freqs, want_k=True)
    assert bad.tolist() == want_bad.tolist() == [1, 1, 1, 1, 1, 0]
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    near = [0, 1, 2, 3, 5]   # positions of sequence 4 pass 2^31
    assert torch.equal(got_q[near], want_q[near]) and torch.equal(got_k[near], want_k[near])
    _check(got_q[4:5], q[4:5], pos[4].cpu().numpy(), freqs, False, 1.0, "fp16")


def test_append_nothing(fa, dev):
    q, k, v, pools, table, start, i32 = _append_case(dev, 5, 2, 4, 2, 3, 64, "bf16", [0, 5])
    freqs, _ = fa.rope_frequencies(64, device=dev)
    before = [x.clone() for x in pools]
    got = fa.kv_append_rope(q[:, :, :0], k[:, :, :0], v[:, :, :0], *pools, table, start, freqs)
    assert got[0].shape == (2, 4, 0, 64) and got[1].tolist() == [0, 0]
    got = fa.kv_append_rope(q, k, v, *pools, table, start, freqs, new_lens=i32([0, -1]), want_k=True)
    assert not got[0].any() and not got[1].any() and got[2].tolist() == [0, 0]
    assert torch.equal(pools[0], before[0]) and torch.equal(pools[1], before[1])


def test_append_padding_may_hold_anything(fa, dev):
    q, k, v, pools, table, start, i32 = _append_case(dev, 6, 2, 4, 2, 9, 128, "fp16", [0, 5])
    freqs, _ = fa.rope_frequencies(128, device=dev)
    lens = i32([9, 4])
    other = [x.clone() for x in pools]
    a = fa.kv_append_rope(q, k, v, *pools, table, start, freqs, new_lens=lens, want_k=True)
    for x in (q, k, v):
        x[1, :, 4:] = math.nan
    b = fa.kv_append_rope(q, k, v, *other, table, start, freqs, new_lens=lens, want_k=True)
    assert all(torch.equal(x, y) for x, y in zip([*a, *pools], [*b, *other]))


def test_append_far_pages(fa, dev):
    """Pages past 2^31 values of a pool."""
    Hkv, D = 8, 128
    pages = (1 << 31) // (Hkv * 16 * D) + 3
    pools = [torch.empty(pages, Hkv, 16, D, dtype=torch.float16, device=dev) for _ in range(2)]
    q, k, v, _, _, _, i32 = _append_case(dev, 7, 2, 8, Hkv, 20, D, "fp16", [0, 0])
    table = i32([[pages - 1, pages - 3], [0, pages - 2]])
    freqs, _ = fa.rope_frequencies(D, device=dev)
    _, kr, bad = fa.kv_append_rope(q, k, v, *pools, table, i32([0, 0]), freqs, want_k=True)
    assert bad.tolist() == [0, 0]
    for b in range(2):
        for x, pool in ((kr, pools[0]), (v, pools[1])):
            rows = torch.cat([pool[int(p)] for p in table[b]], 1)[:, :20]
            assert torch.equal(rows, x[b])


def test_prompt_and_token_as_used(fa, dev):
    """A prompt pass and a token after it through the cache, against attention over rotated rows computed plainly in
    64 bits from the cached rows: positions in the cache are those of the decode's query."""
    B, H, Hkv, T, D = 2, 8, 2, 50, 64
    q, k, v, pools, table, start, i32 = _append_case(dev, 8, B, H, Hkv, T + 1, D, "fp16", [0, 0])
    freqs, _ = fa.rope_frequencies(D, device=dev)
    lens = i32([T, T - 13])
    qp, kp, bad = fa.kv_append_rope(q[:, :, :T], k[:, :, :T], v[:, :, :T], *pools, table, start, freqs, new_lens=lens, want_k=True)
    O, L = fa.forward(qp, kp, v[:, :, :T], causal=True)
    qt, bad2 = fa.kv_append_rope(q[:, :, T:], k[:, :, T:], v[:, :, T:], *pools, table, lens, freqs)
    assert not bad.any() and not bad2.any()
    o, l = fa.decode_paged(qt[:, :, 0].contiguous(), *pools, table, lens + 1)
    for b in range(B):
        n = int(lens[b])
        ka = np.concatenate([_f64(k[b, :, :n]), _f64(k[b, :, T:])], 1)
        va = np.concatenate([_f64(v[b, :, :n]), _f64(v[b, :, T:])], 1)
        qa = np.concatenate([_f64(q[b, :, :n]), _f64(q[b, :, T:])], 1)
        ka, qa = (rotary.rotate(x, np.arange(n + 1), _f64(freqs)) for x in (ka, qa))
        ka, va = (np.repeat(x, H // Hkv, 0) for x in (ka, va))
        s = qa @ ka.transpose(0, 2, 1) / 8
        s = np.where(np.tril(np.ones((n + 1, n + 1), bool)), s, -np.inf)
        e = np.exp(s - s.max(-1, keepdims=True))
        p = e / e.sum(-1, keepdims=True)
        # q and k each rounded once (2^-11 of |q| |k| / sqrt D a score at most), P and O once (2^-11)
        ds = 2 * 2.0 ** -11 * (np.abs(qa) @ np.abs(ka).transpose(0, 2, 1)).max(-1) / 8 + 1e-5
        tol = ((2 * ds + 2.0 ** -10)[..., None] * (p @ np.abs(va)) + 2.0 ** -11 * np.abs(p @ va) + 1e-5)
        got = np.concatenate([_f64(O[b, :, :n]), _f64(o[b])[:, None]], 1)
        assert (np.abs(got - p @ va) <= tol).all()


def test_graph_and_streams(fa, dev):
    """Captured calls replayed with new inputs, eager calls between; calls on a stream of their own."""
    B, H, Hkv, D = 3, 8, 2, 64
    q, k, v, pools, table, start, i32 = _append_case(dev, 9, B, H, Hkv, 1, D, "bf16", [40, 3, 100], slack=9)
    freqs, _ = fa.rope_frequencies(D, device=dev)
    Q = _rows(dev, 1, (2, 4, 70, 64), "fp16")

    def step(pools):
        a = fa.kv_append_rope(q, k, v, *pools, table, start, freqs)
        return [*a, *fa.rope(Q, Q, freqs), *fa.rope_backward(Q, Q, freqs)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(pools)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(pools)
    for i in range(4):
        Q.copy_(_rows(dev, 20 + i, Q.shape, "fp16"))
        for j, x in enumerate((q, k, v)):
            x.copy_(_rows(dev, 100 * i + j, x.shape, "bf16"))
        start.add_(1)
        mine = [x.clone() for x in pools]
        graph.replay()
        want = step(mine)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip([*out, *pools], [*want, *mine])), i


def test_step_graph(fa, dev):
    """A captured step, rope and its way back and the rotated append, replayed with new rows and positions."""
    q, k, v, pools, table, start, i32 = _append_case(dev, 8, 3, 8, 2, 1, 64, "bf16", [0, 15, 40])
    freqs, scale = fa.rope_frequencies(64, scaling="by_parts", factor=4.0, original_len=256, device=dev)
    pos = i32([7, 100, 41])

    def step(pools):
        rows = fa.rope(q, k, freqs, pos[:, None], scale=scale)
        back = fa.rope_backward(*rows, freqs, pos[:, None], scale=scale)
        return [*rows, *back, *fa.kv_append_rope(q, k, v, *pools, table, start, freqs, pos, scale=scale, want_k=True)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step([x.clone() for x in pools])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(pools)
    for i in range(4):
        q.copy_(torch.randn_like(q))
        v.copy_(torch.randn_like(v))
        start.add_(i)
        pos.add_(1000 * i)
        mine = [x.clone() for x in pools]
        graph.replay()
        want = step(mine)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip([*out, *pools], [*want, *mine])), i
