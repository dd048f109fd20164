"""CPU tier of the MX KV cache: the oracle against the definition, the C ABI's
argument checks, and the refusals of the Python entry points."""
import ctypes as C

import numpy as np
import pytest
import torch

from oracle import mx

BITS = [4, 8]
A = 0x10000   # a fake, 16-byte aligned address: never dereferenced by validation


@pytest.mark.parametrize("bits,bf16", [(b, t) for b in BITS for t in (False, True)])
def test_every_value_is_rounded_to_the_nearest(bits, bf16):
    """All finite 16-bit values as rows: the scale is the smallest allowed, and no value of the
    block's grid is nearer than the one taken; codes come back as the same codes."""
    x = np.arange(65536, dtype=np.uint32).astype(np.uint16)
    x = x[np.isfinite(mx.to_f64(x, bf16))]
    x = x[:len(x) // 64 * 64].reshape(-1, 64)
    rng = np.random.default_rng(1)
    x = np.concatenate([x, rng.permutation(x.ravel()).reshape(x.shape)])
    codes, scales = mx.quantize(x, bits, bf16)
    f = mx.to_f64(x, bf16)
    amax = np.abs(f).reshape(len(x), -1, 32).max(-1)
    top = mx.TOP[bits, bf16]
    s = scales.astype(int)
    assert s.min() >= 1 and s.max() <= top
    assert ((amax <= mx.LIM[bits] * np.exp2(s - 127.0)) | (s == top)).all()
    assert ((amax > mx.LIM[bits] * np.exp2(s - 128.0)) | (s == 1)).all()
    unit = np.repeat(np.exp2(s - 127.0), 32, -1)
    vals = np.concatenate([-mx.grid(bits), mx.grid(bits)])
    got = mx.dequantize(codes, scales, bits)
    sub = slice(0, len(x), 7)   # against every value of the grid
    err = np.abs(f[sub, :, None] - vals * unit[sub, :, None]).min(-1)
    assert np.array_equal(np.abs(got[sub] - f[sub]), err)
    assert np.array_equal(mx.to_f64(mx.from_f64(got, bf16), bf16), got)   # exact in the rows' type
    again, _ = mx.quantize(mx.from_f64(got, bf16), bits, bf16)
    assert np.array_equal(mx.dequantize(*mx.quantize(mx.from_f64(got, bf16), bits, bf16), bits), got)
    assert again.shape == codes.shape


@pytest.mark.parametrize("bits,steps", [(4, [(0.25, 0), (0.75, 2), (2.5, 4), (3.5, 6), (5, 6), (7, 7), (-5, 14)]),
                                        (8, [(2.0 ** -10, 0), (3 * 2.0 ** -10, 2), (17, 0x58), (19, 0x5a),
                                             (464, 0x7e), (-464, 0xfe)])])
def test_ties_go_to_the_even_code(bits, steps):
    for v, code in steps:
        row = np.zeros(32)
        row[0], row[1] = v, (7.0 if bits == 4 else 464.0)   # scale 1
        codes, scales = mx.quantize(mx.from_f64(row, False), bits, False)
        assert scales[0] == 127 and codes[0] == code, (v, codes[0], scales[0])


@pytest.mark.parametrize("bits", BITS)
def test_non_finite_blocks(bits):
    row = np.ones(64)
    for x in (np.nan, np.inf, -np.inf):
        row[5] = x
        codes, scales = mx.quantize(mx.from_f64(row, False), bits, False)
        assert scales[0] == 255 and scales[1] != 255 and not codes[:32].any()
        back = mx.dequantize(codes, scales, bits)
        assert np.isnan(back[:32]).all() and (back[32:] == 1).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("is_v", [False, True])
def test_a_page_has_every_byte_once(capi, D, bits, is_v):
    n = mx.page_bytes(D, bits)
    assert capi.load().fa_mx_page_bytes(D, bits) == n
    offs = np.concatenate([mx.code_offsets(D, bits, is_v).ravel(), mx.scale_offsets(D, bits, is_v).ravel()])
    assert np.array_equal(np.sort(offs), np.arange(n))
    rng = np.random.default_rng(D + bits)
    codes = rng.integers(0, 16 if bits == 4 else 256, (3, 16, D)).astype(np.uint8)
    scales = rng.integers(0, 256, (3, 16, D // 32)).astype(np.uint8)
    c, s = mx.unpack_pages(mx.pack_pages(codes, scales, bits, is_v), D, bits, is_v)
    assert np.array_equal(c, codes) and np.array_equal(s, scales)


def _app(**kw):
    b = dict(k=A, v=A, pt=A, st=A, ln=0, kp=A, vp=A, bad=A, B=2, H=4, T=3, D=128, kb=4, vb=8, ps=16, maxp=10, np_=100)
    b.update(kw)
    return tuple(b.values())


@pytest.mark.parametrize("kw,code", [
    (dict(), "FA_OK"), (dict(T=0, k=0, v=0), "FA_OK"), (dict(ln=A), "FA_OK"), (dict(kb=8, vb=4), "FA_OK"),
    (dict(bad=0), "FA_ERR_NULL_POINTER"), (dict(k=0), "FA_ERR_NULL_POINTER"), (dict(vp=0), "FA_ERR_NULL_POINTER"),
    (dict(D=96), "FA_ERR_HEAD_DIM"), (dict(kb=16), "FA_ERR_MX_BITS"), (dict(vb=0), "FA_ERR_MX_BITS"),
    (dict(vb=5), "FA_ERR_MX_BITS"), (dict(T=-1), "FA_ERR_SEQ_LEN"), (dict(B=0), "FA_ERR_BATCH_HEADS"),
    (dict(ps=32), "FA_ERR_PAGE_SIZE"), (dict(maxp=0), "FA_ERR_MAX_PAGES"), (dict(np_=0), "FA_ERR_NUM_PAGES"),
    (dict(k=A + 8), "FA_ERR_ALIGNMENT"), (dict(kp=A + 8), "FA_ERR_ALIGNMENT"), (dict(bad=A + 2), "FA_ERR_ALIGNMENT"),
    (dict(H=70000), "FA_ERR_TOO_LARGE"), (dict(T=1 << 31), "FA_ERR_TOO_LARGE"),
    (dict(T=1 << 28), "FA_ERR_TOO_LARGE"), (dict(T=(1 << 28) - 32), "FA_OK"),
])
def test_validate_append_and_read(capi, kw, code):
    lib = capi.load()
    a = _app(**kw)
    assert lib.fa_validate_kv_append_mx(*a) == capi.STATUS[code]
    if code != "FA_OK":   # the calls themselves stop there, before any HIP call
        assert lib.fa_kv_append_mx(*a, 0, None) == capi.STATUS[code]
        k, v, pt, st, ln, kp, vp, bad = a[:8]
        assert lib.fa_kv_read_mx(kp, vp, pt, st, ln, k, v, bad, *a[8:], 1, None) == capi.STATUS[code]


def _dec(**kw):
    b = dict(q=A, kp=A, vp=A, pt=A, ctx=A, B=4, H=32, Hkv=8, D=128, kb=4, vb=4, ps=16, maxp=100, np_=1000, ws=A, o=A,
             lse=A)
    b.update(kw)
    return tuple(b.values())


@pytest.mark.parametrize("kw,code", [
    (dict(), "FA_OK"), (dict(lse=0), "FA_OK"), (dict(Hkv=32, kb=8), "FA_OK"), (dict(Hkv=1), "FA_OK"),
    (dict(ws=0, maxp=20), "FA_OK"), (dict(q=0), "FA_ERR_NULL_POINTER"), (dict(ws=0), "FA_ERR_NULL_POINTER"), (dict(o=0), "FA_ERR_NULL_POINTER"),
    (dict(D=32), "FA_ERR_HEAD_DIM"), (dict(Hkv=5), "FA_ERR_KV_HEADS"), (dict(Hkv=0), "FA_ERR_KV_HEADS"),
    (dict(kb=2), "FA_ERR_MX_BITS"), (dict(vb=16), "FA_ERR_MX_BITS"), (dict(B=0), "FA_ERR_BATCH_HEADS"),
    (dict(ps=8), "FA_ERR_PAGE_SIZE"), (dict(maxp=0), "FA_ERR_MAX_PAGES"), (dict(np_=0), "FA_ERR_NUM_PAGES"),
    (dict(ws=A + 4), "FA_ERR_ALIGNMENT"), (dict(lse=A + 2), "FA_ERR_ALIGNMENT"), (dict(o=A + 2), "FA_ERR_ALIGNMENT"),
    (dict(B=65536), "FA_ERR_TOO_LARGE"), (dict(B=65535, maxp=1 << 20), "FA_ERR_TOO_LARGE"),
    (dict(np_=1 << 31), "FA_ERR_TOO_LARGE"),
])
def test_validate_decode(capi, kw, code):
    lib = capi.load()
    a = _dec(**kw)
    assert lib.fa_validate_decode_mx(*a) == capi.STATUS[code]
    if code != "FA_OK":
        assert lib.fa_decode_paged_mx(*a, 0, None) == capi.STATUS[code]


def test_sizes_and_strings(capi):
    lib = capi.load()
    assert [lib.fa_mx_page_bytes(D, b) for D in (64, 128) for b in (4, 8)] == [544, 1056, 1088, 2112]
    assert lib.fa_mx_page_bytes(96, 4) == lib.fa_mx_page_bytes(128, 2) == 0
    assert lib.fa_status_str(capi.STATUS["FA_ERR_MX_BITS"]) == b"k_bits and v_bits must be 4 or 8"
    assert lib.fa_decode_mx_workspace_floats(4, 32, 8, 128, 100) > 0
    assert lib.fa_decode_mx_workspace_floats(4, 32, 5, 128, 100) == 0
    assert lib.fa_decode_mx_workspace_floats(4, 32, 8, 128, 0) == 0
    # the workspace grows with a batch that fills the chip by itself only by the table's four words a
    # sequence
    assert (lib.fa_decode_mx_workspace_floats(10000, 32, 8, 128, 2000) - 4 * 5000 ==
            lib.fa_decode_mx_workspace_floats(5000, 32, 8, 128, 2000) <= 1 << 24)


def test_refusals_of_host_tensors(fa):
    kp, vp = fa.kv_pools_mx(4, 2, 64, 4, 8, device="cpu")
    assert kp.shape == (4, 2, 544) and vp.shape == (4, 2, 1056) and kp.dtype == torch.uint8
    x = torch.zeros(1, 2, 3, 64, dtype=torch.half)
    i32 = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="must be CUDA tensors"):
        fa.kv_append_mx(x, x, kp, vp, i32[None], i32)
    with pytest.raises(RuntimeError, match="must be CUDA tensors"):
        fa.kv_read_mx(kp, vp, i32[None], i32, 3)
    with pytest.raises(RuntimeError, match="must be CUDA tensors"):
        fa.decode_paged_mx(x[:, :, 0], kp, vp, i32[None], i32)
    with pytest.raises(RuntimeError, match="64 or 128 and 4 or 8"):
        fa.kv_pools_mx(4, 2, 96, device="cpu")
    with pytest.raises(RuntimeError, match="64 or 128 and 4 or 8"):
        fa.kv_pools_mx(4, 2, 64, 4, 16, device="cpu")
    with pytest.raises(RuntimeError, match="dtype must be"):
        fa.kv_read_mx(kp, vp, i32[None], i32, 3, dtype=torch.float32)


def test_chunk_plan_fits_its_grid(capi):
    """The grid and the workspace are sized from B * max_pages; whatever the lengths (any total up to
    that), the chunks that the device cuts fit them: at most `most` and one a sequence, of cut
    sequences at most `most` and one a cut sequence."""
    import random
    lib = capi.load()
    r = random.Random(3)
    most = C.c_int64()
    for _ in range(3000):
        B = r.choice([1, 2, 3, 8, 60, 64, 65, 200, 256, 300, 1000])
        Hkv = r.choice([1, 2, 4, 8, 32, 128])
        H = Hkv * r.choice([1, 4, 20, 64])
        maxp = int(2 ** r.uniform(0, 14))
        lens = [min(maxp, int(2 ** r.uniform(0, 14)) - 1) for _ in range(B)]
        Cp = lib.fa_probe_mx_chunks(B, H, Hkv, maxp, sum(lens), C.byref(most))
        assert Cp >= min(16, max(1, sum(lens)))
        cut = [-(-p // Cp) if Cp == 16 else (2 * p + Cp) // (2 * Cp) for p in lens]
        if most.value == 0:   # one launch: a sequence is one chunk
            assert Cp >= max(lens)
            cut = [1] * B
        assert sum(max(1, n) for n in cut) <= most.value + B
        cuts = [n for n in cut if n > 1]
        assert sum(cuts) <= most.value + min(B, most.value) < 1 << 15 and len(cuts) <= min(B, most.value)
        assert (lib.fa_decode_mx_workspace_floats(B, H, Hkv, 64, maxp) > 0) == (most.value > 0)
    assert lib.fa_probe_mx_chunks(1, 4, 3, 10, 5, None) == lib.fa_probe_mx_chunks(1, 4, 4, 10, 11, None) == 0


@pytest.mark.parametrize("kw", [dict(B=0), dict(B=65536), dict(H=0), dict(H=65544), dict(Hkv=0), dict(Hkv=5), dict(D=96),
                                dict(D=32), dict(D=0), dict(maxp=0), dict(maxp=1 << 27), dict(B=65535, maxp=1 << 20)])
def test_no_workspace_for_sizes_that_are_refused(capi, kw):
    lib = capi.load()
    a = _dec(**kw)
    B, H, Hkv, D, maxp = a[5], a[6], a[7], a[8], a[12]
    assert lib.fa_validate_decode_mx(*a) != capi.STATUS["FA_OK"]
    assert lib.fa_decode_mx_workspace_floats(B, H, Hkv, D, maxp) == 0


@pytest.mark.parametrize("bits,bf16", [(b, t) for b in BITS for t in (False, True)])
def test_quantised_rows_are_fixed_points(bits, bf16):
    """What a page holds, quantised again, has the same codes under the same scales: a block's largest
    value stays above half the scale's limit where a smaller scale could be taken."""
    x = np.arange(65536, dtype=np.uint32).astype(np.uint16)
    x = x[np.isfinite(mx.to_f64(x, bf16))]
    rng = np.random.default_rng(2)
    x = np.concatenate([x[:len(x) // 64 * 64], rng.permutation(x)[:len(x) // 64 * 64]]).reshape(-1, 64)
    codes, scales = mx.quantize(x, bits, bf16)
    again, scales2 = mx.quantize(mx.from_f64(mx.dequantize(codes, scales, bits), bf16), bits, bf16)
    assert np.array_equal(again, codes) and np.array_equal(scales2, scales)
