"""Measured cases of the microscaled (MX) KV cache: rows quantised into pages, read back, and attended by a decode step.

A cache in MX pages holds each K or V row as 4-bit (E2M1) or 8-bit (E4M3) values; blocks of 32 values along the head
dimension share a power-of-two scale of one byte. K and V pools are uint8 [num_pages, H_kv, page_bytes], and a page holds
16 tokens of one head: first the values' bytes in the order that the decode's lanes read them (_offsets), then the scales.

Four kinds of pass:

  append  new K/V rows quantised into the pages (kv_append_mx), and what those rows now hold, read back (kv_read_mx)
  read    a run of tokens of each sequence read back from its pages as fp16 or bf16 rows (kv_read_mx)
  decode  one query token per sequence over its pages (decode_paged_mx)
  step    one generated token as a server runs it: its K/V row appended, then the decode over the longer context

Sizes are the framework's own benchmark and test shapes, and generic ones of the same ranges.
"""
import importlib.util
import math
import pathlib
import random
import sys

import torch

own = False

DEV = "cuda"
PAGE = 16
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _fa():
    """The package directory has a hyphen in its name, so it is imported by its path."""
    name = "flashattn_cuda_amd"
    if name not in sys.modules:
        pkg = pathlib.Path(__file__).resolve().parent.parent / "flashattn-cuda_amd"
        spec = importlib.util.spec_from_file_location(name, pkg / "__init__.py", submodule_search_locations=[str(pkg)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return sys.modules[name]


def listed():
    return [
        # One generated token of eight conversations written to the cache: bound by latency.
        dict(name="append_token", kind="append", dtype="bf16", B=8, Hkv=8, D=128, T=1, kb=4, vb=4, lo=200, hi=4000, mix=5),
        # The prompts of a small batch of a grouped-query model, padded to an odd length; keys in 8 bits, values in 4.
        dict(name="append_prompts_k8v4", kind="append", dtype="bf16", B=2, Hkv=8, D=128, T=1777, kb=8, vb=4, lo=0, hi=0,
             mix=3),
        # The largest prompt batch of the benchmark, multi-head K/V.
        dict(name="append_prompts_large", kind="append", dtype="fp16", B=4, Hkv=16, D=128, T=4096, kb=4, vb=4, lo=0, hi=0,
             mix=4),
        # A reused prefix of a few conversations taken out of the cache for a prompt pass; starts inside pages.
        dict(name="read_prefix_d64", kind="read", dtype="fp16", B=4, Hkv=8, D=64, T=700, kb=8, vb=8, lo=3, hi=500, mix=7),
        # One long conversation read back whole.
        dict(name="read_long", kind="read", dtype="bf16", B=1, Hkv=8, D=128, T=32000, kb=4, vb=4, lo=0, hi=0, mix=1),
        # The smallest decode: a short context of a small model, bound by latency.
        dict(name="decode_short", kind="decode", dtype="fp16", B=1, H=8, Hkv=8, D=64, kb=4, vb=4, lo=130, hi=130, mix=1),
        # A serving step of a grouped-query model: eight conversations, the new token's row appended first.
        dict(name="step_gqa", kind="step", dtype="bf16", B=8, H=32, Hkv=8, D=128, kb=4, vb=4, lo=200, hi=4000, mix=5),
        # One user's long conversation: a single sequence, bound by how much of the chip it can use.
        dict(name="decode_one_long", kind="decode", dtype="fp16", B=1, H=32, Hkv=8, D=128, kb=4, vb=4, lo=32000, hi=32000,
             mix=1),
        # A ragged serving batch with keys in 8 bits and values in 4.
        dict(name="decode_batch_k8v4", kind="decode", dtype="bf16", B=24, H=32, Hkv=8, D=128, kb=8, vb=4, lo=300, hi=16000,
             mix=9),
        # A batch of a model with 64-wide heads, the whole cache in 8 bits.
        dict(name="decode_batch_d64", kind="decode", dtype="fp16", B=48, H=16, Hkv=4, D=64, kb=8, vb=8, lo=1000, hi=12000,
             mix=2),
        # One KV head for all query heads over a very long document: nothing but the length can be split.
        dict(name="decode_mqa_long", kind="decode", dtype="fp16", B=1, H=32, Hkv=1, D=128, kb=4, vb=4, lo=131072, hi=131072,
             mix=1),
        # The benchmark's decode batch: 32 sequences of up to 32768 tokens, multi-head K/V, bound by memory.
        dict(name="decode_batch_long", kind="decode", dtype="fp16", B=32, H=32, Hkv=32, D=128, kb=4, vb=4, lo=512, hi=32768,
             mix=5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "read", "decode", "decode", "decode", "step"])
    while True:
        c = dict(kind=kind, dtype=rng.choice(["fp16", "bf16"]), B=_log(rng, 1, 48), D=rng.choice([64, 128]),
                 kb=rng.choice([4, 4, 8]), vb=rng.choice([4, 4, 8]), mix=rng.randrange(1000))
        if kind in ("append", "read"):
            c.update(Hkv=rng.choice([1, 2, 4, 8, 16]), T=_log(rng, 1, 4096) if kind == "append" else _log(rng, 30, 32000))
            c["lo"] = rng.choice([0, _log(rng, 1, 4000)])
            c["hi"] = c["lo"] * rng.choice([1, 2])
        else:
            c["H"] = rng.choice([4, 8, 16, 32])
            c["Hkv"] = max(1, c["H"] // rng.choice([1, 2, 4, 8, 32]))
            c["lo"] = _log(rng, 40, 32000)
            c["hi"] = min(131072, c["lo"] * rng.choice([1, 4, 16]))
        if work(c)["bytes"] <= (2.6e8 if kind in ("append", "read") else 2e9):
            return c


def _lens(case):
    """Context lengths (decode, step) or first positions (append, read): part of the case, not of its inputs."""
    r = random.Random(case["mix"])
    return [r.randint(case["lo"], case["hi"]) for _ in range(case["B"])]


def _rows(case):
    """Rows of each sequence that an append or a read covers: the longest has T."""
    r = random.Random(case["mix"] + 1)
    T = case["T"]
    return [T] + [r.randint(max(1, T // 3), T) for _ in range(case["B"] - 1)]


# ---------------------------------------------------------------------------
# The format
# ---------------------------------------------------------------------------
def _page_bytes(D, bits):
    return PAGE * D * bits // 8 + PAGE * D // 32


def _offsets(D, bits, value):
    """Byte offsets within a page of each token's value bytes [16, D * bits / 8] (byte j of a row holds its values 2j and
    2j + 1, the first in the low half, or its value j) and of its scales [16, D / 32]."""
    row = D * bits // 8
    t = torch.arange(PAGE)[:, None]
    j = torch.arange(row)[None]
    blk = torch.arange(D // 32)[None]
    if not value:
        # K: token rows; a row of 128 bytes is kept as two planes of 16-byte pieces, one piece of every quarter row each.
        codes = (j % 32) // 16 * 1024 + (t * 4 + j // 32) * 16 + j % 16 if row == 128 else t * row + j
        scales = PAGE * row + t * (D // 32) + blk
    else:
        # V: groups of four tokens, and in a group the sixteenths of the rows, the four tokens' pieces side by side (two
        # planes of token pairs where the pieces are 8 bytes long).
        w = row // 16
        cell = t // 4 * 16 + j // w
        codes = t % 4 // 2 * 1024 + cell * 16 + t % 2 * 8 + j % w if w == 8 else cell * 4 * w + t % 4 * w + j % w
        scales = PAGE * row + blk * PAGE + t
    return codes.to(DEV), scales.to(DEV)


def _top_scale(dtype, bits):
    """The largest scale code whose largest value is finite in the rows' type."""
    return {("fp16", 4): 140, ("fp16", 8): 134, ("bf16", 4): 252, ("bf16", 8): 246}[dtype, bits]


def _pow2(code):
    """2^(code - 127), from the code's place in a 32-bit number."""
    return (code.to(torch.int32) << 23).view(torch.float32)


def _quantize(x, dtype, bits):
    """Rows [..., D] to value bytes [..., D * bits / 8] and scale codes [..., D / 32], in 32 bits. Division by a power of
    two is exact, and so is everything else but the one rounding."""
    D = x.shape[-1]
    blocks = x.float().unflatten(-1, (D // 32, 32))
    amax = blocks.abs().amax(-1)
    lim, top, low, mant = (7.0, 6.0, 0, 1) if bits == 4 else (464.0, 448.0, -6, 3)
    m, e = torch.frexp(amax / lim)   # amax / lim = m 2^e, m in [0.5, 1): the scale is 2^e, or 2^(e-1) where m is 0.5
    # amax / lim is rounded; whether it lies above a power of two is decided by products, which are exact
    code = (e + 127).clamp(1, _top_scale(dtype, bits))
    down = (amax <= lim * _pow2((code - 1).clamp(min=1))) & (code > 1)
    code = torch.where(down, code - 1, code)
    up = (amax > lim * _pow2(code)) & (code < _top_scale(dtype, bits))
    code = torch.where(up, code + 1, code)
    y = blocks / _pow2(code)[..., None]
    a = y.abs()
    ex = (torch.frexp(a)[1] - 1).clamp(min=low)
    ex = torch.where(a == 0, torch.full_like(ex, low), ex)
    step = _pow2(ex - mant + 127)
    q = (torch.round(a / step) * step).clamp(max=top)
    ex = torch.where(q >= 2 * _pow2(ex + 127), ex + 1, ex)   # rounded up to the next power of two
    step = _pow2(ex - mant + 127)
    n = (q / step).to(torch.int32)   # a normal value's 1 and fraction bits, a subnormal one's fraction bits
    c = torch.where(n >= (1 << mant), ((ex - low) << mant) + n, n)
    c = torch.where(torch.signbit(y), c + (8 if bits == 4 else 128), c)
    c = c.flatten(-2).to(torch.uint8)
    if bits == 4:
        c = c[..., 0::2] | (c[..., 1::2] << 4)
    ok = torch.isfinite(amax)
    c = torch.where(ok.repeat_interleave(c.shape[-1] // (D // 32), -1), c, torch.zeros_like(c))
    return c, torch.where(ok, code, torch.full_like(code, 255)).to(torch.uint8)


def _values(bits):
    """The value of each code."""
    i = torch.arange(16 if bits == 4 else 256, device=DEV)
    mant, low, sign = (1, 0, 8) if bits == 4 else (3, -6, 128)
    ex, fr = (i % sign) >> mant, i % (1 << mant)
    v = torch.where(ex > 0, (1 + fr / (1 << mant)) * _pow2(ex - 1 + low + 127), fr / (1 << mant) * _pow2(ex * 0 + low + 127))
    if bits == 8:
        v = torch.where(i % 128 == 127, torch.full_like(v, math.nan), v)
    return torch.where(i >= sign, -v, v)


def _dequantize(codes, scales, bits):
    """Value bytes and scale codes to rows in 32 bits (exact)."""
    if bits == 4:
        codes = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    v = _values(bits)[codes.int()].unflatten(-1, (scales.shape[-1], 32))
    s = torch.where(scales == 255, torch.full_like(scales, math.nan, dtype=torch.float32), _pow2(scales))
    return (v * s[..., None]).flatten(-2)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _keys(g, shape, dt):
    """Rows as a model's keys are: some channels carry larger values than the others."""
    x = torch.randn(shape, generator=g, device=DEV, dtype=dt)
    gain = torch.exp(0.7 * torch.randn(shape[-1], generator=g, device=DEV))
    return x * gain.to(dt)


def _fill(g, case, pages, bits, value):
    """A pool of quantised rows, made in runs of pages."""
    D, H = case["D"], case["Hkv"]
    codes, scales = _offsets(D, bits, value)
    pool = torch.empty(pages, H, _page_bytes(D, bits), dtype=torch.uint8, device=DEV)
    run_of = max(1, (1 << 26) // (H * PAGE * D))
    for p in range(0, pages, run_of):
        n = min(run_of, pages - p)
        shape, dt = (n, H, PAGE, D), DTYPES[case["dtype"]]
        x = torch.randn(shape, generator=g, device=DEV, dtype=dt) if value else _keys(g, shape, dt)
        c, s = _quantize(x, case["dtype"], bits)
        pool[p:p + n, :, codes.flatten()] = c.flatten(2)
        pool[p:p + n, :, scales.flatten()] = s.flatten(2)
    return pool


def _table(lens, g):
    """A page table whose pages are scattered over the pool, as a serving allocator leaves them."""
    need = [-(-n // PAGE) for n in lens]
    perm = torch.randperm(sum(need), generator=g, device=DEV).to(torch.int32)
    table = torch.zeros(len(lens), max(need), dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    return table, at


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    dt, kind, B, Hkv, D = DTYPES[case["dtype"]], case["kind"], case["B"], case["Hkv"], case["D"]
    lens = _lens(case)
    st = {"case": case}
    i32 = dict(dtype=torch.int32, device=DEV)
    if kind in ("append", "read"):
        rows = _rows(case)
        st["table"], pages = _table([p + n for p, n in zip(lens, rows)], g)
        st["start"], st["rows"] = torch.tensor(lens, **i32), torch.tensor(rows, **i32)
    else:
        st["table"], pages = _table(lens, g)
        st["ctx"] = torch.tensor(lens, **i32)
        st["q"] = torch.randn((B, case["H"], D), generator=g, device=DEV, dtype=dt)
    if kind == "append":   # a cache that other sequences use: zeros here, as only the new rows are read
        st["k_pool"], st["v_pool"] = (torch.zeros(pages, Hkv, _page_bytes(D, b), dtype=torch.uint8, device=DEV)
                                      for b in (case["kb"], case["vb"]))
    else:
        st["k_pool"], st["v_pool"] = _fill(g, case, pages, case["kb"], False), _fill(g, case, pages, case["vb"], True)
    if kind in ("append", "step"):
        T = case["T"] if kind == "append" else 1
        st["k"], st["v"] = _keys(g, (B, Hkv, T, D), dt), torch.randn((B, Hkv, T, D), generator=g, device=DEV, dtype=dt)
        if kind == "step":   # the new token is the context's last
            st["start"], st["rows"] = st["ctx"] - 1, torch.ones(B, **i32)
    return st


# ---------------------------------------------------------------------------
# The passes
# ---------------------------------------------------------------------------
def _places(st, T):
    """Page and slot of tokens start .. start + T of each sequence, and which of them the pass covers."""
    t = torch.arange(T, device=DEV)
    live = t[None] < st["rows"][:, None]
    pos = st["start"].long()[:, None] + t[None]
    page = torch.gather(st["table"].long(), 1, (pos // PAGE).clamp(max=st["table"].shape[1] - 1))
    return page, pos % PAGE, live


def _append(st):
    case = st["case"]
    page, slot, live = _places(st, st["k"].shape[2])
    heads = torch.arange(case["Hkv"], device=DEV)[None, :, None]
    for x, pool, bits, value in ((st["k"], st["k_pool"], case["kb"], False), (st["v"], st["v_pool"], case["vb"], True)):
        codes, scales = _offsets(case["D"], bits, value)
        c, s = _quantize(x.transpose(1, 2)[live], case["dtype"], bits)
        pool[page[live][:, None, None], heads, codes[slot[live]][:, None]] = c
        pool[page[live][:, None, None], heads, scales[slot[live]][:, None]] = s


def _read(st, T):
    case = st["case"]
    page, slot, live = _places(st, T)
    heads = torch.arange(case["Hkv"], device=DEV)[None, :, None]
    out = []
    for pool, bits, value in ((st["k_pool"], case["kb"], False), (st["v_pool"], case["vb"], True)):
        codes, scales = _offsets(case["D"], bits, value)
        c = pool[page[live][:, None, None], heads, codes[slot[live]][:, None]]
        s = pool[page[live][:, None, None], heads, scales[slot[live]][:, None]]
        x = torch.zeros(case["B"], T, case["Hkv"], case["D"], device=DEV)
        x[live] = _dequantize(c, s, bits)
        out.append(x.transpose(1, 2).to(DTYPES[case["dtype"]]).contiguous())
    return out


def _decode(st):
    case = st["case"]
    B, H, Hkv, D = case["B"], case["H"], case["Hkv"], case["D"]
    place = [_offsets(D, bits, value) for bits, value in ((case["kb"], False), (case["vb"], True))]
    o, l = torch.empty(B, H, D, device=DEV), torch.empty(B, H, device=DEV)
    for b, n in enumerate(_lens(case)):
        pages = st["table"][b, :-(-n // PAGE)].long()
        kv = []
        for pool, bits, (codes, scales) in ((st["k_pool"], case["kb"], place[0]), (st["v_pool"], case["vb"], place[1])):
            rec = pool[pages].transpose(0, 1)   # [Hkv, pages, bytes]
            c = rec[..., codes.flatten()].reshape(Hkv, -1, codes.shape[1])[:, :n]
            s = rec[..., scales.flatten()].reshape(Hkv, -1, scales.shape[1])[:, :n]
            kv.append(_dequantize(c, s, bits))
        k, v = kv
        s = torch.matmul(st["q"][b].float().reshape(Hkv, H // Hkv, D), k.transpose(1, 2).contiguous()) / math.sqrt(D)
        m = s.amax(-1, keepdim=True)
        p = torch.exp(s - m)
        z = p.sum(-1, keepdim=True)
        o[b] = (torch.matmul(p, v) / z).reshape(H, D)
        l[b] = (m + torch.log(z)).reshape(H)
    return [o.to(DTYPES[case["dtype"]]), l]


def run(st):
    case = st["case"]
    kind = case["kind"]
    if not own:
        if kind in ("append", "step"):
            _append(st)
        if kind in ("append", "read"):
            return _read(st, case["T"])
        return _decode(st)
    fa = _fa()
    k_pool, v_pool, table = st["k_pool"], st["v_pool"], st["table"]
    if kind == "append":
        fa.kv_append_mx(st["k"], st["v"], k_pool, v_pool, table, st["start"], st["rows"])
    elif kind == "step":
        fa.kv_append_mx(st["k"], st["v"], k_pool, v_pool, table, st["start"])   # the last of the rows attended below
    if kind in ("append", "read"):
        return fa.kv_read_mx(k_pool, v_pool, table, st["start"], case["T"], st["rows"], dtype=DTYPES[case["dtype"]])[:2]
    return fa.decode_paged_mx(st["q"], k_pool, v_pool, table, st["ctx"])


def work(case):
    """Bytes: 16-bit rows in, page bytes of the rows (written, or read), 16-bit rows out, the page table; products of the
    decode (two per value of K and of V and query head)."""
    D, Hkv, B = case["D"], case["Hkv"], case["B"]
    row = sum(_page_bytes(D, b) / PAGE for b in (case["kb"], case["vb"]))   # a token of one head, K and V
    if case["kind"] in ("append", "read"):
        n = sum(_rows(case))
        b = Hkv * n * row + 2 * 2 * Hkv * B * case["T"] * D + 4 * n / PAGE
        return {"bytes": b + (2 * 2 * Hkv * n * D if case["kind"] == "append" else 0), "flops": 0}
    n, H = sum(_lens(case)), case["H"]
    b = Hkv * n * row + 2 * 2 * B * H * D + 4 * B * H + 4 * n / PAGE + 4 * B
    if case["kind"] == "step":
        b += B * Hkv * (row + 2 * 2 * D)
    return {"bytes": b, "flops": 4 * H * n * D}


# ---------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------
def _grid(bits):
    """The format's values from 0 up, in 64 bits."""
    if bits == 4:
        return torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=DEV)
    v = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)]
    return torch.tensor(v[:-1], dtype=torch.float64, device=DEV)


def _nearest(x, dtype, bits):
    """What the rows x [..., D] hold once quantised: each value's nearest neighbour on the block's grid, a tie to the one
    of even index, values past the grid to its end."""
    grid = _grid(bits)
    blocks = x.double().reshape(*x.shape[:-1], -1, 32)
    lim = 7.0 if bits == 4 else 464.0
    edges = torch.tensor([lim * 2.0 ** (s - 127) for s in range(1, _top_scale(dtype, bits))], dtype=torch.float64, device=DEV)
    unit = torch.exp2((torch.bucketize(blocks.abs().amax(-1, keepdim=True), edges) + 1 - 127).double())
    y = blocks.abs() / unit
    mid = (grid[1:] + grid[:-1]) / 2
    below, above = torch.bucketize(y, mid), torch.bucketize(y, mid, right=True)   # they differ on a tie
    i = torch.where(below % 2 == 0, below, above)
    return (torch.sign(blocks) * grid[i] * unit).reshape(x.shape)


def _page_rows(pool, D, bits, value):
    """Pages [..., page_bytes] to rows [..., 16, D] in 64 bits: the bytes put in row order by reshapes."""
    lead, row = pool.shape[:-1], D * bits // 8
    data, sc = pool[..., :PAGE * row], pool[..., PAGE * row:]
    n = len(lead)

    def order(x, sizes, perm):
        return x.reshape(*lead, *sizes).permute(*range(n), *(n + i for i in perm)).reshape(*lead, PAGE, row)

    if value:
        if row == 128:   # [pair of a group, group, sixteenth, token of the pair, byte]
            data = order(data, (2, 4, 16, 2, 8), (1, 0, 3, 2, 4))
        else:            # [group, sixteenth, token, byte]
            data = order(data, (4, 16, 4, row // 16), (0, 2, 1, 3))
        sc = sc.reshape(*lead, D // 32, PAGE).transpose(-1, -2)
    else:
        if row == 128:   # [half of a quarter, token, quarter, byte]
            data = order(data, (2, 16, 4, 16), (1, 2, 0, 3))
        else:
            data = data.reshape(*lead, PAGE, row)
        sc = sc.reshape(*lead, PAGE, D // 32)
    data = data.long()
    if bits == 4:
        data = torch.stack((data % 16, data // 16), -1).reshape(*lead, PAGE, D)
    half = 8 if bits == 4 else 128
    grid = torch.cat((_grid(bits), torch.full((half - _grid(bits).numel(),), math.nan, dtype=torch.float64, device=DEV)))
    x = torch.cat((grid, -grid))[data]
    unit = torch.exp2(sc.double() - 127)
    return x * unit.repeat_interleave(32, -1)


def exact(case, seed):
    st = prepare(case, seed)
    kind, B, Hkv, D = case["kind"], case["B"], case["Hkv"], case["D"]
    bits = (case["kb"], case["vb"])
    f64 = dict(dtype=torch.float64, device=DEV)
    if kind in ("append", "read"):
        out = [torch.zeros(B, Hkv, case["T"], D, **f64) for _ in range(2)]
        for b, (p, n) in enumerate(zip(_lens(case), _rows(case))):
            for i, name in enumerate("kv"):
                if kind == "append":
                    out[i][b, :, :n] = _nearest(st[name][b, :, :n], case["dtype"], bits[i])
                else:
                    pages = st["table"][b, p // PAGE:-(-(p + n) // PAGE)].long()
                    rows = _page_rows(st[name + "_pool"][pages].transpose(0, 1), D, bits[i], i == 1)
                    out[i][b, :, :n] = rows.reshape(Hkv, -1, D)[:, p % PAGE:p % PAGE + n]
        return out
    H = case["H"]
    o, l = torch.empty(B, H, D, **f64), torch.empty(B, H, **f64)
    for b, n in enumerate(_lens(case)):
        pages = st["table"][b, :-(-n // PAGE)].long()
        for h in range(Hkv):
            kv = []
            for i, name in enumerate("kv"):
                x = _page_rows(st[name + "_pool"][pages, h], D, bits[i], i == 1).reshape(-1, D)[:n]
                if kind == "step":
                    x[n - 1] = _nearest(st[name][b, h, 0], case["dtype"], bits[i])
                kv.append(x)
            g = slice(h * (H // Hkv), (h + 1) * (H // Hkv))
            s = st["q"][b, g].double() @ kv[0].t().contiguous() / math.sqrt(D)
            l[b, g] = torch.logsumexp(s, 1)
            o[b, g] = torch.exp(s - l[b, g, None]) @ kv[1]
    return [o, l]
