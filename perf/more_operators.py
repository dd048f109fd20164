"""Measured cases of what a rotary model needs around its attention and its paged cache: rotary positions, the fused append,
a prompt prefix shared by a batch, and a cache kept within a budget.

Six kinds of pass:

  rope      Q and K of one layer rotated by their positions (rope)
  rope_bwd  the gradients of rotated Q and K turned back to those of Q and K (rope_backward)
  append    q and K of new tokens rotated, K and V written into the paged cache (kv_append_rope)
  shared    one query token per sequence over a prefix that all sequences share and pages of its own (decode_shared)
  weights   the paged decode that also adds up the attention weight of every cached token (decode_paged_weights)
  evict     the newest and the heaviest tokens of each head packed into new pages (kv_evict)

Pools are [num_pages, H_kv, 16, D], page tables int32 [B, max_pages], lengths int32 [B]. Sizes are the framework's own
benchmark and test shapes, and generic ones of the same ranges.
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
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SIZE = {"fp16": 2, "bf16": 2, "fp32": 4}


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
        # The benchmark's shortest sequence, rotated before its attention: bound by latency.
        dict(name="rope_n1024", kind="rope", dtype="fp16", B=1, H=8, Hkv=8, N=1024, D=64, R=64, inter=False, token_major=False,
             long=False, mix=1),
        # One layer of the benchmark's largest batch: Q and K as the projection leaves them, token by token.
        dict(name="rope_train_d128", kind="rope", dtype="bf16", B=4, H=16, Hkv=16, N=4096, D=128, R=128, inter=False,
             token_major=True, long=False, mix=2),
        # The way back in training a grouped-query model on documents that start anew within a row: the backward's float32
        # gradients, half of the head rotated, neighbouring dims in pairs, frequencies stretched for a longer context.
        dict(name="rope_bwd_gqa", kind="rope_bwd", dtype="bf16", B=2, H=32, Hkv=8, N=2000, D=128, R=64, inter=True,
             token_major=False, long=True, mix=3),
        # One generated token of eight conversations: bound by latency.
        dict(name="append_token", kind="append", dtype="bf16", B=8, H=32, Hkv=8, T=1, D=128, R=128, inter=False, want_k=False,
             lo=200, hi=4000, mix=5),
        # The prompts of a small batch, padded to an odd length, out of one projection of q, k and v; K comes back for the
        # prompt's own attention.
        dict(name="append_prompts", kind="append", dtype="bf16", B=2, H=32, Hkv=8, T=1777, D=128, R=128, inter=False,
             want_k=True, lo=0, hi=0, mix=3),
        # A few conversations of a small model that share a short instruction.
        dict(name="shared_short_d64", kind="shared", dtype="fp16", B=4, H=8, Hkv=8, D=64, P=500, lo=1, hi=60, mix=4),
        # A serving batch of a grouped-query model under one long instruction of odd length.
        dict(name="shared_gqa", kind="shared", dtype="bf16", B=32, H=32, Hkv=8, D=128, P=7999, lo=50, hi=1500, mix=7),
        # Many questions about one long document.
        dict(name="shared_document", kind="shared", dtype="fp16", B=64, H=32, Hkv=8, D=128, P=32768, lo=20, hi=1000, mix=8),
        # A decode step that keeps count of what its tokens attend to.
        dict(name="weights_gqa", kind="weights", dtype="bf16", B=8, H=32, Hkv=8, D=128, lo=200, hi=4000, mix=5),
        # The same for a batch of long contexts, bound by memory.
        dict(name="weights_batch_long", kind="weights", dtype="fp16", B=16, H=32, Hkv=8, D=128, lo=2000, hi=32768, mix=6),
        # A small model's cache brought back to its budget after some tokens more.
        dict(name="evict_d64", kind="evict", dtype="fp16", B=4, Hkv=8, D=64, lo=300, hi=1100, keep=512, recent=64, mix=4),
        # Long prompts cut down to a budget before their answers are generated.
        dict(name="evict_prompts", kind="evict", dtype="bf16", B=8, Hkv=8, D=128, lo=6000, hi=32000, keep=4096, recent=256,
             mix=9),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "rope", "rope_bwd", "append", "append", "shared", "shared", "shared", "weights", "weights", "evict",
                       "evict"])
    while True:
        D = rng.choice([64, 128])
        H = rng.choice([4, 8, 16, 32])
        c = dict(kind=kind, dtype=rng.choice(["fp16", "bf16"]), B=_log(rng, 1, 48), H=H, Hkv=max(1, H // rng.choice([1, 2, 4, 8])),
                 D=D, mix=rng.randrange(1000))
        if kind in ("rope", "rope_bwd"):
            c.update(dtype=rng.choice(["fp16", "bf16", "bf16", "fp32"]), B=rng.choice([1, 1, 2, 4]), N=_log(rng, 60, 8192),
                     R=rng.choice([D, D, D // 2, D // 4]), inter=rng.random() < 0.4, token_major=rng.random() < 0.5,
                     long=rng.random() < 0.4)
        elif kind == "append":
            c.update(T=rng.choice([1, 1, _log(rng, 2, 4096)]), R=rng.choice([D, D, D // 2]), inter=rng.random() < 0.4)
            c.update(want_k=c["T"] > 1 and rng.random() < 0.5, lo=rng.choice([0, _log(rng, 1, 4000)]))
            c["hi"] = c["lo"] * rng.choice([1, 4])
        elif kind == "shared":
            c.update(P=_log(rng, 30, 32768), lo=_log(rng, 1, 1000))
            c["hi"] = c["lo"] * rng.choice([1, 4])
        else:
            c["lo"] = _log(rng, 40, 16000)
            c["hi"] = min(32768, c["lo"] * rng.choice([1, 2, 4]))
            if kind == "evict":
                c["keep"] = max(2, int(c["lo"] * rng.uniform(0.1, 1.1)))
                c["recent"] = rng.randint(0, c["keep"])
                del c["H"]
        w = work(c)
        if w["bytes"] <= 6e8 and w["flops"] <= 3.5e10:
            return c


def _ints(case, lo, hi, n, add=0):
    """Lengths and the like: part of the case, not of its inputs."""
    r = random.Random(case["mix"] + add)
    return [r.randint(lo, hi) for _ in range(n)]


def _lens(case):
    return _ints(case, case["lo"], case["hi"], case["B"])


def _rows(case):
    """New tokens of each sequence of an append: the longest has T."""
    T = case["T"]
    return [T] + _ints(case, max(1, T // 3), T, case["B"] - 1, 1)


def _randn(g, shape, dtype):
    return torch.randn(shape, generator=g, device=DEV, dtype=dtype)


def _pages(lens, g, first=0):
    """A page table whose pages are scattered over the pool, as a serving allocator leaves them, and their number."""
    need = [-(-n // PAGE) for n in lens]
    perm = torch.randperm(sum(need), generator=g, device=DEV).to(torch.int32) + first
    table = torch.zeros(len(lens), max(1, max(need)), dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    return table, at


def _freqs(case):
    """Radians per position: base 10000, or for a context eight times as long the slow half of them slowed down by that."""
    i = torch.arange(case["R"] // 2, dtype=torch.float64, device=DEV)
    f = 10000.0 ** (-2.0 * i / case["R"])
    return torch.where(f < f[f.numel() // 2], f / 8, f) if case.get("long") else f


def _positions(case):
    """Positions [B, N]: documents that start anew at places of the case's own, or rows of one long context."""
    N, B = case["N"], case["B"]
    if not case["long"]:
        return torch.arange(N, dtype=torch.int32, device=DEV).expand(B, N).contiguous()
    pos = torch.arange(N, dtype=torch.int32).repeat(B, 1)
    for b, cut in enumerate(_ints(case, 0, N - 1, B)):
        pos[b, cut:] -= cut
        pos[b, :cut] += 100000
    return pos.to(DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    kind, dt, B, D, Hkv = case["kind"], DTYPES[case["dtype"]], case["B"], case["D"], case["Hkv"]
    H = case.get("H", Hkv)
    st = {"case": case}

    def i32(x):
        return torch.tensor(x, dtype=torch.int32, device=DEV)

    if kind in ("rope", "rope_bwd"):
        N = case["N"]
        st["freqs"], st["positions"] = _freqs(case), _positions(case)
        st["scale"] = 0.1 * math.log(8.0) + 1.0 if case["long"] else 1.0
        dt_in = torch.float32 if kind == "rope_bwd" else dt
        for name, h in (("q", H), ("k", Hkv)):
            if case["token_major"]:
                st[name] = _randn(g, (B, N, h, D), dt_in).transpose(1, 2)
            else:
                st[name] = _randn(g, (B, h, N, D), dt_in)
        return st
    if kind == "append":
        T, starts, rows = case["T"], _lens(case), _rows(case)
        st["freqs"] = _freqs(case)
        qkv = _randn(g, (B, T, H + 2 * Hkv, D), dt)   # one projection's rows
        st["q"], st["k"], st["v"] = (x.transpose(1, 2) for x in qkv.split([H, Hkv, Hkv], 2))
        st["table"], n = _pages([s + r for s, r in zip(starts, rows)], g)
        st["start"], st["rows"] = i32(starts), i32(rows)
    elif kind == "shared":
        lens = _lens(case)
        st["lens"], st["prefix_len"] = i32(lens), i32([case["P"]])
        prefix, m = _pages([case["P"]], g)
        st["prefix"] = prefix[0].contiguous()
        st["table"], n = _pages(lens, g, m)
        st["q"] = _randn(g, (B, H, D), dt)
        n += m
    elif kind == "weights":
        lens = _lens(case)
        st["table"], n = _pages(lens, g)
        st["lens"], st["q"] = i32(lens), _randn(g, (B, H, D), dt)
        st["weights"] = _old_weights(case, st["table"], st["lens"], g)
    else:
        lens = _lens(case)
        st["table"], m = _pages(lens, g)
        st["new_table"], n = _pages([min(x, case["keep"]) for x in lens], g, m)
        wide = -(-case["keep"] // PAGE)
        st["new_table"] = torch.nn.functional.pad(st["new_table"], (0, wide - st["new_table"].shape[1]))
        st["lens"], st["first_new"] = i32(lens), m
        st["weights"] = _old_weights(case, st["table"], st["lens"], g)
        n += m
    st["k_pool"], st["v_pool"] = (_randn(g, (n, Hkv, PAGE, D), dt) for _ in range(2))
    return st


def _old_weights(case, table, lens, g):
    """Weights added up over earlier steps [B, H_kv, slots]: a few heavy tokens, many light ones, some of them alike."""
    n = table.shape[1] * PAGE
    w = torch.exp(2.5 * _randn(g, (case["B"], case["Hkv"], n), torch.float32))
    w = torch.where(w < 0.5, torch.floor(w * 64) / 64, w)
    return torch.where(torch.arange(n, device=DEV) < lens[:, None, None], w, torch.zeros((), device=DEV))


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------
def _rotated(x, positions, freqs, inter, scale):
    """x [B, h, T, D] by positions [B, T]: pairs (i, i + R/2), or neighbours, of the first R dims; in 32 bits, the angles in 64."""
    a = positions.double()[:, None, :, None] * freqs
    cos, sin = (torch.cos(a) * scale).float(), (torch.sin(a) * scale).float()
    R = 2 * freqs.numel()
    y = x.float()
    y1, y2 = (y[..., 0:R:2], y[..., 1:R:2]) if inter else (y[..., :R // 2], y[..., R // 2:R])
    z1, z2 = y1 * cos - y2 * sin, y2 * cos + y1 * sin
    z = torch.stack((z1, z2), -1).flatten(-2) if inter else torch.cat((z1, z2), -1)
    return torch.cat((z, y[..., R:]), -1)


def _rows_of(pool, table):
    """Rows [..., H_kv, pages * 16, D] of a page table in 32 bits."""
    x = pool[table.long()].float()               # [..., pages, H_kv, 16, D]
    x = x.transpose(-4, -3)
    return x.reshape(*x.shape[:-3], -1, x.shape[-1])


def _attend(s, v_parts, sizes, valid):
    """Softmax of scores s [B, H_kv, G, n] over the valid ones; products with V's parts; O, L and the weights."""
    s = torch.where(valid, s, torch.full((), -math.inf, device=DEV))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - m)
    z = p.sum(-1, keepdim=True)
    p = p / z
    o = 0
    for part, v in zip(p.split(sizes, -1), v_parts):
        o = o + v(part)
    return o, (m + torch.log(z)).squeeze(-1), p


def _plain(st):
    case = st["case"]
    kind, dt, B, D, Hkv = case["kind"], DTYPES[case["dtype"]], case["B"], case["D"], case["Hkv"]
    if kind == "rope":
        return [_rotated(st[x], st["positions"], st["freqs"], case["inter"], st["scale"]).to(dt) for x in "qk"]
    if kind == "rope_bwd":   # the transpose of the rotation: by the angle back, the dims past R as they are
        return [_rotated(st[x], -st["positions"], st["freqs"], case["inter"], st["scale"]).to(dt) for x in "qk"]
    if kind == "append":
        T = case["T"]
        t = torch.arange(T, device=DEV)
        pos = st["start"][:, None] + t
        live = t < st["rows"][:, None]
        qr, kr = (torch.where(live[:, None, :, None], _rotated(st[x], pos, st["freqs"], case["inter"], 1.0), 0.0).to(dt)
                  for x in "qk")
        b, i = torch.nonzero(live, as_tuple=True)
        p = pos[b, i].long()
        page, slot = st["table"][b, p // PAGE].long(), p % PAGE
        st["k_pool"][page, :, slot] = kr[b, :, i]
        st["v_pool"][page, :, slot] = st["v"][b, :, i]
        bad = torch.zeros(B, dtype=torch.int32, device=DEV)
        return [qr, *([kr] if case["want_k"] else []), bad, st["k_pool"], st["v_pool"]]
    n = st["table"].shape[1] * PAGE
    live = torch.arange(n, device=DEV) < st["lens"][:, None]              # [B, n]
    if kind == "evict":
        return _plain_evict(st, n, live)
    G = case["H"] // Hkv
    q = st["q"].float().reshape(B, Hkv, G, D) / math.sqrt(D)
    k, v = _rows_of(st["k_pool"], st["table"]), _rows_of(st["v_pool"], st["table"])   # [B, H_kv, n, D]
    s = torch.matmul(q, k.transpose(-1, -2).contiguous())
    if kind == "weights":
        o, lse, p = _attend(s, [lambda x: torch.matmul(x, v)], [n], live[:, None, None])
        w = st["weights"] + p.sum(2)
        return [o.reshape(B, -1, D).to(dt), lse.reshape(B, -1), w]
    m = st["prefix"].numel() * PAGE
    pk, pv = _rows_of(st["k_pool"], st["prefix"]), _rows_of(st["v_pool"], st["prefix"])   # [H_kv, m, D]
    ps = torch.matmul(q.transpose(0, 1).reshape(Hkv, B * G, D), pk.transpose(-1, -2).contiguous())
    ps = ps.reshape(Hkv, B, G, m).transpose(0, 1)
    valid = torch.cat(((torch.arange(m, device=DEV) < st["prefix_len"]).expand(B, m), live), 1)

    def prefix_product(x):   # [B, H_kv, G, m] with [H_kv, m, D]
        y = torch.matmul(x.transpose(0, 1).reshape(Hkv, B * G, m), pv)
        return y.reshape(Hkv, B, G, D).transpose(0, 1)

    o, lse, _ = _attend(torch.cat((ps, s), -1), [prefix_product, lambda x: torch.matmul(x, v)], [m, n], valid[:, None, None])
    return [o.reshape(B, -1, D).to(dt), lse.reshape(B, -1)]


def _plain_evict(st, n, live):
    case = st["case"]
    B, Hkv, keep = case["B"], case["Hkv"], case["keep"]
    slot = torch.arange(n, device=DEV)
    lens = st["lens"].long()
    newest = slot >= lens[:, None] - case["recent"]
    key = torch.where(newest[:, None], torch.full((), math.inf, device=DEV), st["weights"])
    key = torch.where(live[:, None], key, torch.full((), -1.0, device=DEV))
    first = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :keep]     # equal ones: the lowest slot first
    new_lens = torch.clamp(lens, max=keep)
    j = torch.arange(first.shape[-1], device=DEV)
    kept = torch.sort(torch.where(j < new_lens[:, None, None], first, n), dim=-1).values   # by slot; n: none
    kept = torch.nn.functional.pad(kept, (0, keep - kept.shape[-1]), value=n)
    there = kept < n
    old = torch.where(there, kept, 0)
    wide = st["new_table"].shape[1] * PAGE
    w = torch.where(there, torch.gather(st["weights"], 2, old), 0.0)
    w = torch.nn.functional.pad(w, (0, wide - keep))
    b, h, j = torch.nonzero(there, as_tuple=True)
    o = old[b, h, j]
    src, dst = st["table"][b, o // PAGE].long(), st["new_table"][b, j // PAGE].long()
    for pool in (st["k_pool"], st["v_pool"]):
        pool[dst, h, j % PAGE] = pool[src, h, o % PAGE]
    kept = torch.where(there, kept, -1).to(torch.int32)
    bad = torch.zeros(B, dtype=torch.int32, device=DEV)
    return [kept, w, new_lens.to(torch.int32), bad, *(st[x][st["first_new"]:] for x in ("k_pool", "v_pool"))]


def run(st):
    if not own:
        return _plain(st)
    fa, case, kind = _fa(), st["case"], st["case"]["kind"]
    if kind == "rope":
        return fa.rope(st["q"], st["k"], st["freqs"], st["positions"], interleaved=case["inter"], scale=st["scale"])
    if kind == "rope_bwd":
        return fa.rope_backward(st["q"], st["k"], st["freqs"], st["positions"], interleaved=case["inter"], scale=st["scale"],
                                dtype=DTYPES[case["dtype"]])
    if kind == "append":
        out = fa.kv_append_rope(st["q"], st["k"], st["v"], st["k_pool"], st["v_pool"], st["table"], st["start"], st["freqs"],
                                new_lens=st["rows"], interleaved=case["inter"], want_k=case["want_k"])
        return [*out, st["k_pool"], st["v_pool"]]
    if kind == "shared":
        return fa.decode_shared(st["q"], st["k_pool"], st["v_pool"], st["prefix"], st["prefix_len"], st["table"], st["lens"])
    if kind == "weights":
        return fa.decode_paged_weights(st["q"], st["k_pool"], st["v_pool"], st["table"], st["lens"], st["weights"])
    out = fa.kv_evict(st["k_pool"], st["v_pool"], st["table"], st["lens"], st["weights"], st["new_table"], case["keep"],
                      case["recent"])
    return [*out, *(st[x][st["first_new"]:] for x in ("k_pool", "v_pool"))]


def work(case):
    kind, D, Hkv, e = case["kind"], case["D"], case["Hkv"], SIZE[case["dtype"]]
    H = case.get("H", Hkv)
    if kind in ("rope", "rope_bwd"):
        rows = case["B"] * case["N"]
        n = rows * (H + Hkv) * D
        return {"bytes": n * ((4 if kind == "rope_bwd" else e) + e) + 4 * rows + 4 * case["R"], "flops": 3 * n}
    if kind == "append":
        rows = sum(_rows(case))
        moved = rows * (2 * H + (5 if case["want_k"] else 4) * Hkv) * D * e
        return {"bytes": moved + 12 * case["B"], "flops": 3 * rows * (H + Hkv) * D}
    lens = _lens(case)
    n = sum(lens)
    if kind == "evict":
        m = sum(min(x, case["keep"]) for x in lens)
        return {"bytes": (4 * n + m * (4 * D * e + 8)) * Hkv, "flops": n * Hkv}
    rows = case["B"] * H * (2 * D * e + 4)
    if kind == "weights":
        return {"bytes": n * Hkv * (2 * D * e + 8) + rows, "flops": 4 * n * H * D}
    return {"bytes": (n + case["P"]) * Hkv * 2 * D * e + rows, "flops": 4 * (n + case["B"] * case["P"]) * H * D}


# ---------------------------------------------------------------------------
# The definitions in 64 bits, apart from the plain forms
# ---------------------------------------------------------------------------
def _turned(x, positions, freqs, inter, scale, back=False):
    """Each pair as a complex number times scale e^(i angle), or e^(-i angle)."""
    R = 2 * freqs.numel()
    y = x.double()
    r = y[..., :R]
    pairs = r.reshape(*r.shape[:-1], R // 2, 2) if inter else torch.stack(r.chunk(2, -1), -1)
    a = positions.double()[:, None, :, None] * freqs
    z = torch.view_as_complex(pairs.contiguous()) * torch.polar(torch.full_like(a, scale), -a if back else a)
    z = torch.view_as_real(z)
    z = z.reshape(r.shape) if inter else torch.cat((z[..., 0], z[..., 1]), -1)
    return torch.cat((z, y[..., R:]), -1)


def exact(case, seed):
    st = prepare(case, seed)
    kind, B, D, Hkv = case["kind"], case["B"], case["D"], case["Hkv"]
    f64 = dict(dtype=torch.float64, device=DEV)
    if kind in ("rope", "rope_bwd"):
        return [_turned(st[x], st["positions"], st["freqs"], case["inter"], st["scale"], kind == "rope_bwd") for x in "qk"]
    if kind == "append":
        T = case["T"]
        pos = st["start"][:, None] + torch.arange(T, device=DEV)
        qr, kr = (_turned(st[x], pos, st["freqs"], case["inter"], 1.0) for x in "qk")
        pools = [st["k_pool"].double(), st["v_pool"].double()]
        for b, (p, n) in enumerate(zip(_lens(case), _rows(case))):
            qr[b, :, n:] = 0
            kr[b, :, n:] = 0
            for page in range(p // PAGE, -(-(p + n) // PAGE)):
                lo, hi = max(p, page * PAGE), min(p + n, (page + 1) * PAGE)
                at = st["table"][b, page].long()
                for pool, x in zip(pools, (kr, st["v"])):
                    pool[at, :, lo - page * PAGE:hi - page * PAGE] = x[b, :, lo - p:hi - p].double()
        return [qr, *([kr] if case["want_k"] else []), None, *pools]
    lens = _lens(case)

    def rows(pool, pages, n, h):
        return st[pool][pages.long(), h].reshape(-1, D)[:n].double()

    if kind == "evict":
        keep, wide = case["keep"], st["new_table"].shape[1] * PAGE
        w = torch.zeros(B, Hkv, wide, **f64)
        pools = [st[x][st["first_new"]:].double() for x in ("k_pool", "v_pool")]
        new_table = (st["new_table"].long() - st["first_new"]).cpu()
        for b, n in enumerate(lens):
            m, r = min(n, keep), min(n, case["recent"], keep)
            for h in range(Hkv):
                old = st["weights"][b, h, :n - r].double()
                light = torch.argsort(-old, stable=True)[:m - r]
                idx = torch.cat((torch.sort(light).values, torch.arange(n - r, n, device=DEV)))
                w[b, h, :m] = st["weights"][b, h, idx].double()
                dst = new_table[b, :-(-m // PAGE)].to(DEV)
                for pool, name in zip(pools, ("k_pool", "v_pool")):
                    x = pool[dst, h].reshape(-1, D)
                    x[:m] = rows(name, st["table"][b, :-(-n // PAGE)], n, h)[idx]
                    pool[dst, h] = x.reshape(-1, PAGE, D)
        return [None, w, None, None, *pools]
    H = case["H"]
    G = H // Hkv
    o, l = torch.empty(B, H, D, **f64), torch.empty(B, H, **f64)
    w = st["weights"].double() if kind == "weights" else None
    for h in range(Hkv):
        g = slice(h * G, (h + 1) * G)
        shared = [rows(x, st["prefix"], case["P"], h) for x in ("k_pool", "v_pool")] if kind == "shared" else None
        for b, n in enumerate(lens):
            k, v = (rows(x, st["table"][b, :-(-n // PAGE)], n, h) for x in ("k_pool", "v_pool"))
            if shared is not None:
                k, v = torch.cat((shared[0], k)), torch.cat((shared[1], v))
            s = st["q"][b, g].double() @ k.t().contiguous() / math.sqrt(D)
            l[b, g] = torch.logsumexp(s, 1)
            p = torch.exp(s - l[b, g, None])
            o[b, g] = p @ v
            if w is not None:
                w[b, h, :n] += p.sum(0)
    return [o, l] if w is None else [o, l, w]
