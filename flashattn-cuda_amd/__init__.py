"""MI355X (gfx950) FlashAttention forward and split-KV paged decode.

Drop-in for the reference's torch-extension module
(cuda/flash_attn_fa3_db_full.cu:405-418):

    O, L = forward(Q, K, V)           # O fp16 [B,H,N,D], L fp32 [B,H,N]
    O = forward_only(Q, K, V)         # bitwise the same O, no L

Both accept ``causal=True``, D in {64, 128} and K/V with fewer heads than Q
(GQA/MQA: [B, H_kv, N, D], H a multiple of H_kv); ``forward_varlen`` takes
packed variable-length sequences. The backward of the
reference's first module (cuda/flash_attn_kernel.cu:417-503):

    dQ, dK, dV = backward(Q, K, V, O, dO, L)   # fp32 [B,H,N,D]

New entry points:

    bad = kv_append(k_new, v_new, k_pool, v_pool, page_table, start_pos)   # in place
    O, L = decode_paged(q, k_pool, v_pool, page_table, ctx_lens, num_splits=16)
    part_o, part_lse = decode_partials(...);  O, L = lse_combine(part_o, part_lse)

The same cache in 4 or 8 bits a value (MX pages, K and V each of its own width):

    k_pool, v_pool = kv_pools_mx(num_pages, H_kv, D, k_bits=4, v_bits=4, device=...)
    bad = kv_append_mx(k_new, v_new, k_pool, v_pool, page_table, start_pos)   # in place
    k, v, bad = kv_read_mx(k_pool, v_pool, page_table, start_pos, num_tokens)
    O, L = decode_paged_mx(q, k_pool, v_pool, page_table, ctx_lens)

Rotary positions, a prefix shared by a batch, and a cache kept within a budget:

    freqs, scale = rope_frequencies(rot_dim, base=10000.0)
    Qr, Kr = rope(Q, K, freqs, positions)
    dQ, dK = rope_backward(dQr, dKr, freqs, positions)
    q, bad = kv_append_rope(q, k_new, v_new, k_pool, v_pool, page_table, start_pos, freqs)
    O, L = decode_shared(q, k_pool, v_pool, prefix_table, prefix_len, page_table, ctx_lens)
    O, L, weights = decode_paged_weights(q, k_pool, v_pool, page_table, ctx_lens, weights)
    kept, weights, lens, bad = kv_evict(k_pool, v_pool, page_table, ctx_lens, weights,
                                        new_page_table, keep, recent)

Every call runs the hand-written HIP kernels of ``libfa_mi355x.so`` through
the C ABI in include/fa_mi355x.h. There is no fallback: importing this package
without the built extension raises ImportError.
"""
from __future__ import annotations

import importlib.machinery
import importlib.util
import math
import os
import pathlib
import sysconfig

import torch  # noqa: F401  (loads the HIP runtime the extension links against)

_HERE = pathlib.Path(__file__).resolve().parent
_EXT = _HERE / ("_fa_torch" + sysconfig.get_config_var("EXT_SUFFIX"))
LIB_PATH = _HERE / "libfa_mi355x.so"


def _load_ext():
    if not _EXT.exists() or not LIB_PATH.exists():
        raise ImportError(
            f"flashattn-cuda_amd is not built ({_EXT.name} / {LIB_PATH.name} missing); "
            f"run `python {_HERE / 'build.py'}`")
    loader = importlib.machinery.ExtensionFileLoader("_fa_torch", str(_EXT))
    spec = importlib.util.spec_from_file_location("_fa_torch", str(_EXT), loader=loader)
    mod = importlib.util.module_from_spec(spec)
    loader.exec_module(mod)
    return mod


_C = _load_ext()
EXT_PATH = _EXT


def forward(Q, K, V, causal: bool = False):
    """[O, L]: O = softmax(Q K^T / sqrt(D)) V (fp16), L = row logsumexp (fp32)."""
    return _C.forward(Q, K, V, causal)


def forward_bf16(Q, K, V, causal: bool = False, want_L: bool = True):
    """bfloat16 forward: [O bf16 [B,H,N,D], L fp32 [B,H,N]] ([O] if not want_L)."""
    return _C.forward_bf16(Q, K, V, causal, want_L)


def forward_varlen(q, k, v, cu_seqlens, max_seqlen: int, causal: bool = False):
    """[O, L] of B packed sequences, head-major: q [H, total, D], k/v [H_kv, total, D].

    Sequence b is rows cu_seqlens[b] .. cu_seqlens[b+1] (int32 [B+1]) of every
    head and attends only within itself; max_seqlen must cover every sequence.
    Rows past cu_seqlens[B] belong to no sequence: O = 0 and L = -inf there.
    """
    return _C.forward_varlen(q, k, v, cu_seqlens, max_seqlen, causal)


def forward_only(Q, K, V, causal: bool = False):
    """O only; bitwise equal to forward(...)[0]."""
    return _C.forward_only(Q, K, V, causal)


def backward(Q, K, V, O, dO, L, causal: bool = False):
    """[dQ, dK, dV] (fp32 [B,H,N,D]) of sum(O * dO), from forward()'s O and L.

    The reference's backward(Q, K, V, O, dO, L) (cuda/flash_attn_kernel.cu:417-503).
    """
    return _C.backward(Q, K, V, O, dO, L, causal)


def backward_bf16(Q, K, V, O, dO, L, causal: bool = False):
    """[dQ, dK, dV] (fp32) of forward_bf16(): inputs in bfloat16, P and dS
    rounded to bf16 for their products; K/V may have fewer heads (GQA)."""
    return _C.backward_bf16(Q, K, V, O, dO, L, causal)


def backward_varlen(q, k, v, o, dO, L, cu_seqlens, max_seqlen: int, causal: bool = False):
    """[dQ, dK, dV] (fp32, head-major packed like forward_varlen's inputs) of
    forward_varlen(); rows outside every sequence are zeros."""
    return _C.backward_varlen(q, k, v, o, dO, L, cu_seqlens, max_seqlen, causal)


def kv_append(k_new, v_new, k_pool, v_pool, page_table, start_pos, new_lens=None):
    """Write k_new/v_new [B,H,T,D] into the pools at start_pos[b] + t, in place
    (all four fp16, or all four bf16).

    Returns bad int32 [B]: 1 where a token of the sequence had no valid page
    (that token is not written).
    """
    return _C.kv_append(k_new, v_new, k_pool, v_pool, page_table, start_pos, new_lens)


def decode_paged(q, k_pool, v_pool, page_table, ctx_lens, num_splits: int = 16):
    """[O, L] of one query token per sequence over its paged K/V (split pass + combine).

    q and the pools are all fp16 or all bf16; O has q's dtype, L is fp32.
    """
    return _C.decode_paged(q, k_pool, v_pool, page_table, ctx_lens, num_splits)


def decode_partials(q, k_pool, v_pool, page_table, ctx_lens, num_splits: int = 16):
    """[part_o fp32 [B,H,S,D], part_lse fp32 [B,H,S]] of the split pass alone."""
    return _C.decode_partials(q, k_pool, v_pool, page_table, ctx_lens, num_splits)


def lse_combine(part_o, part_lse):
    """[O fp16 [B,H,D], L fp32 [B,H]] merged from split partials."""
    return _C.lse_combine(part_o, part_lse)


def mx_page_bytes(D: int, bits: int) -> int:
    """Bytes of an MX page (16 tokens of one head): 16 * D values of 4 or 8 bits
    and a scale byte for every 32 of them."""
    n = _C.mx_page_bytes(D, bits)
    if n == 0:
        raise RuntimeError("MX pages need a head dimension of 64 or 128 and 4 or 8 bits")
    return n


def kv_pools_mx(num_pages: int, H_kv: int, D: int, k_bits: int = 4, v_bits: int = 4, device="cuda"):
    """(k_pool, v_pool): zeroed uint8 [num_pages, H_kv, mx_page_bytes(D, bits)].

    Blocks of 32 values along D share a power-of-two scale; values are E2M1 (4
    bits) or E4M3 (8 bits). The layout of a page is in include/fa_mi355x.h.
    """
    return tuple(torch.zeros(num_pages, H_kv, mx_page_bytes(D, b), dtype=torch.uint8, device=device)
                 for b in (k_bits, v_bits))


def kv_append_mx(k_new, v_new, k_pool, v_pool, page_table, start_pos, new_lens=None):
    """kv_append into MX pages: k_new/v_new [B,H,T,D] (both fp16 or both bf16) are
    quantised as they are written, in place; returns bad int32 [B] as kv_append.

    Every value is rounded to the nearest its block's scale allows (blocks that
    hold a NaN or an infinity read back as NaN).
    """
    return _C.kv_append_mx(k_new, v_new, k_pool, v_pool, page_table, start_pos, new_lens)


def kv_read_mx(k_pool, v_pool, page_table, start_pos, num_tokens: int, lens=None,
               dtype=torch.float16):
    """[k, v, bad]: tokens start_pos[b] .. + num_tokens out of MX pages, k/v
    [B,H_kv,num_tokens,D] in dtype (fp16 or bf16), without rounding for pages
    written from rows of that dtype.

    Rows from lens[b] on are zeros; a token with no valid page reads as NaN and
    sets bad[b] (int32 [B]).
    """
    if dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError("dtype must be torch.float16 or torch.bfloat16")
    return _C.kv_read_mx(k_pool, v_pool, page_table, start_pos, num_tokens, lens,
                         dtype == torch.bfloat16)


def decode_paged_mx(q, k_pool, v_pool, page_table, ctx_lens):
    """[O, L] of one query token per sequence over its MX pages (decode_paged's
    results for what the pages hold); q fp16 or bf16, O in q's dtype, L fp32.

    q has the dtype of the rows that were appended, which no call can check:
    values of bf16 rows may lie beyond fp16's range.

    The split over the pages follows the batch's lengths, on the device.
    """
    return _C.decode_paged_mx(q, k_pool, v_pool, page_table, ctx_lens)


def rope_frequencies(rot_dim: int, base: float = 10000.0, scaling=None, factor: float = 1.0,
                     original_len: int = 0, slow_turns: float = 1.0, fast_turns: float = 32.0,
                     device="cuda"):
    """(freqs, scale) for rope(): freqs float64 [rot_dim / 2], radians a position.

    freqs[i] = base ** (-2 i / rot_dim), and for contexts `factor` times as long as
    the original_len positions that a model was trained on, by `scaling`:

      None        as they are
      "linear"    all divided by factor (positions interpolated)
      "ntk"       base * factor ** (rot_dim / (rot_dim - 2)): the slowest is divided
                  by factor, the fastest kept
      "by_parts"  those that make fewer than slow_turns turns within original_len
                  divided by factor, those that make more than fast_turns kept, a
                  linear ramp over their index between the two; scale is 0.1 ln factor + 1
                  (YaRN, Peng et al. 2023). The ramp's ends, rounded outwards, may lie
                  before the first frequency or past the last one: a trained length
                  above 2 pi base leaves even the slowest partly kept

    scale is 1 otherwise. It multiplies the rotated dims of Q and of K.
    """
    if rot_dim <= 0 or rot_dim % 2 != 0:
        raise RuntimeError("rot_dim must be positive and even")
    if not (base > 1.0 and factor >= 1.0):
        raise RuntimeError("base must be > 1 and factor >= 1")
    half = rot_dim // 2
    i = torch.arange(half, dtype=torch.float64)
    scale = 1.0
    if scaling == "ntk":
        if rot_dim < 4:
            raise RuntimeError("scaling 'ntk' needs rot_dim >= 4")
        base = base * factor ** (rot_dim / (rot_dim - 2))
    freqs = base ** (-2.0 * i / rot_dim)
    if scaling == "linear":
        freqs = freqs / factor
    elif scaling == "by_parts":
        if original_len <= 0 or not 0.0 < slow_turns < fast_turns:
            raise RuntimeError("scaling 'by_parts' needs original_len > 0 and 0 < slow_turns < fast_turns")

        def index(turns):   # of the frequency that makes so many turns within original_len
            return rot_dim * math.log(original_len / (2.0 * math.pi * turns)) / (2.0 * math.log(base))

        lo = math.floor(index(fast_turns))
        hi = max(math.ceil(index(slow_turns)), lo + 1)   # both one index: kept up to it
        ramp = torch.clamp((i - lo) / (hi - lo), 0.0, 1.0)   # 0: kept, 1: divided
        freqs = freqs * (1.0 - ramp) + freqs / factor * ramp
        scale = 0.1 * math.log(factor) + 1.0
    elif scaling not in (None, "ntk"):
        raise RuntimeError("scaling must be None, 'linear', 'ntk' or 'by_parts'")
    return freqs.to(device), scale


_ROPE_TYPES = {None: -1, torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


def rope(Q, K, freqs, positions=None, interleaved: bool = False, scale: float = 1.0):
    """[Q', K']: the first R = 2 * len(freqs) dims of every row turned by its position,
    contiguous, in the dtype of Q and K (fp16, bf16 or fp32). [Q'] if K is None.

    Q [B,H,N,D] and K [B,H_kv,N,D] may be views (a projection's [B,N,H,D] transposed)
    and are read as they lie where rows are contiguous and 16-byte aligned; packed
    rows are [H,total,D]. positions: int32 [N] or [B,N] (packed [total]); None: 0 to
    N - 1. Pairs are dims (i, i + R/2), or neighbours if interleaved. Angles are exact
    for any position (reduced in 64 bits).
    """
    return _C.rope(Q, K, freqs, positions, interleaved, scale, False, -1)


def rope_backward(dQ, dK, freqs, positions=None, interleaved: bool = False, scale: float = 1.0,
                  dtype=None):
    """[dQ, dK] of rope's inputs from those of its outputs (backward()'s fp32 ones, or
    16-bit ones), in dtype: theirs, or for fp32 gradients also fp16 or bf16.

    freqs, positions, interleaved and scale as in the call of rope.
    """
    if dtype not in _ROPE_TYPES:
        raise RuntimeError("dtype must be torch.float16, torch.bfloat16 or torch.float32")
    return _C.rope(dQ, dK, freqs, positions, interleaved, scale, True, _ROPE_TYPES[dtype])


def kv_append_rope(q, k_new, v_new, k_pool, v_pool, page_table, start_pos, freqs, positions=None,
                   new_lens=None, interleaved: bool = False, scale: float = 1.0, want_k: bool = False):
    """[q', bad]: rope of q [B,H,T,D] and k_new [B,H_kv,T,D], and kv_append of the rotated
    k_new and of v_new, in one launch. With want_k [q', k', bad] (a prompt's own attention
    needs k').

    positions: int32 [B], the position of each sequence's first new token where it is
    not its slot start_pos[b] (after kv_evict). q, k_new, v_new may be views as in
    rope (slices of a joined q, k, v). Rows of q' and k' from new_lens[b] on are zeros.
    """
    return _C.kv_append_rope(q, k_new, v_new, k_pool, v_pool, page_table, start_pos, freqs, positions,
                             new_lens, interleaved, scale, want_k)


def decode_shared(q, k_pool, v_pool, prefix_table, prefix_len, page_table, ctx_lens):
    """[O, L] of one query token per sequence over a prefix that all sequences share and
    then its own paged K/V, as one softmax; decode_paged's dtypes.

    The prefix is the first prefix_len (int32, one value, on the device) tokens of the
    pages prefix_table (int32 [prefix_pages]), read once for every 128 query rows (b, h)
    of a KV head, for every 16 where there are up to 32, and of short tables once a sequence;
    page_table and ctx_lens are those of the sequences' own tokens (lengths may be 0).
    An invalid prefix makes every O and L NaN, an invalid own page those of its sequence.
    """
    return _C.decode_shared(q, k_pool, v_pool, prefix_table, prefix_len, page_table, ctx_lens)


def decode_paged_weights(q, k_pool, v_pool, page_table, ctx_lens, weights, inplace: bool = False):
    """[O, L, W]: decode_paged, and W = weights with the attention weight of every cached
    token added, summed over the query heads of its KV head (fp32 [B,H_kv,max_pages*16]).

    inplace: W is weights itself. Slots past a context keep their value; where O and L
    are NaN (an invalid page or length), W is NaN over the context. The split over the
    pages follows the batch's lengths, on the device, and the table's width.
    """
    return _C.decode_paged_weights(q, k_pool, v_pool, page_table, ctx_lens, weights, inplace)


def kv_evict(k_pool, v_pool, page_table, ctx_lens, weights, new_page_table, keep: int, recent: int):
    """[kept, new_weights, new_lens, bad]: at most `keep` tokens of each head stay, the
    `recent` last ones and of the others the heaviest by weights (of equal ones the
    earliest; NaN counts as lightest), copied in order into the pages of new_page_table.

    kept int32 [B,H_kv,keep]: old slot of each new one, then -1; new_weights fp32
    [B,H_kv,new_max_pages*16]: their weights, then zeros; new_lens int32 [B]. bad int32
    [B]: 1 where a row had no valid page, old or new (it is not copied), or the length
    is invalid (then new_lens is 0). The new pages must not be among the old ones,
    which are the caller's to free afterwards.
    """
    return _C.kv_evict(k_pool, v_pool, page_table, ctx_lens, weights, new_page_table, keep, recent)


def loaded_libraries():
    """Paths of this package's native libraries mapped into the process."""
    out = []
    try:
        with open(f"/proc/{os.getpid()}/maps") as f:
            for line in f:
                p = line.split()[-1]
                if p.startswith(str(_HERE)) and p.endswith(".so") and p not in out:
                    out.append(p)
    except OSError:
        pass
    return out


probe = _C  # probe_mfma32, probe_mfma16, probe_tr16_raw, probe_frags, probe_chain
