// fa_capi.cpp — host-only part of the C ABI: argument validation and status
// strings. No HIP call is made here, so every error path runs without a GPU.
//
// fa_validate_fwd mirrors the argument checks of the reference launcher
// fa3db_full_forward_impl (cuda/flash_attn_fa3_db_full.cu:352-363): head dim,
// N > 0, and the B*H grid limit, widened to D in {64, 128}; shape/device
// equality of Q/K/V is the binding's job because the C ABI only sees
// pointers.
#include <stdint.h>

#include "fa_mi355x.h"

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Largest element count the kernels index with 32-bit in-head offsets.
constexpr int64_t kMaxHeadElems = (int64_t(1) << 31) - 1;
constexpr int64_t kMaxGrid = (int64_t(1) << 31) - 1;

}  // namespace

extern "C" const char* fa_status_str(int status) {
  switch (status) {
    case FA_OK: return "ok";
    case FA_ERR_NULL_POINTER: return "a required pointer is NULL";
    case FA_ERR_HEAD_DIM: return "Head dimension must be 64 or 128";
    case FA_ERR_SEQ_LEN: return "N must be > 0";
    case FA_ERR_BATCH_HEADS: return "B and H must be > 0";
    case FA_ERR_ALIGNMENT: return "tensor pointers must be 16-byte aligned";
    case FA_ERR_TOO_LARGE: return "size exceeds the kernels' 32-bit index range";
    case FA_ERR_PAGE_SIZE: return "page_size must be 16";
    case FA_ERR_NUM_SPLITS: return "num_splits must be in [1, 16]";
    case FA_ERR_MAX_PAGES: return "max_pages must be > 0";
    case FA_ERR_NUM_PAGES: return "num_pages must be > 0";
    case FA_ERR_KV_HEADS: return "H must be a positive multiple of H_kv";
    case FA_ERR_SCRATCH_SIZE:
      return "B*H*num_splits*(D+1) exceeds FA_DECODE_SCRATCH_FLOATS (no-alloc decode)";
    case FA_ERR_MX_BITS: return "k_bits and v_bits must be 4 or 8";
    case FA_ERR_ROT_DIM: return "rot_dim must be a positive multiple of 16, at most the head dimension";
    case FA_ERR_STRIDE: return "row strides must be multiples of 16 bytes";
    case FA_ERR_TYPE: return "element types must be alike, or float32 in";
    case FA_ERR_BUDGET: return "keep must be in [1, new_max_pages * 16] and recent in [0, keep]";
    default: break;
  }
  if (status < 0) return "HIP error (negated hipError_t)";
  return "unknown fa_mi355x status";
}

extern "C" int fa_abi_version(void) { return FA_ABI_VERSION; }

extern "C" int fa_validate_fwd(const void* q, const void* k, const void* v, const void* o,
                               int64_t B, int64_t H, int64_t N, int64_t D) {
  if (!q || !k || !v || !o) return FA_ERR_NULL_POINTER;
  if (D != 64 && D != 128) return FA_ERR_HEAD_DIM;
  if (N <= 0) return FA_ERR_SEQ_LEN;
  if (B <= 0 || H <= 0) return FA_ERR_BATCH_HEADS;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o)) return FA_ERR_ALIGNMENT;
  // One head of K or V is addressed through a 32-bit buffer range (bytes).
  if (N * D * 2 > kMaxHeadElems) return FA_ERR_TOO_LARGE;
  if (B > kMaxGrid / H) return FA_ERR_TOO_LARGE;
  const int64_t bh = B * H;
  const int64_t num_qb = (N + 127) / 128;
  if (bh > kMaxGrid / num_qb) return FA_ERR_TOO_LARGE;
  return FA_OK;
}

// GQA: the dense checks plus the head grouping.
extern "C" int fa_validate_fwd_gqa(const void* q, const void* k, const void* v, const void* o,
                                   int64_t B, int64_t H, int64_t H_kv, int64_t N, int64_t D) {
  const int st = fa_validate_fwd(q, k, v, o, B, H, N, D);
  if (st != FA_OK) return st;
  if (H_kv <= 0 || H % H_kv != 0) return FA_ERR_KV_HEADS;
  return FA_OK;
}

// Varlen: one head's packed rows are addressed with size_t offsets; one
// sequence (at most max_seqlen rows) through a 32-bit buffer range.
extern "C" int fa_validate_fwd_varlen(const void* q, const void* k, const void* v, const void* o,
                                      const int32_t* cu_seqlens, int64_t B, int64_t H,
                                      int64_t H_kv, int64_t max_seqlen, int64_t total,
                                      int64_t D) {
  if (!q || !k || !v || !o || !cu_seqlens) return FA_ERR_NULL_POINTER;
  if (D != 64 && D != 128) return FA_ERR_HEAD_DIM;
  if (max_seqlen <= 0 || total < 0) return FA_ERR_SEQ_LEN;
  if (B <= 0 || H <= 0) return FA_ERR_BATCH_HEADS;
  if (H_kv <= 0 || H % H_kv != 0) return FA_ERR_KV_HEADS;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o)) return FA_ERR_ALIGNMENT;
  if (reinterpret_cast<uintptr_t>(cu_seqlens) & 3u) return FA_ERR_ALIGNMENT;
  if (max_seqlen * D * 2 > kMaxHeadElems || total > kMaxGrid) return FA_ERR_TOO_LARGE;
  if (B > kMaxGrid / H) return FA_ERR_TOO_LARGE;
  const int64_t num_qb = (max_seqlen + 127) / 128;
  if (B * H > kMaxGrid / num_qb) return FA_ERR_TOO_LARGE;
  return FA_OK;
}

// Mirrors the reference backward launcher's checks (cuda/flash_attn_kernel.cu:
// 425-432: CUDA tensors, head dimension), widened to D in {64, 128}, plus the
// C ABI's own pointer, alignment and index-range checks.
extern "C" int fa_validate_bwd(const void* q, const void* k, const void* v, const void* o,
                               const void* dout, const float* lse, const float* dq,
                               const float* dk, const float* dv, const float* workspace,
                               int64_t B, int64_t H, int64_t N, int64_t D) {
  if (!dout || !lse || !dq || !dk || !dv || !workspace) return FA_ERR_NULL_POINTER;
  const int st = fa_validate_fwd(q, k, v, o, B, H, N, D);
  if (st != FA_OK) return st;
  if (!aligned16(dout) || !aligned16(dq) || !aligned16(dk) || !aligned16(dv))
    return FA_ERR_ALIGNMENT;
  if ((reinterpret_cast<uintptr_t>(lse) & 3u) != 0 ||
      (reinterpret_cast<uintptr_t>(workspace) & 3u) != 0)
    return FA_ERR_ALIGNMENT;
  // The row-sum kernel's grid (32 rows per workgroup) and the per-head float
  // offsets of the gradients.
  if (B * H > kMaxGrid / N) return FA_ERR_TOO_LARGE;
  if ((B * H * N + 31) / 32 > kMaxGrid) return FA_ERR_TOO_LARGE;
  return FA_OK;
}

// Varlen backward (no reference counterpart): the varlen forward's checks on
// q/k/v/o plus the backward's gradient, L and workspace pointers and the row
// grid of the D_i pass.
extern "C" int fa_validate_bwd_varlen(const void* q, const void* k, const void* v, const void* o,
                                      const void* dout, const float* lse, const float* dq,
                                      const float* dk, const float* dv, const float* workspace,
                                      const int32_t* cu_seqlens, int64_t B, int64_t H,
                                      int64_t H_kv, int64_t max_seqlen, int64_t total,
                                      int64_t D) {
  if (!dout || !lse || !dq || !dk || !dv || !workspace) return FA_ERR_NULL_POINTER;
  const int st = fa_validate_fwd_varlen(q, k, v, o, cu_seqlens, B, H, H_kv, max_seqlen, total, D);
  if (st != FA_OK) return st;
  if (!aligned16(dout) || !aligned16(dq) || !aligned16(dk) || !aligned16(dv))
    return FA_ERR_ALIGNMENT;
  if ((reinterpret_cast<uintptr_t>(lse) & 3u) != 0 ||
      (reinterpret_cast<uintptr_t>(workspace) & 3u) != 0)
    return FA_ERR_ALIGNMENT;
  if (H > kMaxGrid / (total > 0 ? total : 1)) return FA_ERR_TOO_LARGE;
  if ((H * total + 31) / 32 > kMaxGrid) return FA_ERR_TOO_LARGE;
  return FA_OK;
}

// Decode arguments (no reference counterpart): pool/page-table shapes, the
// split count and the grid limits of the split pass.
extern "C" int fa_validate_decode(const void* q, const void* k_pool, const void* v_pool,
                                  const int32_t* page_table, const int32_t* ctx_lens,
                                  int64_t B, int64_t H, int64_t D, int64_t page_size,
                                  int64_t max_pages, int64_t num_pages, int64_t num_splits) {
  if (!q || !k_pool || !v_pool || !page_table || !ctx_lens) return FA_ERR_NULL_POINTER;
  if (D != 64 && D != 128) return FA_ERR_HEAD_DIM;
  if (B <= 0 || H <= 0) return FA_ERR_BATCH_HEADS;
  if (page_size != 16) return FA_ERR_PAGE_SIZE;
  if (num_splits < 1 || num_splits > 16) return FA_ERR_NUM_SPLITS;
  if (max_pages <= 0) return FA_ERR_MAX_PAGES;
  if (num_pages <= 0) return FA_ERR_NUM_PAGES;
  if (!aligned16(q) || !aligned16(k_pool) || !aligned16(v_pool)) return FA_ERR_ALIGNMENT;
  if ((reinterpret_cast<uintptr_t>(page_table) & 3u) || (reinterpret_cast<uintptr_t>(ctx_lens) & 3u))
    return FA_ERR_ALIGNMENT;
  // Grid is (num_splits, H, B); y and z are limited to 65535 on this target.
  if (H > 65535 || B > 65535) return FA_ERR_TOO_LARGE;
  if (B > kMaxHeadElems / max_pages) return FA_ERR_TOO_LARGE;
  if (max_pages > kMaxHeadElems / page_size) return FA_ERR_TOO_LARGE;
  return FA_OK;
}

// KV page writer arguments (no reference counterpart). T = 0 is a valid
// no-op; grid is (ceil(T / rows), H, B).
extern "C" int fa_validate_kv_append(const void* k_new, const void* v_new,
                                     const int32_t* page_table, const int32_t* start_pos,
                                     const int32_t* new_lens, const void* k_pool,
                                     const void* v_pool, const int32_t* bad, int64_t B, int64_t H,
                                     int64_t T, int64_t D, int64_t page_size, int64_t max_pages,
                                     int64_t num_pages) {
  // k_new/v_new may be NULL when there is nothing to copy (T = 0: an empty
  // tensor has no storage).
  if ((T != 0 && (!k_new || !v_new)) || !page_table || !start_pos || !k_pool || !v_pool)
    return FA_ERR_NULL_POINTER;
  if (D != 64 && D != 128) return FA_ERR_HEAD_DIM;
  if (T < 0) return FA_ERR_SEQ_LEN;
  if (B <= 0 || H <= 0) return FA_ERR_BATCH_HEADS;
  if (page_size != 16) return FA_ERR_PAGE_SIZE;
  if (max_pages <= 0) return FA_ERR_MAX_PAGES;
  if (num_pages <= 0) return FA_ERR_NUM_PAGES;
  if (!aligned16(k_new) || !aligned16(v_new) || !aligned16(k_pool) || !aligned16(v_pool))
    return FA_ERR_ALIGNMENT;
  const auto a4 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; };
  if (!a4(page_table) || !a4(start_pos) || !a4(new_lens) || !a4(bad)) return FA_ERR_ALIGNMENT;
  if (H > 65535 || B > 65535) return FA_ERR_TOO_LARGE;
  if (T > kMaxGrid || max_pages > kMaxGrid || num_pages > kMaxGrid) return FA_ERR_TOO_LARGE;
  return FA_OK;
}

extern "C" int64_t fa_decode_workspace_floats(int64_t B, int64_t H, int64_t D,
                                              int64_t num_splits) {
  if (B <= 0 || H <= 0 || D <= 0 || num_splits <= 0) return 0;
  return B * H * num_splits * (D + 1);
}

extern "C" int64_t fa_mx_page_bytes(int64_t D, int64_t bits) {
  if ((D != 64 && D != 128) || (bits != 4 && bits != 8)) return 0;
  return 16 * D * bits / 8 + 16 * D / 32;
}

// MX pages (no reference counterpart): the 16-bit writer's checks, the widths
// and the flags, which the MX calls always write.
extern "C" int fa_validate_kv_append_mx(const void* k, const void* v, const int32_t* page_table,
                                        const int32_t* start_pos, const int32_t* lens,
                                        const void* k_pool, const void* v_pool, const int32_t* bad,
                                        int64_t B, int64_t H, int64_t T, int64_t D, int64_t k_bits,
                                        int64_t v_bits, int64_t page_size, int64_t max_pages,
                                        int64_t num_pages) {
  if (!bad) return FA_ERR_NULL_POINTER;
  const int st = fa_validate_kv_append(k, v, page_table, start_pos, lens, k_pool, v_pool, bad, B, H,
                                       T, D, page_size, max_pages, num_pages);
  if (st != FA_OK) return st;
  if (fa_mx_page_bytes(D, k_bits) == 0 || fa_mx_page_bytes(D, v_bits) == 0) return FA_ERR_MX_BITS;
  // A workgroup of 256 threads has 16 tokens, and a grid fewer than 2^32 threads.
  if (T > (int64_t(1) << 28) - 32) return FA_ERR_TOO_LARGE;
  return FA_OK;
}

// The paged decode's checks, but for num_splits, which the MX decode has not.
// Its grid is (chunks, head groups).
extern "C" int fa_validate_decode_mx(const void* q, const void* k_pool, const void* v_pool,
                                     const int32_t* page_table, const int32_t* ctx_lens, int64_t B,
                                     int64_t H, int64_t H_kv, int64_t D, int64_t k_bits,
                                     int64_t v_bits, int64_t page_size, int64_t max_pages,
                                     int64_t num_pages, const float* workspace, const void* o,
                                     const float* lse) {
  const int st = fa_validate_decode(q, k_pool, v_pool, page_table, ctx_lens, B, H, D, page_size,
                                    max_pages, num_pages, /*num_splits=*/1);
  if (st != FA_OK) return st;
  if (H_kv <= 0 || H % H_kv != 0) return FA_ERR_KV_HEADS;
  if (fa_mx_page_bytes(D, k_bits) == 0 || fa_mx_page_bytes(D, v_bits) == 0) return FA_ERR_MX_BITS;
  if (!o || (!workspace && fa_decode_mx_workspace_floats(B, H, H_kv, D, max_pages) > 0))
    return FA_ERR_NULL_POINTER;
  if (!aligned16(workspace) || !aligned16(o)) return FA_ERR_ALIGNMENT;
  if (reinterpret_cast<uintptr_t>(lse) & 3u) return FA_ERR_ALIGNMENT;
  if (num_pages > kMaxGrid) return FA_ERR_TOO_LARGE;
  return FA_OK;
}

// Rotary positions (no reference counterpart). Strides of dimensions of one index
// are not looked at; rows are read as 16-byte pieces.
static int check_rows(const void* p, const int64_t* st, int64_t B, int64_t H, int64_t N, int64_t size) {
  if (!p) return FA_OK;
  if (!st) return FA_ERR_NULL_POINTER;
  const int64_t n[3] = {B, H, N};
  for (int i = 0; i < 3; ++i)
    if (n[i] > 1 && (st[i] < 0 || st[i] * size % 16 != 0)) return FA_ERR_STRIDE;
  return aligned16(p) ? FA_OK : FA_ERR_ALIGNMENT;
}

static int check_rot(const double* freqs, int64_t B, int64_t H, int64_t H_kv, int64_t N, int64_t D,
                     int64_t rot_dim) {
  if (!freqs) return FA_ERR_NULL_POINTER;
  if (D != 64 && D != 128) return FA_ERR_HEAD_DIM;
  if (rot_dim <= 0 || rot_dim > D || rot_dim % 16 != 0) return FA_ERR_ROT_DIM;
  if (B <= 0 || H <= 0) return FA_ERR_BATCH_HEADS;
  if (reinterpret_cast<uintptr_t>(freqs) & 7u) return FA_ERR_ALIGNMENT;
  // Grid (token blocks, head slots, B).
  if (B > 65535 || H + 2 * H_kv > 65535 || N > (int64_t(1) << 28)) return FA_ERR_TOO_LARGE;
  return FA_OK;
}

extern "C" int fa_validate_rope(const void* q, const int64_t q_strides[3], const void* k,
                                const int64_t k_strides[3], const double* freqs,
                                const int32_t* positions, int64_t pos_stride, const void* q_out,
                                const void* k_out, int64_t B, int64_t H, int64_t H_kv, int64_t N,
                                int64_t D, int64_t rot_dim, int in_type, int out_type) {
  if (!q || !q_out || (H_kv != 0 && (!k || !k_out))) return FA_ERR_NULL_POINTER;
  if (H_kv < 0) return FA_ERR_KV_HEADS;
  if (N <= 0) return FA_ERR_SEQ_LEN;
  int st = check_rot(freqs, B, H, H_kv, N, D, rot_dim);
  if (st != FA_OK) return st;
  if (in_type < FA_F16 || in_type > FA_F32 || out_type < FA_F16 || out_type > FA_F32 ||
      (in_type != out_type && in_type != FA_F32))
    return FA_ERR_TYPE;
  const int64_t size = in_type == FA_F32 ? 4 : 2;
  st = check_rows(q, q_strides, B, H, N, size);
  if (st == FA_OK && H_kv > 0) st = check_rows(k, k_strides, B, H_kv, N, size);
  if (st != FA_OK) return st;
  if (!aligned16(q_out) || (H_kv > 0 && !aligned16(k_out))) return FA_ERR_ALIGNMENT;
  if (reinterpret_cast<uintptr_t>(positions) & 3u) return FA_ERR_ALIGNMENT;
  if (positions && pos_stride < 0) return FA_ERR_STRIDE;
  return FA_OK;
}

extern "C" int fa_validate_kv_append_rope(const void* q, const int64_t q_strides[3], const void* k,
                                          const int64_t k_strides[3], const void* v,
                                          const int64_t v_strides[3], const double* freqs,
                                          const int32_t* page_table, const int32_t* start_pos,
                                          const int32_t* positions, const int32_t* new_lens,
                                          const void* k_pool, const void* v_pool, const void* q_out,
                                          const void* k_out, const int32_t* bad, int64_t B, int64_t H,
                                          int64_t H_kv, int64_t T, int64_t D, int64_t rot_dim,
                                          int64_t page_size, int64_t max_pages, int64_t num_pages) {
  if (!bad || (T != 0 && (!q || !q_out))) return FA_ERR_NULL_POINTER;
  int st = fa_validate_kv_append(k, v, page_table, start_pos, new_lens, k_pool, v_pool, bad, B, H_kv,
                                 T, D, page_size, max_pages, num_pages);
  if (st != FA_OK) return st;
  if (H <= 0 || H % H_kv != 0) return FA_ERR_KV_HEADS;
  st = check_rot(freqs, B, H, H_kv, T, D, rot_dim);
  if (st == FA_OK) st = check_rows(q, q_strides, B, H, T, 2);
  if (st == FA_OK) st = check_rows(k, k_strides, B, H_kv, T, 2);
  if (st == FA_OK) st = check_rows(v, v_strides, B, H_kv, T, 2);
  if (st != FA_OK) return st;
  if (!aligned16(q_out) || !aligned16(k_out)) return FA_ERR_ALIGNMENT;
  if (reinterpret_cast<uintptr_t>(positions) & 3u) return FA_ERR_ALIGNMENT;
  return FA_OK;
}

// The paged decode's checks and those of the prefix: its grid is one-dimensional.
extern "C" int fa_validate_decode_shared(const void* q, const void* k_pool, const void* v_pool,
                                         const int32_t* prefix_table, const int32_t* prefix_len,
                                         const int32_t* page_table, const int32_t* ctx_lens, int64_t B,
                                         int64_t H, int64_t H_kv, int64_t D, int64_t page_size,
                                         int64_t prefix_pages, int64_t max_pages, int64_t num_pages,
                                         const float* workspace, const void* o, const float* lse) {
  const int st = fa_validate_decode(q, k_pool, v_pool, page_table, ctx_lens, B, H, D, page_size,
                                    max_pages, num_pages, /*num_splits=*/1);
  if (st != FA_OK) return st;
  if (H_kv <= 0 || H % H_kv != 0) return FA_ERR_KV_HEADS;
  if (!prefix_table || !prefix_len || !o || !lse) return FA_ERR_NULL_POINTER;
  if (prefix_pages <= 0) return FA_ERR_MAX_PAGES;
  if (!aligned16(workspace) || !aligned16(o)) return FA_ERR_ALIGNMENT;
  const auto a4 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; };
  if (!a4(prefix_table) || !a4(prefix_len) || !a4(lse)) return FA_ERR_ALIGNMENT;
  // Positions within the prefix are 32-bit numbers; the chunks and the join have a
  // workgroup of 256 threads for a row (b, h) and some more, fewer than 2^32 threads.
  if (prefix_pages > (int64_t(1) << 27) - 8 || num_pages > kMaxGrid) return FA_ERR_TOO_LARGE;
  if (B * H >= int64_t(1) << 23) return FA_ERR_TOO_LARGE;
  if (!workspace && fa_decode_shared_workspace_floats(B, H, H_kv, D, prefix_pages, max_pages) > 0)
    return FA_ERR_NULL_POINTER;
  return FA_OK;
}

extern "C" int fa_validate_decode_weights(const void* q, const void* k_pool, const void* v_pool,
                                          const int32_t* page_table, const int32_t* ctx_lens,
                                          const float* weights, int64_t B, int64_t H, int64_t H_kv,
                                          int64_t D, int64_t page_size, int64_t max_pages,
                                          int64_t num_pages, const float* workspace, const void* o,
                                          const float* lse, const float* weights_out) {
  const int st = fa_validate_decode(q, k_pool, v_pool, page_table, ctx_lens, B, H, D, page_size,
                                    max_pages, num_pages, /*num_splits=*/1);
  if (st != FA_OK) return st;
  if (H_kv <= 0 || H % H_kv != 0) return FA_ERR_KV_HEADS;
  if (!weights || !weights_out || !o || !lse) return FA_ERR_NULL_POINTER;
  if (!workspace && fa_decode_weights_workspace_floats(B, H, H_kv, D, max_pages) > 0)
    return FA_ERR_NULL_POINTER;
  if (!aligned16(workspace) || !aligned16(o) || !aligned16(weights) || !aligned16(weights_out))
    return FA_ERR_ALIGNMENT;
  if (reinterpret_cast<uintptr_t>(lse) & 3u) return FA_ERR_ALIGNMENT;
  // The join has a workgroup of 256 threads for 1024 slots of a (b, KV head), and one
  // for a row: fewer than 2^32 threads.
  const int64_t chunks = (max_pages * 16 + 1023) / 1024, most = int64_t(1) << 23;
  if (num_pages > kMaxGrid || B * H >= most || B * H_kv > (most - 1) / chunks) return FA_ERR_TOO_LARGE;
  return FA_OK;
}

extern "C" int fa_validate_kv_evict(const void* k_pool, const void* v_pool, const int32_t* page_table,
                                    const int32_t* ctx_lens, const float* weights,
                                    const int32_t* new_page_table, const int32_t* kept,
                                    const float* new_weights, const int32_t* new_lens,
                                    const int32_t* bad, const int32_t* workspace, int64_t B,
                                    int64_t H_kv, int64_t D, int64_t keep, int64_t recent, int64_t page_size,
                                    int64_t max_pages, int64_t new_max_pages, int64_t num_pages) {
  if (!k_pool || !v_pool || !page_table || !ctx_lens || !weights || !new_page_table || !kept ||
      !new_weights || !new_lens || !bad)
    return FA_ERR_NULL_POINTER;
  if (!workspace && fa_kv_evict_workspace_words(B, H_kv, max_pages) > 0) return FA_ERR_NULL_POINTER;
  if (D != 64 && D != 128) return FA_ERR_HEAD_DIM;
  if (B <= 0 || H_kv <= 0) return FA_ERR_BATCH_HEADS;
  if (page_size != 16) return FA_ERR_PAGE_SIZE;
  if (max_pages <= 0 || new_max_pages <= 0) return FA_ERR_MAX_PAGES;
  if (num_pages <= 0) return FA_ERR_NUM_PAGES;
  if (!aligned16(k_pool) || !aligned16(v_pool)) return FA_ERR_ALIGNMENT;
  const void* words[] = {page_table, ctx_lens, weights, new_page_table, kept, new_weights, new_lens, bad,
                         workspace};
  for (const void* p : words)
    if (reinterpret_cast<uintptr_t>(p) & 3u) return FA_ERR_ALIGNMENT;
  if (B > 65535 || H_kv > 65535 || num_pages > kMaxGrid) return FA_ERR_TOO_LARGE;
  // Slots are 32-bit numbers, and a thread's steps of 1024 past the last one too; the
  // copy has up to 16 threads for a new slot, fewer than 2^32.
  if (max_pages > (int64_t(1) << 27) - 128 || new_max_pages > (int64_t(1) << 24) - 128) return FA_ERR_TOO_LARGE;
  if (keep < 1 || keep > new_max_pages * 16 || recent < 0 || recent > keep) return FA_ERR_BUDGET;
  return FA_OK;
}
