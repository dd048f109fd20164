// fa_cache.hip — a paged cache kept within a budget, for MI355X: the decode that
// adds up how much attention each cached token gets, and the eviction that
// packs a head's newest and heaviest tokens into new pages.
//
// No reference counterpart (the reference has no KV cache). Of a decode step,
// token j of sequence b gets from the G query heads that share a KV head
//   W'[j] = W[j] + sum_g exp(s_gj - L_g),
// s the scaled scores and L their logsumexp over the whole context. L is known
// only after the last key, so the split pass keeps its scores (4 G bytes a token
// and KV head beside the 4 D of its K and V rows) and the launch that joins the
// splits turns them into weights; a second pass over K would read 2 D bytes.
#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include "fa_decode.hpp"
#include "fa_mi355x.h"
#include "fa_pages.hpp"
#include "fa_tile.hpp"

namespace fa {
namespace cache {

using pages::kPageSize;
constexpr int kThreads = 256;
constexpr int kMaxSplits = 16;

template <int D, bool BF16>
__global__ void __launch_bounds__(kDecThreads)
fa_weights_split_kernel(const typename DecT<BF16>::e* __restrict__ q,
                        const typename DecT<BF16>::e* __restrict__ kpool,
                        const typename DecT<BF16>::e* __restrict__ vpool,
                        const int32_t* __restrict__ page_table,
                        const int32_t* __restrict__ ctx_lens, float* __restrict__ part_o,
                        float* __restrict__ part_ml, float* __restrict__ scores, int H, int Hkv,
                        int max_pages, int num_pages, int S, int ordered, float c) {
  __shared__ DecShared<D> sh;
  decode_split_body<D, BF16, true, true>(sh, blockIdx.x, blockIdx.y, blockIdx.z, gridDim.z, q, kpool,
                                         vpool, page_table, ctx_lens, part_o, part_ml, nullptr, nullptr,
                                         H, Hkv, max_pages, num_pages, S, ordered, c, scores);
}

// Maximum and sum over a row's S splits, in units of log 2: (-inf, 0) where all
// are empty, a NaN sum where one is.
__device__ __forceinline__ float2 join_splits(const float2* __restrict__ ml, int S) {
  float2 x[kMaxSplits];
#pragma unroll
  for (int s = 0; s < kMaxSplits; ++s) x[s] = s < S ? ml[s] : make_float2(-INFINITY, 0.f);
  float M = -INFINITY, z = 0.f;
#pragma unroll
  for (int s = 0; s < kMaxSplits; ++s) M = fmaxf(M, x[s].x);
#pragma unroll
  for (int s = 0; s < kMaxSplits; ++s) z += x[s].x == -INFINITY ? x[s].y : x[s].y * exp2_hw(x[s].x - M);
  return make_float2(M, z);
}

constexpr int kChunk = 4 * kThreads;   // slots of a workgroup that writes weights

// Workgroups [0, rows): O and L of one row (b, h) out of its S partials. The
// others: weights of kChunk slots of one (b, KV head), group heads in order, so
// the same call gives the same bits.
template <int D, bool BF16>
__global__ void __launch_bounds__(kThreads)
fa_weights_join_kernel(const float* __restrict__ part_o, const float2* __restrict__ part_ml,
                       const float* __restrict__ scores, const int32_t* __restrict__ ctx_lens,
                       const float* w_in, float* w_out, typename DecT<BF16>::e* __restrict__ o,
                       float* __restrict__ lse, int H, int Hkv, int max_pages, int S, int rows,
                       int row_blocks, int chunks) {
  typedef typename DecT<BF16>::e e4 __attribute__((ext_vector_type(4)));
  const int tid = threadIdx.x;
  constexpr int PER = D / 4;
  if ((int)blockIdx.x < row_blocks) {
    const int row = blockIdx.x * (kThreads / PER) + tid / PER;
    if (row >= rows) return;
    const int d = 4 * (tid % PER);
    const float2* ml = part_ml + (size_t)row * S;
    const float* po = part_o + (size_t)row * S * D + d;
    f32x4 ps[kMaxSplits];
#pragma unroll
    for (int s = 0; s < kMaxSplits; ++s)
      ps[s] = s < S ? *reinterpret_cast<const f32x4*>(po + (size_t)s * D) : f32x4{};
    const float2 J = join_splits(ml, S);
    f32x4 out = f32x4{};
    if (J.y != 0.f) {   // a NaN sum: NaN
      const float inv = 1.f / J.y;
#pragma unroll
      for (int s = 0; s < kMaxSplits; ++s) {
        if (s < S) {
          const float2 x = ml[s];
          const float w = x.x == -INFINITY ? x.y : x.y * exp2_hw(x.x - J.x) * inv;
#pragma unroll
          for (int i = 0; i < 4; ++i) out[i] = fmaf(w, ps[s][i], out[i]);
        }
      }
    }
    e4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (typename DecT<BF16>::e)out[i];
    *reinterpret_cast<e4*>(o + (size_t)row * D + d) = v;
    if (d == 0) lse[row] = J.y == 0.f ? -INFINITY : (J.x + log2_hw(J.y)) * kLn2;
    return;
  }
  const int unit = (int)blockIdx.x - row_blocks;
  const int bh = unit / chunks;   // b * Hkv + hk
  const int b = bh / Hkv, hk = bh - b * Hkv;
  const int G = H / Hkv;
  const int64_t width = (int64_t)max_pages * kPageSize;
  const int64_t first = (int64_t)(unit - bh * chunks) * kChunk;
  int64_t ctx = ctx_lens[b];
  ctx = ctx < 0 ? 0 : (ctx > width ? width : ctx);
  const bool in_place = w_in == w_out;
  if (first >= ctx && in_place) return;
  const int64_t j = first + 4 * tid;
  const bool there = j < width;   // width is a multiple of 16
  const int64_t at = (int64_t)bh * width + j;
  f32x4 w = f32x4{};
  if (there) w = *reinterpret_cast<const f32x4*>(w_in + at);
  if (first < ctx) {
    __shared__ float M[kThreads], inv[kThreads];   // of a group's heads
    f32x4 sum = f32x4{};
    for (int g0 = 0; g0 < G; g0 += kThreads) {
      const int gs = min(kThreads, G - g0);
      if (g0 > 0) __syncthreads();
      if (tid < gs) {
        const float2 J = join_splits(part_ml + ((size_t)b * H + (size_t)hk * G + g0 + tid) * S, S);
        M[tid] = J.x;
        inv[tid] = 1.f / J.y;
      }
      __syncthreads();
      if (there && j < ctx) {
        const float* sc = scores + ((size_t)b * H + (size_t)hk * G + g0) * width + j;
#pragma unroll 4
        for (int g = 0; g < gs; ++g) {
          const f32x4 x = *reinterpret_cast<const f32x4*>(sc + (size_t)g * width);
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[i] = fmaf(exp2_hw(x[i] - M[g]), inv[g], sum[i]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (j + i < ctx) w[i] += sum[i];
  }
  if (there) *reinterpret_cast<f32x4*>(w_out + at) = w;
}

template <bool BF16>
static int decode_weights(const void* q, const void* k_pool, const void* v_pool,
                          const int32_t* page_table, const int32_t* ctx_lens, const float* w_in,
                          int64_t B, int64_t H, int64_t Hkv, int64_t D, int64_t max_pages,
                          int64_t num_pages, int64_t S, float* ws, void* o, float* lse, float* w_out,
                          void* stream) {
  using E = typename DecT<BF16>::e;
  const float c = (float)(1.0 / sqrt((double)D)) * kLog2e;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int64_t width = max_pages * kPageSize, rows = B * H;
  float* scores = ws;   // first: 16-byte aligned rows
  float* part_o = scores + rows * width;
  float* part_ml = part_o + rows * S * D;
  const dim3 grid((unsigned)S, (unsigned)decode_head_groups(H, Hkv), (unsigned)B);
  const int ordered = decode_ordered(B, H, Hkv, D, S, stream_topology(s).cus);
  const int64_t row_blocks = (rows + kThreads / (D / 4) - 1) / (kThreads / (D / 4));
  const int64_t chunks = (width + kChunk - 1) / kChunk;
  const int64_t join = row_blocks + B * Hkv * chunks;
#define FA_WEIGHTS(DD)                                                                             \
  do {                                                                                             \
    hipLaunchKernelGGL((fa_weights_split_kernel<DD, BF16>), grid, dim3(kDecThreads), 0, s,         \
                       (const E*)q, (const E*)k_pool, (const E*)v_pool, page_table, ctx_lens,      \
                       part_o, part_ml, scores, (int)H, (int)Hkv, (int)max_pages, (int)num_pages, \
                       (int)S, ordered, c);                                                        \
    hipLaunchKernelGGL((fa_weights_join_kernel<DD, BF16>), dim3((unsigned)join), dim3(kThreads), 0, \
                       s, part_o, (const float2*)part_ml, scores, ctx_lens, w_in, w_out, (E*)o, lse, (int)H,     \
                       (int)Hkv, (int)max_pages, (int)S, (int)rows, (int)row_blocks, (int)chunks); \
  } while (0)
  if (D == 128) FA_WEIGHTS(128);
  else FA_WEIGHTS(64);
#undef FA_WEIGHTS
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? FA_OK : -(int)e;
}

// ---------------------------------------------------------------------------
// Eviction
// ---------------------------------------------------------------------------
// Order of weights as unsigned numbers: larger weight, larger key; -0 as 0, a NaN
// below every number.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0;
  const uint32_t u = __float_as_uint(w == 0.f ? 0.f : w);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / 64;
constexpr int kCopies = 16;   // histograms side by side: lanes of a wave share a counter four at most

// One workgroup per (b, KV head): which tokens stay. The `recent` last ones do,
// and of the others the keep - recent heaviest: the key of the last of these is
// found digit by digit (8 bits, histograms in LDS), equal ones stay from the
// lowest slot on. Then the stayers are written out in order, waves taking one
// run of slots each.
__global__ void __launch_bounds__(kSelThreads)
fa_evict_select_kernel(const float* __restrict__ weights, const int32_t* __restrict__ ctx_lens,
                       int32_t* __restrict__ kept, float* __restrict__ w_new,
                       int32_t* __restrict__ new_lens, int32_t* __restrict__ bad, int Hkv,
                       int max_pages, int keep, int recent, int new_width) {
  __shared__ uint32_t hist[256 * kCopies];
  __shared__ uint32_t sh_digit, sh_above;
  __shared__ int sh_gt[kSelWaves], sh_eq[kSelWaves];
  const int hk = blockIdx.x, b = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t width = (int64_t)max_pages * kPageSize;
  const size_t bh = (size_t)b * Hkv + hk;
  int n = ctx_lens[b];
  const bool invalid = n < 0 || n > width;
  if (invalid) n = 0;
  const int m = min(n, keep);
  const float* w = weights + bh * width;
  int32_t* kp = kept + bh * keep;
  float* wn = w_new + bh * new_width;
  if (hk == 0 && tid == 0) {
    new_lens[b] = m;
    bad[b] = invalid;
  }
  for (int j = m + tid; j < new_width; j += kSelThreads) {
    wn[j] = 0.f;
    if (j < keep) kp[j] = -1;
  }
  if (n <= keep) {
    for (int j = tid; j < m; j += kSelThreads) {
      kp[j] = j;
      wn[j] = w[j];
    }
    return;
  }
  const int cand = n - recent, need = keep - recent;   // 0 <= need < cand
  for (int j = tid; j < recent; j += kSelThreads) {
    kp[need + j] = cand + j;
    wn[need + j] = w[cand + j];
  }
  if (need == 0) return;
  uint32_t prefix = 0;   // digits of the threshold found so far
  int left = need;       // of the tokens that share them, how many stay
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256 * kCopies; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    for (int j = tid; j < cand; j += kSelThreads) {
      const uint32_t k = weight_key(w[j]);
      if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8)))
        atomicAdd(&hist[((k >> shift) & 255) * kCopies + (lane & (kCopies - 1))], 1u);
    }
    __syncthreads();
    // Wave 0: lane l has digits 255 - 4 l down to 252 - 4 l.
    if (wave == 0) {
      uint32_t c[4], sum = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        c[i] = 0;
        for (int x = 0; x < kCopies; ++x) c[i] += hist[(255 - 4 * lane - i) * kCopies + x];
        sum += c[i];
      }
      uint32_t above = (uint32_t)scan_sum((int)sum) - sum;   // tokens of larger digits
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (above < (uint32_t)left && above + c[i] >= (uint32_t)left) {   // exactly one lane and i
          sh_digit = 255 - 4 * lane - i;
          sh_above = above;
        }
        above += c[i];
      }
    }
    __syncthreads();
    prefix |= sh_digit << shift;
    left -= (int)sh_above;
  }
  // Keys above `prefix` stay, and the first `left` equal to it.
  const int run = (cand + kSelWaves * 64 - 1) / (kSelWaves * 64) * 64;   // slots of a wave
  const int lo = min(wave * run, cand), hi = min(lo + run, cand);
  int gt = 0, eq = 0;
  for (int j0 = lo; j0 < hi; j0 += 64) {
    const int j = j0 + lane;
    const uint32_t k = j < hi ? weight_key(w[j]) : 0;
    gt += __popcll(__ballot(j < hi && k > prefix));
    eq += __popcll(__ballot(j < hi && k == prefix));
  }
  if (lane == 0) {
    sh_gt[wave] = gt;
    sh_eq[wave] = eq;
  }
  __syncthreads();
  gt = eq = 0;
  for (int i = 0; i < wave; ++i) {
    gt += sh_gt[i];
    eq += sh_eq[i];
  }
  const uint64_t below = ((uint64_t)1 << lane) - 1;
  for (int j0 = lo; j0 < hi; j0 += 64) {
    const int j = j0 + lane;
    const float x = j < hi ? w[j] : 0.f;
    const uint32_t k = weight_key(x);
    const uint64_t mg = __ballot(j < hi && k > prefix), me = __ballot(j < hi && k == prefix);
    const int g = gt + __popcll(mg & below), e = eq + __popcll(me & below);
    const bool is_eq = (me >> lane) & 1;
    if (((mg >> lane) & 1) || (is_eq && e < left)) {
      const int at = g + min(e, left);
      kp[at] = j;
      wn[at] = x;
    }
    gt += __popcll(mg);
    eq += __popcll(me);
  }
}

constexpr int kMoveRows = 4;   // rows a thread has in flight

// The stayers' rows into the new pages: 16-byte pieces, each row read and
// written once. Bound: memory, by the gather of 2 D byte rows.
template <int D>
__global__ void __launch_bounds__(kThreads)
fa_evict_move_kernel(uint4* k_pool, uint4* v_pool, const int32_t* __restrict__ page_table,
                     const int32_t* __restrict__ new_table, const int32_t* __restrict__ kept,
                     int32_t* __restrict__ bad, int Hkv, int max_pages, int new_max_pages,
                     int num_pages, int keep) {
  constexpr int CH = D / 8;            // pieces of a row
  constexpr int SIDE = kThreads / CH;  // rows side by side
  const int hk = blockIdx.y, b = blockIdx.z;
  const int c = (int)threadIdx.x % CH;
  const int32_t* kp = kept + ((size_t)b * Hkv + hk) * keep;
  uint4 x[kMoveRows], y[kMoveRows];
  int64_t dst[kMoveRows];
#pragma unroll
  for (int i = 0; i < kMoveRows; ++i) {
    const int j = ((int)blockIdx.x * kMoveRows + i) * SIDE + (int)threadIdx.x / CH;
    dst[i] = -1;
    const int old = j < keep ? kp[j] : -1;
    if (old >= 0) {
      const int from = page_table[(size_t)b * max_pages + old / kPageSize];
      const int to = new_table[(size_t)b * new_max_pages + j / kPageSize];
      if (from >= 0 && from < num_pages && to >= 0 && to < num_pages) {
        const int64_t src = (((int64_t)from * Hkv + hk) * kPageSize + old % kPageSize) * CH + c;
        dst[i] = (((int64_t)to * Hkv + hk) * kPageSize + j % kPageSize) * CH + c;
        x[i] = k_pool[src];
        y[i] = v_pool[src];
      } else if (c == 0) {
        bad[b] = 1;   // the same value from every writer
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kMoveRows; ++i) {
    if (dst[i] >= 0) {
      k_pool[dst[i]] = x[i];
      v_pool[dst[i]] = y[i];
    }
  }
}

}  // namespace cache
}  // namespace fa

extern "C" int64_t fa_decode_weights_workspace_floats(int64_t B, int64_t H, int64_t D,
                                                      int64_t max_pages, int64_t num_splits) {
  if (B <= 0 || H <= 0 || D <= 0 || max_pages <= 0 || num_splits <= 0) return 0;
  return B * H * (max_pages * 16 + num_splits * (D + 2));
}

extern "C" int fa_decode_paged_weights(const void* q, const void* k_pool, const void* v_pool,
                                       const int32_t* page_table, const int32_t* ctx_lens,
                                       const float* weights, int64_t B, int64_t H, int64_t H_kv,
                                       int64_t D, int64_t page_size, int64_t max_pages,
                                       int64_t num_pages, int64_t num_splits, float* workspace,
                                       void* o, float* lse, float* weights_out, int bf16,
                                       void* stream) {
  const int st = fa_validate_decode_weights(q, k_pool, v_pool, page_table, ctx_lens, weights, B, H,
                                            H_kv, D, page_size, max_pages, num_pages, num_splits,
                                            workspace, o, lse, weights_out);
  if (st != FA_OK) return st;
  const auto fn = bf16 ? fa::cache::decode_weights<true> : fa::cache::decode_weights<false>;
  return fn(q, k_pool, v_pool, page_table, ctx_lens, weights, B, H, H_kv, D, max_pages, num_pages,
            num_splits, workspace, o, lse, weights_out, stream);
}

extern "C" int fa_kv_evict(void* k_pool, void* v_pool, const int32_t* page_table,
                           const int32_t* ctx_lens, const float* weights,
                           const int32_t* new_page_table, int32_t* kept, float* new_weights,
                           int32_t* new_lens, int32_t* bad, int64_t B, int64_t H_kv, int64_t D,
                           int64_t keep, int64_t recent, int64_t page_size, int64_t max_pages,
                           int64_t new_max_pages, int64_t num_pages, void* stream) {
  using namespace fa::cache;
  const int st = fa_validate_kv_evict(k_pool, v_pool, page_table, ctx_lens, weights, new_page_table,
                                      kept, new_weights, new_lens, bad, B, H_kv, D, keep, recent,
                                      page_size, max_pages, new_max_pages, num_pages);
  if (st != FA_OK) return st;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(fa_evict_select_kernel, dim3((unsigned)H_kv, (unsigned)B), dim3(kSelThreads), 0,
                     s, weights, ctx_lens, kept, new_weights, new_lens, bad, (int)H_kv,
                     (int)max_pages, (int)keep, (int)recent, (int)(new_max_pages * kPageSize));
  const int64_t rows = kMoveRows * (kThreads / (D / 8));
  const dim3 grid((unsigned)((keep + rows - 1) / rows), (unsigned)H_kv, (unsigned)B);
#define FA_MOVE(DD)                                                                                \
  hipLaunchKernelGGL((fa_evict_move_kernel<DD>), grid, dim3(kThreads), 0, s, (uint4*)k_pool,       \
                     (uint4*)v_pool, page_table, new_page_table, kept, bad, (int)H_kv,             \
                     (int)max_pages, (int)new_max_pages, (int)num_pages, (int)keep)
  if (D == 128) FA_MOVE(128);
  else FA_MOVE(64);
#undef FA_MOVE
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? FA_OK : -(int)e;
}
