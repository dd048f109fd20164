// fa_cache.hip — a paged cache kept within a budget, for MI355X: the decode that
// adds up how much attention each cached token gets, and the eviction that
// packs a head's newest and heaviest tokens into new pages.
//
// No reference counterpart (the reference has no KV cache). Of a decode step,
// token j of sequence b gets from the G query heads that share a KV head
//   W'[j] = W[j] + sum_g exp(s_gj - L_g),
// s the scaled scores and L their logsumexp over the whole context. L is known
// only after the last key, so the chunk pass keeps its scores (4 G bytes a token
// and KV head beside the 4 D of its K and V rows) and the launch that joins the
// chunks turns them into weights; a second pass over K would read 2 D bytes.
//
// Bound: memory. 16 sequences of 2000 to 32768 tokens, H32 over 8, D = 128 (1.14 GB
// of K and V, 36 MB of scores written and read again): 227 us, the chunks 215 and the join
// 13; without their scores the chunks take 186 us, and the decode without weights 180.
#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include "fa_mi355x.h"
#include "fa_pages.hpp"
#include "fa_stream.hpp"
#include "fa_tile.hpp"

namespace fa {
namespace cache {

using namespace stream;
using pages::kPageSize;

// What the scores of a head are turned into weights by, from their maximum and sum: (maximum, 1 /
// sum). Where every score is -inf, O is 0, L -inf and every weight 0: (0, 0), as -inf has no
// difference to itself; a NaN sum keeps its NaN.
__device__ __forceinline__ float2 by_head(float m, float z) {
  return make_float2(m == -INFINITY ? 0.f : m, z == 0.f ? 0.f : 1.f / z);
}

template <int D, bool BF16, bool NT>
__global__ void __launch_bounds__(stream::kThreads)
fa_weights_chunk_kernel(const uint16_t* __restrict__ q, const char* __restrict__ k_pool,
                        const char* __restrict__ v_pool, const int32_t* __restrict__ page_table,
                        const int32_t* __restrict__ ctx_lens, const int4* __restrict__ table,
                        float* __restrict__ part_o, float2* __restrict__ part_ml,
                        int2* __restrict__ first, float* __restrict__ scores, int B, int H, int Hkv,
                        int group, int ngrp, int max_pages, int num_pages, Plan plan, float c) {
  __shared__ Shared<D> sh;
  const Place at = place_of(blockIdx.x, Hkv * ngrp);
  const Run r = run_of(ctx_lens, table, B, max_pages, plan, at.number);
  if (r.b < 0) return;
  if (at.hg == 0 && r.split == 0 && threadIdx.x == 0) first[r.b] = make_int2(at.number, r.splits);
  const int hk = at.hg / ngrp, sub = at.hg - hk * ngrp, col = threadIdx.x & 15;
  const int h = hk * group + 16 * sub + col;
  const bool live = 16 * sub + col < group;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t width = (int64_t)max_pages * kPageSize;
  const ScoresOut scores_out{scores + ((int64_t)r.b * H + h - col) * width, width, min(16, group - 16 * sub)};
  const PartOut<D> out{part_o, part_ml, (int64_t)at.number * H + h};
  chunk_body<D, BF16, NT>(sh, wave, q, k_pool, v_pool, Pages{page_table + (size_t)r.b * max_pages, r.ctx},
                          r.p0, r.p1, r.bad, live, ((int64_t)r.b * H + h) * D, hk, Hkv, num_pages, c,
                          scores_out, out, out);
}

// Short contexts, a workgroup of kOneWaves waves for a sequence and KV head: the scores
// stay in LDS until the sums are known, and one launch writes everything. Taken for tables
// of up to kOnePages pages and up to two workgroups a CU. A call by itself, us, in one
// launch and in chunks: D = 64, 64 workgroups, 4 pages 3.9 and 8.4, 32 pages 6.3 and 8.8;
// D = 128, 256 workgroups, 4 pages 4.8 and 9.5, 32 pages 10.7 and 15.0; 1024 workgroups
// of 24 pages 34.1 and 34.3.
constexpr int kOneWaves = 8;
constexpr int kOnePages = 32, kOneBlocks = 512;

template <int D, bool BF16>
__global__ void __launch_bounds__(64 * kOneWaves)
fa_weights_one_kernel(const uint16_t* __restrict__ q, const char* __restrict__ k_pool,
                      const char* __restrict__ v_pool, const int32_t* __restrict__ page_table,
                      const int32_t* __restrict__ ctx_lens, const float* w_in, float* w_out,
                      uint16_t* __restrict__ o, float* __restrict__ lse, int H, int Hkv, int max_pages,
                      int num_pages, float c) {
  constexpr int STRIDE = kOnePages * kTokens + 4;
  __shared__ Shared<D, kOneWaves> sh;
  __shared__ __attribute__((aligned(16))) float scores[16 * STRIDE];
  __shared__ float2 J[16];   // of a group's heads, see by_head
  const int hk = blockIdx.x, b = blockIdx.y, G = H / Hkv;
  const int col = threadIdx.x & 15, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ctx = __builtin_amdgcn_readfirstlane(ctx_lens[b]), pages = pages_of(ctx, max_pages);
  const bool live = col < G;
  const int64_t row = (int64_t)b * H + hk * G + col;
  const RowOut<D, BF16> out{o, lse, row, c};
  chunk_body<D, BF16, false>(sh, wave, q, k_pool, v_pool, Pages{page_table + (size_t)b * max_pages, ctx}, 0,
                             pages, ctx < 0 || (ctx > 0 && pages == 0), live, row * D, hk, Hkv, num_pages,
                             c, ScoresKept{scores, STRIDE}, out, [&](float m, float z) {
                               out(m, z);
                               J[col] = by_head(m, z);
                             });
  __syncthreads();
  const int width = max_pages * kPageSize, n = min(max(ctx, 0), width);
  const int64_t at = ((int64_t)b * Hkv + hk) * width;
  for (int j = threadIdx.x; j < (w_in == w_out ? n : width); j += 64 * kOneWaves) {
    float w = w_in[at + j];
    if (j < n) {
      float sum = 0.f;
      for (int g = 0; g < G; ++g) sum = fmaf(exp2_hw((scores[g * STRIDE + j] - J[g].x) * c), J[g].y, sum);
      w += sum;
    }
    w_out[at + j] = w;
  }
}

constexpr int kChunk = 4 * kJoinThreads;   // slots of a workgroup that writes weights

// Workgroups [0, rows): O and L of one row (b, h) out of its chunks. The others:
// weights of kChunk slots of one (b, KV head), group heads in order, so the same
// call gives the same bits.
template <int D, bool BF16>
__global__ void __launch_bounds__(kJoinThreads)
fa_weights_join_kernel(const float* __restrict__ part_o, const float2* __restrict__ part_ml,
                       const int2* __restrict__ first_of, const float* __restrict__ scores,
                       const int32_t* __restrict__ ctx_lens, const float* w_in, float* w_out,
                       uint16_t* __restrict__ o, float* __restrict__ lse, int H, int Hkv,
                       int max_pages, int rows, int chunks, float c) {
  const int tid = threadIdx.x, wave = tid >> 6;
  if ((int)blockIdx.x < rows) {
    __shared__ JoinShared<D> sh;
    const int row = blockIdx.x, b = row / H;
    const int2 f = first_of[b];
    const Parts a{part_o, part_ml, (int64_t)f.x * H + (row - b * H), H, f.y};
    join_row<D, BF16>(sh, a, Parts{part_o, part_ml, 0, 0, 0}, c, o + (int64_t)row * D, lse + row);
    return;
  }
  const int unit = (int)blockIdx.x - rows;
  const int bh = unit / chunks;   // b * Hkv + hk
  const int b = bh / Hkv, hk = bh - b * Hkv;
  const int G = H / Hkv;
  const int64_t width = (int64_t)max_pages * kPageSize;
  const int64_t start = (int64_t)(unit - bh * chunks) * kChunk;
  int64_t ctx = ctx_lens[b];
  ctx = ctx < 0 ? 0 : (ctx > width ? width : ctx);
  if (start >= ctx && w_in == w_out) return;
  const int64_t j = start + 4 * tid;
  const bool there = j < width;   // width is a multiple of 16
  const int64_t at = (int64_t)bh * width + j;
  f32x4 w = f32x4{};
  if (there) w = *reinterpret_cast<const f32x4*>(w_in + at);
  if (start < ctx) {
    __shared__ float2 J[kJoinThreads];   // of a group's heads, see by_head
    const int2 f = first_of[b];
    f32x4 sum = f32x4{};
    for (int g0 = 0; g0 < G; g0 += kJoinThreads) {
      const int gs = min(kJoinThreads, G - g0);
      if (g0 > 0) __syncthreads();
      for (int g = wave; g < gs; g += kJoinThreads / 64) {
        const float2 x = join_wave(Parts{part_o, part_ml, (int64_t)f.x * H + hk * G + g0 + g, H, f.y}, c);
        if ((tid & 63) == 0) J[g] = by_head(x.x, x.y);
      }
      __syncthreads();
      if (there && j < ctx) {
        const float* sc = scores + ((int64_t)b * H + hk * G + g0) * width + j;
#pragma unroll 4
        for (int g = 0; g < gs; ++g) {
          const f32x4 x = *reinterpret_cast<const f32x4*>(sc + g * width);
          const float2 Jg = J[g];
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[i] = fmaf(exp2_hw((x[i] - Jg.x) * c), Jg.y, sum[i]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (j + i < ctx) w[i] += sum[i];
  }
  if (there) *reinterpret_cast<f32x4*>(w_out + at) = w;
}

// Whether a call is one launch.
static bool in_one(int64_t B, int64_t H, int64_t Hkv, int64_t max_pages) {
  return max_pages <= kOnePages && H / Hkv <= 16 && B * Hkv <= kOneBlocks;
}

// The workspace, in floats: the scores first, then the
// chunks' partial O, their maxima and sums, the sequences' first chunks and, of
// more sequences than a wave plans, the table of chunks.
struct Workspace {
  int64_t most, part_o, part_ml, first, table, floats;
};
static Workspace workspace_of(int64_t B, int64_t H, int64_t Hkv, int64_t D, int64_t max_pages) {
  Workspace w;
  w.most = most_chunks(B, max_pages, plan_of(head_groups(H, Hkv)));
  w.part_o = B * H * max_pages * kPageSize;
  w.part_ml = w.part_o + w.most * H * D;
  w.table = w.part_ml + (2 * w.most * H + 3) / 4 * 4;
  w.first = w.table + (B > kWavePlan ? 4 * (1 + w.most) : 0);
  w.floats = w.first + 2 * B;
  return w;
}

template <int D, bool BF16>
static int decode_weights(const void* q, const void* k_pool, const void* v_pool,
                          const int32_t* page_table, const int32_t* ctx_lens, const float* w_in,
                          int64_t B, int64_t H, int64_t Hkv, int64_t max_pages, int64_t num_pages,
                          float* ws, void* o, float* lse, float* w_out, void* stream) {
  const float c = (float)(1.0 / sqrt((double)D)) * kLog2e;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (in_one(B, H, Hkv, max_pages)) {
    hipLaunchKernelGGL((fa_weights_one_kernel<D, BF16>), dim3((unsigned)Hkv, (unsigned)B),
                       dim3(64 * kOneWaves), 0, s, (const uint16_t*)q, (const char*)k_pool,
                       (const char*)v_pool, page_table, ctx_lens, w_in, w_out, (uint16_t*)o, lse, (int)H,
                       (int)Hkv, (int)max_pages, (int)num_pages, c);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? FA_OK : -(int)e;
  }
  const Workspace w = workspace_of(B, H, Hkv, D, max_pages);
  const int64_t groups = head_groups(H, Hkv), rows = B * H;
  const Plan plan = plan_of(groups);
  float* part_o = ws + w.part_o;
  float2* part_ml = (float2*)(ws + w.part_ml);
  int2* first = (int2*)(ws + w.first);
  int4* table = B > kWavePlan ? (int4*)(ws + w.table) : nullptr;
  if (table != nullptr)
    hipLaunchKernelGGL(fa_stream_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, ctx_lens, (int)B,
                       (int)max_pages, plan, table);
  const bool nt = pass_through(num_pages, Hkv, D);
  const auto kernel = nt ? fa_weights_chunk_kernel<D, BF16, true> : fa_weights_chunk_kernel<D, BF16, false>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)chunk_blocks(w.most, groups)), dim3(stream::kThreads), 0, s,
                     (const uint16_t*)q, (const char*)k_pool, (const char*)v_pool, page_table, ctx_lens,
                     table, part_o, part_ml, first, ws, (int)B, (int)H, (int)Hkv, (int)(H / Hkv),
                     (int)(groups / Hkv), (int)max_pages, (int)num_pages, plan, c);
  const int64_t chunks = (max_pages * kPageSize + kChunk - 1) / kChunk;
  hipLaunchKernelGGL((fa_weights_join_kernel<D, BF16>), dim3((unsigned)(rows + B * Hkv * chunks)),
                     dim3(kJoinThreads), 0, s, part_o, part_ml, first, ws, ctx_lens, w_in, w_out,
                     (uint16_t*)o, lse, (int)H, (int)Hkv, (int)max_pages, (int)rows, (int)chunks, c);
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
constexpr int kBins = 2048, kCopies = 4;   // counters of a digit, side by side for lanes of a wave
constexpr int kMostKeys = 32;              // of a thread's keys in registers
constexpr int kListKeys = 4;               // up to which the selection also lists the stayers

// Sum of the first `waves` of a workgroup's waves' counts, by a whole wave.
__device__ __forceinline__ int sum_before(const int* sh, int waves) {
  const int lane = threadIdx.x & 63;
  return __builtin_amdgcn_readlane(scan_sum(lane < waves ? sh[lane] : 0), 63);
}

// What is known of a (b, KV head) after its selection: tokens with keys above
// `key` stay, and of those equal to it the first `left`. The candidates, all but
// the newest tokens, are cut into kSelWaves runs of `per` slots; gt and eq count the
// keys above and equal before a run.
struct Selection {
  int n, cand, per, left;   // n: the length, 0 of an invalid one; cand 0: every token stays
  uint32_t key;
  int gt[kSelWaves], eq[kSelWaves];
};
constexpr int kSelWords = sizeof(Selection) / 4;

// One workgroup per (b, KV head): which tokens stay. The `recent` last ones do,
// and of the others the keep - recent heaviest: the key of the last of these is
// found digit by digit (11, 11 and 10 bits, histograms in LDS). A wave has one run of
// slots, 64 E of them in registers, read once and all at a time; E = 0: longer
// tables, read again for every digit. Slots that there are not have the lowest key:
// beside real ones they come last, so none of them ever stays. With up to kListKeys
// keys a thread it also writes the stayers' old slots and weights, in order; beyond,
// that is spread over the chip (fa_evict_list_kernel: 32000 slots of 64 heads 28 us in
// one launch, 15.0 + 5.5 in two; 1100 slots of 32 heads 6.1, and 6.1 + 3.6).
template <int E>
__global__ void __launch_bounds__(kSelThreads)
fa_evict_select_kernel(const float* __restrict__ weights, const int32_t* __restrict__ ctx_lens,
                       int32_t* __restrict__ kept, float* __restrict__ w_new,
                       int32_t* __restrict__ new_lens, int32_t* __restrict__ bad,
                       Selection* __restrict__ out, int Hkv, int max_pages, int keep, int recent,
                       int new_width) {
  constexpr int N = E > 0 ? E : 1;
  __shared__ __attribute__((aligned(16))) uint32_t hist[kBins * kCopies];
  __shared__ uint32_t sh_digit, sh_above;
  __shared__ int sh_sum[kSelWaves], sh_gt[kSelWaves], sh_eq[kSelWaves];
  const int hk = blockIdx.x, b = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int width = max_pages * kPageSize;
  const size_t bh = (size_t)b * Hkv + hk;
  const float* w = weights + bh * width;
  int n = ctx_lens[b];
  const bool invalid = n < 0 || n > width;
  if (invalid) n = 0;
  const int m = min(n, keep);
  for (int j = m + tid; j < new_width; j += kSelThreads) {
    w_new[bh * new_width + j] = 0.f;
    if (j < keep) kept[bh * keep + j] = -1;
  }
  const int cand = n > keep ? n - recent : 0, need = keep - recent;   // 0 <= need < cand
  constexpr bool LIST = E > 0 && E <= kListKeys;
  if (tid == 0) {
    if constexpr (!LIST) {
      out[bh].n = n;
      out[bh].cand = cand;
    }
    if (hk == 0) {
      new_lens[b] = m;
      bad[b] = invalid;
    }
  }
  if constexpr (LIST) {   // those that stay unseen
    const int stay = cand > 0 ? recent : n, to = cand > 0 ? need : 0;
    for (int j = tid; j < stay; j += kSelThreads) {
      kept[bh * keep + to + j] = cand + j;
      w_new[bh * new_width + to + j] = w[cand + j];
    }
  }
  if (cand == 0) return;
  // The wave's slots lo + 64 i + lane < hi: as many for every wave, so that their
  // runs give the packing workgroups of like size.
  const int per = (cand + kSelWaves * 64 - 1) / (kSelWaves * 64) * 64;   // at most 64 E
  const int lo = min(wave * per, cand), hi = min(lo + per, cand);
  uint32_t key[N];
  if constexpr (E > 0) {
    float x[N];
#pragma unroll
    for (int i = 0; i < E; ++i) x[i] = w[min(lo + 64 * i + lane, cand - 1)];
#pragma unroll
    for (int i = 0; i < E; ++i) key[i] = lo + 64 * i + lane < hi ? weight_key(x[i]) : 0;
  }
  const auto each = [&](auto&& f) {   // f(first slot of 64 - lo, key)
    if constexpr (E > 0) {
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (lo + 64 * i < hi) f(64 * i, key[i]);
    } else {
      for (int j = lo; j < hi; j += 64) f(j - lo, j + lane < hi ? weight_key(w[j + lane]) : 0);
    }
  };
  // Thread t has the counters of bins 2047 - 2 t and one below.
  u32x4* const mine = reinterpret_cast<u32x4*>(hist + (kBins - 2 - 2 * tid) * kCopies);
  mine[0] = mine[1] = u32x4{};
  uint32_t prefix = 0;   // digits of the threshold found so far
  int left = need;       // of the tokens that share them, how many stay
  for (int pass = 0; pass < 3 && need > 0; ++pass) {
    const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
    const int above_bits = pass == 0 ? 31 : (pass == 1 ? 21 : 10);   // of pass 0 nothing is compared
    const uint32_t same = pass == 0 ? 0 : prefix >> above_bits, mask = pass == 2 ? 1023 : 2047;
    __syncthreads();
    each([&](int, uint32_t k) {
      if (pass == 0 || (k >> above_bits) == same)
        atomicAdd(&hist[((k >> shift) & mask) * kCopies + (lane & (kCopies - 1))], 1u);
    });
    __syncthreads();
    const u32x4 x1 = mine[0], x0 = mine[1];   // x0: the larger bin
    mine[0] = mine[1] = u32x4{};
    const int c0 = (int)(x0[0] + x0[1] + x0[2] + x0[3]), c1 = (int)(x1[0] + x1[1] + x1[2] + x1[3]);
    int above = scan_sum(c0 + c1);
    if (lane == 63) sh_sum[wave] = above;
    above -= c0 + c1;
    __syncthreads();
    above += sum_before(sh_sum, wave);   // tokens of larger digits
    if (above < left && above + c0 + c1 >= left) {        // exactly one thread
      const bool first = above + c0 >= left;
      sh_digit = kBins - 1 - 2 * tid - (first ? 0 : 1);
      sh_above = above + (first ? 0 : c0);
    }
    __syncthreads();
    prefix |= sh_digit << shift;
    left -= (int)sh_above;
  }
  if (need == 0) prefix = 0xffffffffu;   // of no number: every NaN has 0
  int gt = 0, eq = 0;   // of the wave, then before it
  each([&](int, uint32_t k) {
    gt += __popcll(__ballot(k > prefix));
    eq += __popcll(__ballot(k == prefix));
  });
  if (lane == 0) {
    sh_gt[wave] = gt;
    sh_eq[wave] = eq;
  }
  __syncthreads();
  gt = sum_before(sh_gt, wave);
  eq = sum_before(sh_eq, wave);
  if constexpr (LIST) {
    const uint64_t below = ((uint64_t)1 << lane) - 1;
    each([&](int at, uint32_t k) {
      const uint64_t mg = __ballot(k > prefix), me = __ballot(k == prefix);
      const int q = eq + __popcll(me & below);
      if (k > prefix || (k == prefix && q < left)) {
        const int to = gt + __popcll(mg & below) + min(q, left), j = lo + at + lane;
        kept[bh * keep + to] = j;
        w_new[bh * new_width + to] = w[j];
      }
      gt += __popcll(mg);
      eq += __popcll(me);
    });
    return;
  }
  if (lane == 0) {
    out[bh].gt[wave] = gt;
    out[bh].eq[wave] = eq;
  }
  if (tid == 0) {
    out[bh].per = per;
    out[bh].left = left;
    out[bh].key = prefix;
  }
}

constexpr int kMoveThreads = 256;
constexpr int kListSlots = 1024;   // slots that a workgroup looks through at a time

// Old slots and weights of the stayers, in order. Workgroups x < kSelWaves have a run of
// candidates, the others kListSlots of the tokens that stay unseen (the newest, or
// all of a short cache).
__global__ void __launch_bounds__(kMoveThreads)
fa_evict_list_kernel(const float* __restrict__ weights, const Selection* __restrict__ sel,
                     int32_t* __restrict__ kept, float* __restrict__ w_new, int Hkv, int max_pages,
                     int new_max_pages, int keep, int recent) {
  constexpr int WAVES = kMoveThreads / 64;
  constexpr int ROUNDS = kListSlots / kMoveThreads;
  __shared__ int sh_gt[WAVES], sh_eq[WAVES];
  const int hk = blockIdx.y, b = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const size_t bh = (size_t)b * Hkv + hk;
  const Selection& se = sel[bh];
  const float* w = weights + bh * ((size_t)max_pages * kPageSize);
  int32_t* kp = kept + bh * keep;
  float* wn = w_new + bh * ((size_t)new_max_pages * kPageSize);
  const int cand = se.cand;
  if (blockIdx.x >= kSelWaves) {
    const int stay = cand > 0 ? recent : se.n;    // tokens cand .. + stay - 1
    const int to = cand > 0 ? keep - recent : 0;
    const int first = ((int)blockIdx.x - kSelWaves) * kListSlots;
    for (int i = first + tid; i < min(first + kListSlots, stay); i += kMoveThreads) {
      kp[to + i] = cand + i;
      wn[to + i] = w[cand + i];
    }
    return;
  }
  if (cand == 0) return;
  const int left = se.left, lo = (int)blockIdx.x * se.per, hi = min(lo + se.per, cand);
  if (lo >= hi) return;
  const uint32_t key = se.key;
  int gt = se.gt[blockIdx.x], eq = se.eq[blockIdx.x];
  for (int j0 = lo; j0 < hi; j0 += kListSlots) {
    // A wave has kListSlots / WAVES slots in a row, so that the waves' counts
    // follow one another.
    float x[ROUNDS];
    const int mine = j0 + wave * (kListSlots / WAVES) + lane;
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) x[i] = w[min(mine + 64 * i, hi - 1)];
    int g = 0, e = 0;
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
      const uint32_t k = weight_key(x[i]);
      const bool in = mine + 64 * i < hi;
      g += __popcll(__ballot(in && k > key));
      e += __popcll(__ballot(in && k == key));
    }
    if (j0 > lo) __syncthreads();
    if (lane == 0) {
      sh_gt[wave] = g;
      sh_eq[wave] = e;
    }
    __syncthreads();
    int G = gt, Q = eq;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
      if (i < wave) {
        G += sh_gt[i];
        Q += sh_eq[i];
      }
      gt += sh_gt[i];
      eq += sh_eq[i];
    }
    const uint64_t below = ((uint64_t)1 << lane) - 1;
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
      const uint32_t k = weight_key(x[i]);
      const bool in = mine + 64 * i < hi;
      const uint64_t mg = __ballot(in && k > key), me = __ballot(in && k == key);
      const int q = Q + __popcll(me & below);
      if (in && (k > key || (k == key && q < left))) {
        const int at = G + __popcll(mg & below) + min(q, left);
        kp[at] = mine + 64 * i;
        wn[at] = x[i];
      }
      G += __popcll(mg);
      Q += __popcll(me);
    }
  }
}

// The stayers' rows into the new pages, a 16-byte piece of K and of V a thread, each row
// read and written once. Bound: memory, by the gather of 2 D byte rows (8 sequences of 8
// heads, 4096 of up to 32000 tokens, D = 128: 268 MB in 57 us, 4.7 TB/s, near a plain copy
// of that size). Four rows a thread and non-temporal loads gained 2 us of it at most.
template <int D>
__global__ void __launch_bounds__(kMoveThreads)
fa_evict_move_kernel(u32x4* k_pool, u32x4* v_pool, const int32_t* __restrict__ page_table,
                     const int32_t* __restrict__ new_table, const int32_t* __restrict__ kept,
                     int32_t* __restrict__ bad, int Hkv, int max_pages, int new_max_pages,
                     int num_pages, int keep) {
  constexpr int CH = D / 8;                // pieces of a row
  constexpr int SIDE = kMoveThreads / CH;  // rows side by side
  const int hk = blockIdx.y, b = blockIdx.z;
  const int c = (int)threadIdx.x % CH, j = (int)blockIdx.x * SIDE + (int)threadIdx.x / CH;
  if (j >= keep) return;
  const int old = kept[((size_t)b * Hkv + hk) * keep + j];
  const int to = new_table[(size_t)b * new_max_pages + j / kPageSize];
  if (old < 0) return;
  const int from = page_table[(size_t)b * max_pages + old / kPageSize];
  if (from < 0 || from >= num_pages || to < 0 || to >= num_pages) {
    bad[b] = 1;   // the same value from every writer
    return;
  }
  const int64_t src = (((int64_t)from * Hkv + hk) * kPageSize + old % kPageSize) * CH + c;
  const int64_t dst = (((int64_t)to * Hkv + hk) * kPageSize + j % kPageSize) * CH + c;
  const u32x4 x = k_pool[src], y = v_pool[src];
  k_pool[dst] = x;
  v_pool[dst] = y;
}

}  // namespace cache
}  // namespace fa

extern "C" int64_t fa_decode_weights_workspace_floats(int64_t B, int64_t H, int64_t H_kv, int64_t D,
                                                      int64_t max_pages) {
  // the sizes that fa_validate_decode_weights refuses
  constexpr int64_t kIndexes = (int64_t(1) << 31) - 1;
  if (B <= 0 || B > 65535 || H <= 0 || H > 65535 || H_kv <= 0 || H % H_kv != 0 ||
      (D != 64 && D != 128) || max_pages <= 0 || max_pages > kIndexes / 16 || B > kIndexes / max_pages)
    return 0;
  if (fa::cache::in_one(B, H, H_kv, max_pages)) return 0;
  return fa::cache::workspace_of(B, H, H_kv, D, max_pages).floats;
}

extern "C" int fa_decode_paged_weights(const void* q, const void* k_pool, const void* v_pool,
                                       const int32_t* page_table, const int32_t* ctx_lens,
                                       const float* weights, int64_t B, int64_t H, int64_t H_kv,
                                       int64_t D, int64_t page_size, int64_t max_pages,
                                       int64_t num_pages, float* workspace, void* o, float* lse,
                                       float* weights_out, int bf16, void* stream) {
  const int st = fa_validate_decode_weights(q, k_pool, v_pool, page_table, ctx_lens, weights, B, H,
                                            H_kv, D, page_size, max_pages, num_pages, workspace, o, lse,
                                            weights_out);
  if (st != FA_OK) return st;
  using fa::cache::decode_weights;
  const auto fn = D == 128 ? (bf16 ? decode_weights<128, true> : decode_weights<128, false>)
                           : (bf16 ? decode_weights<64, true> : decode_weights<64, false>);
  return fn(q, k_pool, v_pool, page_table, ctx_lens, weights, B, H, H_kv, max_pages, num_pages, workspace,
            o, lse, weights_out, stream);
}

extern "C" int64_t fa_kv_evict_workspace_words(int64_t B, int64_t H_kv, int64_t max_pages) {
  using namespace fa::cache;
  if (B <= 0 || H_kv <= 0 || B > 65535 || H_kv > 65535) return 0;
  if (max_pages <= kListKeys * kSelThreads / kPageSize) return 0;
  return B * H_kv * kSelWords;
}

extern "C" int fa_kv_evict(void* k_pool, void* v_pool, const int32_t* page_table,
                           const int32_t* ctx_lens, const float* weights,
                           const int32_t* new_page_table, int32_t* kept, float* new_weights,
                           int32_t* new_lens, int32_t* bad, int32_t* workspace, int64_t B, int64_t H_kv,
                           int64_t D, int64_t keep, int64_t recent, int64_t page_size,
                           int64_t max_pages, int64_t new_max_pages, int64_t num_pages, void* stream) {
  using namespace fa::cache;
  const int st = fa_validate_kv_evict(k_pool, v_pool, page_table, ctx_lens, weights, new_page_table,
                                      kept, new_weights, new_lens, bad, workspace, B, H_kv, D, keep,
                                      recent, page_size, max_pages, new_max_pages, num_pages);
  if (st != FA_OK) return st;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  Selection* sel = reinterpret_cast<Selection*>(workspace);
  const int64_t width = max_pages * kPageSize;
  const int64_t keys = (width + kSelThreads - 1) / kSelThreads;   // of a thread
  const auto select = keys <= 1    ? fa_evict_select_kernel<1>
                      : keys <= 4  ? fa_evict_select_kernel<4>
                      : keys <= 16 ? fa_evict_select_kernel<16>
                      : keys <= kMostKeys ? fa_evict_select_kernel<kMostKeys>
                                          : fa_evict_select_kernel<0>;
  hipLaunchKernelGGL(select, dim3((unsigned)H_kv, (unsigned)B), dim3(kSelThreads), 0, s, weights, ctx_lens,
                     kept, new_weights, new_lens, bad, sel, (int)H_kv, (int)max_pages, (int)keep,
                     (int)recent, (int)(new_max_pages * kPageSize));
  if (keys > kListKeys) {
    const int64_t plain = ((keep < width ? keep : width) + kListSlots - 1) / kListSlots;
    hipLaunchKernelGGL(fa_evict_list_kernel, dim3((unsigned)(kSelWaves + plain), (unsigned)H_kv, (unsigned)B),
                       dim3(kMoveThreads), 0, s, weights, sel, kept, new_weights, (int)H_kv,
                       (int)max_pages, (int)new_max_pages, (int)keep, (int)recent);
  }
  const int64_t rows = kMoveThreads / (D / 8);
  const dim3 grid((unsigned)((keep + rows - 1) / rows), (unsigned)H_kv, (unsigned)B);
  const auto move = D == 128 ? fa_evict_move_kernel<128> : fa_evict_move_kernel<64>;
  hipLaunchKernelGGL(move, grid, dim3(kMoveThreads), 0, s, (fa::u32x4*)k_pool, (fa::u32x4*)v_pool,
                     page_table, new_page_table, kept, bad, (int)H_kv, (int)max_pages,
                     (int)new_max_pages, (int)num_pages, (int)keep);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? FA_OK : -(int)e;
}
