// fa_stream.hpp — decode attention over runs of 16-bit pages, for the kernels
// that run it: one query token per sequence, cut into chunks of pages that a
// later launch joins by their maxima and sums (see chunk_body), or, of short
// sequences, whole.
//
// Bound by memory: a page of 16 tokens of one KV head is 32 D bytes each of K and
// V, read once for up to 16 query rows. A wave loads whole pages straight into
// registers in operand layout, two at a time, and multiplies
//   S   = K Q^T     (16x16x32: 16 tokens x 16 query rows; rows past the last are zero columns)
//   O^T += V^T P^T  (16x16x32 over the two pages: rows c of block db are dims
//                    c D/16 + db, P^T straight from the S accumulators)
// K's pieces are operands as they lie; V's tokens are paired by v_perm. Nothing
// goes through LDS, so a CU has three waves a SIMD with 16 KiB each in flight (D
// = 128; held to the registers of four, 1.14 GB took 240 us against 215, with two
// 219). Lane l has query row l % 16 in both products, so a row's maximum and sum stay
// in its lane column.
//
// Maxima are kept as K Q^T gives them, in the partials and the joins too, and differences
// are scaled, so that no weight passes 1 however large the scores are: a scaled maximum
// of 2^31 is rounded by up to 2^7, a factor of 2^128. P goes into its product as two
// 16-bit terms, rounded and then what that leaves out (22 bits in fp16, 16 in
// bf16), beside a sum of P that is not rounded.
#pragma once

#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "fa_tile.hpp"

namespace fa {
namespace stream {

constexpr int kTokens = 16;    // of a page
constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kBatch = 2;      // pages a wave takes at a time
constexpr int kXcds = 8;

// Chunks. The pages of all sequences, T in all, are cut into runs of about C
// pages, a sequence into equal ones: workgroups of like size whatever the
// lengths, from lengths that only the device knows. The grid has the most
// chunks that any lengths can give, and the rest end at once. C is what makes
// kFill workgroups, between kMinChunk and kMaxChunk pages; beyond that, what
// makes kMost. Weights of 8 sequences of 200 to 4000 tokens, H32 over 8, D = 128, for kFill
// 256, 512 and 1024: 24.6, 26.1 and 26.8 us a call; 32 of 50 to 1500 under a prefix of
// 7999: 40.4, 39.0 and 38.7. kMaxChunk 128: 16 of 2000 to 32768 tokens 227 -> 232 us, the
// last chunks run alone; 16: 64 of 20 to 1000 under 32768 75 -> 80.
constexpr int kFill = 512, kMost = 4096;
constexpr int kMinChunk = kWaves * kBatch, kMaxChunk = 32;

// Pools from 64 MiB on do not stay in the caches between two steps; their pages are
// read with the non-temporal hint (the 1.14 GB of the above: 251 -> 227 us; 91 MB
// that are read again at once: 25.8 -> 26.7).
inline bool pass_through(int64_t num_pages, int64_t Hkv, int64_t D) {
  return num_pages * Hkv * kTokens * D * 4 >= (int64_t)64 << 20;
}

struct Plan {
  unsigned fill, most;   // chunks along the pages that make kFill and kMost workgroups
};
inline Plan plan_of(int64_t groups) {
  return {(unsigned)((kFill + groups - 1) / groups), (unsigned)((kMost + groups - 1) / groups)};
}

// Pages of a chunk where the batch has `total`.
__host__ __device__ inline int chunk_pages(int total, Plan plan) {
  const unsigned c = ((unsigned)total + plan.fill - 1) / plan.fill;
  if (c <= kMaxChunk) return (int)(c < kMinChunk ? kMinChunk : c);
  const unsigned d = ((unsigned)total + plan.most - 1) / plan.most;
  return d < kMaxChunk ? kMaxChunk : (int)d;
}

__host__ __device__ inline int chunks_of(int pages, int C) {
  const int n = (int)(((unsigned)pages + (unsigned)C - 1) / (unsigned)C);
  return n < 1 ? 1 : n;   // an empty sequence has one, which says so
}

// The most chunks of B sequences in a table of max_pages: sum ceil(p / C) is
// below T / C + B, and T / chunk_pages(T) is at most plan.fill, or plan.most where
// T is more than plan.fill * kMaxChunk.
inline int64_t most_chunks(int64_t B, int64_t max_pages, Plan plan) {
  const int64_t total = B * max_pages;
  const int64_t by_max = total / kMaxChunk < plan.most ? total / kMaxChunk : plan.most;
  const int64_t by_min = total / kMinChunk, n = plan.fill > by_max ? plan.fill : by_max;
  return (n < by_min ? n : by_min) + B;
}

__device__ __forceinline__ int pages_of(int ctx, int max_pages) {
  const int p = (int)(((unsigned)max(ctx, 0) + kTokens - 1) / kTokens);
  return p > max_pages ? 0 : p;   // of an invalid length: none
}

struct Chunk {
  int b, ctx;          // sequence, -1: none; its length
  int split, splits;   // number of the chunk in the sequence, and how many there are
};

// Sequences up to which every wave finds its chunk by itself, a lane for up to
// four of them; more are planned by a launch of their own.
constexpr int kWavePlan = 256;

// Chunk number x of a batch of up to kWavePlan sequences.
__device__ __forceinline__ Chunk chunk_of(const int32_t* __restrict__ ctx_lens, int B, int max_pages,
                                          Plan plan, int x) {
  constexpr int MOST = kWavePlan / 64;
  const int per = (B + 63) / 64, i0 = (int)(threadIdx.x & 63) * per;
  int ctx[MOST], n[MOST], pages = 0, ns = 0;
#pragma unroll
  for (int k = 0; k < MOST; ++k) {
    ctx[k] = k < per && i0 + k < B ? ctx_lens[i0 + k] : 0;
    pages += pages_of(ctx[k], max_pages);
  }
  const int C = chunk_pages(__builtin_amdgcn_readlane(scan_sum(pages), 63), plan);
#pragma unroll
  for (int k = 0; k < MOST; ++k) {
    n[k] = k < per && i0 + k < B ? chunks_of(pages_of(ctx[k], max_pages), C) : 0;
    ns += n[k];
  }
  int e = scan_sum(ns) - ns;   // chunks before the lane's first sequence
  int b = -1, len = 0, split = 0, splits = 0;
#pragma unroll
  for (int k = 0; k < MOST; ++k) {
    if (x >= e && x < e + n[k]) {
      b = i0 + k;
      len = ctx[k];
      split = x - e;
      splits = n[k];
    }
    e += n[k];
  }
  Chunk r{-1, 0, 0, 1};
  const uint64_t one = __ballot(b >= 0);
  if (one == 0) return r;
  const int at = __builtin_ctzll(one);
  r.b = __builtin_amdgcn_readlane(b, at);
  r.ctx = __builtin_amdgcn_readlane(len, at);
  r.split = __builtin_amdgcn_readlane(split, at);
  r.splits = __builtin_amdgcn_readlane(splits, at);
  return r;
}

// Pages of the batch, by a whole wave.
__device__ __forceinline__ int total_pages(const int32_t* __restrict__ ctx_lens, const int4* __restrict__ table,
                                           int B, int max_pages) {
  if (table != nullptr) return table[0].y;
  int pages = 0;
#pragma unroll
  for (int k = 0; k < kWavePlan / 64; ++k) {
    const int i = 64 * k + (int)(threadIdx.x & 63);
    pages += i < B ? pages_of(ctx_lens[i], max_pages) : 0;
  }
  return __builtin_amdgcn_readlane(scan_sum(pages), 63);
}

// The chunks of a batch of any size: table[0] has their number and the pages of the
// batch, table[1 + x] chunk x as (sequence, its length, split, splits). One workgroup, a run of sequences a
// thread; a sequence's entries are written by the whole wave.
constexpr int kPlanThreads = 1024;
static __global__ void __launch_bounds__(kPlanThreads)
fa_stream_plan_kernel(const int32_t* __restrict__ ctx_lens, int B, int max_pages, Plan plan,
                      int4* __restrict__ table) {
  constexpr int WAVES = kPlanThreads / 64;
  __shared__ int sh[2][WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int per = (B + kPlanThreads - 1) / kPlanThreads;
  const int i0 = min(tid * per, B), i1 = min(i0 + per, B);
  int pages = 0;
  for (int i = i0; i < i1; ++i) pages += pages_of(ctx_lens[i], max_pages);
  const int sum = scan_sum(pages);
  if (lane == 63) sh[0][wave] = sum;
  __syncthreads();
  int total = 0;
  for (int w = 0; w < WAVES; ++w) total += sh[0][w];
  const int C = chunk_pages(total, plan);
  int n = 0;
  for (int i = i0; i < i1; ++i) n += chunks_of(pages_of(ctx_lens[i], max_pages), C);
  const int before = scan_sum(n) - n;
  if (lane == 63) sh[1][wave] = before + n;
  __syncthreads();
  int e = before, chunks = 0;
  for (int w = 0; w < WAVES; ++w) {
    if (w < wave) e += sh[1][w];
    chunks += sh[1][w];
  }
  if (tid == 0) table[0] = int4{chunks, total, 0, 0};
  for (int k = 0; k < per; ++k) {
    const int i = i0 + k;
    const int ctx = i < i1 ? ctx_lens[i] : 0;
    const int s = i < i1 ? chunks_of(pages_of(ctx, max_pages), C) : 0;
    for (uint64_t rest = __ballot(s > 0); rest != 0; rest &= rest - 1) {
      const int l = __builtin_ctzll(rest);
      const int b = __builtin_amdgcn_readlane(i, l), cl = __builtin_amdgcn_readlane(ctx, l);
      const int sl = __builtin_amdgcn_readlane(s, l), el = __builtin_amdgcn_readlane(e, l);
      for (int j = lane; j < sl; j += 64) table[1 + el + j] = int4{b, cl, j, sl};
    }
    e += s;
  }
}

// One for every KV head and 16 of its query heads.
inline int64_t head_groups(int64_t H, int64_t Hkv) { return Hkv * ((H / Hkv + 15) / 16); }

// Workgroups of a launch over chunks: they go to the XCDs in turn, an XCD has every
// eighth chunk and the head groups of a chunk one after the other, so that what is
// read of a page at about the same time goes through one L2 and is contiguous.
__host__ __device__ inline int64_t chunk_blocks(int64_t chunks, int64_t groups) {
  return (chunks + kXcds - 1) / kXcds * kXcds * groups;
}
struct Place {
  int number, hg;   // chunk and head group of a workgroup
};
__device__ __forceinline__ Place place_of(int g, int groups) {
  const int y = g / (kXcds * groups), x = g - y * (kXcds * groups);
  return Place{y * kXcds + x % kXcds, x / kXcds};
}

// The workgroup's chunk and its pages p0 .. p1 - 1; b < 0: there is none.
struct Run {
  int b, ctx, splits, split, p0, p1;
  bool bad;   // the length is invalid
};
__device__ __forceinline__ Run run_of(const int32_t* __restrict__ ctx_lens, const int4* __restrict__ table,
                                      int B, int max_pages, Plan plan, int number) {
  Chunk ch;
  if (table != nullptr) {
    const int4 e = number < table[0].x ? table[1 + number] : int4{-1, 0, 0, 1};
    ch = Chunk{e.x, e.y, e.z, e.w};
  } else {
    ch = chunk_of(ctx_lens, B, max_pages, plan, number);
  }
  Run r;
  r.b = __builtin_amdgcn_readfirstlane(ch.b);
  r.ctx = __builtin_amdgcn_readfirstlane(ch.ctx);
  r.split = __builtin_amdgcn_readfirstlane(ch.split);
  r.splits = __builtin_amdgcn_readfirstlane(ch.splits);
  const int pages = pages_of(r.ctx, max_pages);
  r.bad = r.ctx < 0 || (r.ctx > 0 && pages == 0);
  // The first pages % splits chunks have a page more.
  const int each = (int)((unsigned)pages / (unsigned)r.splits), more = pages - each * r.splits;
  r.p0 = r.split * each + min(r.split, more);
  r.p1 = r.p0 + each + (r.split < more);
  return r;
}

// Max and sum over the four lane groups of a column.
__device__ __forceinline__ float col_max(float x) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  return max_xor32(x);
}
__device__ __forceinline__ float col_sum(float x) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  return sum_xor32(x);
}

// f over the 16 lanes of a row (quad_perm twice, row_half_mirror, row_mirror); max and
// sum over the wave.
template <typename F>
__device__ __forceinline__ float over_row(float x, F f) {
  const auto at = [&](auto ctrl) {
    return __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  x = f(x, at(std::integral_constant<int, 0xb1>{}));
  x = f(x, at(std::integral_constant<int, 0x4e>{}));
  x = f(x, at(std::integral_constant<int, 0x141>{}));
  return f(x, at(std::integral_constant<int, 0x140>{}));
}
__device__ __forceinline__ float wave_max(float x) {
  return col_max(over_row(x, [](float a, float b) { return fmaxf(a, b); }));
}
__device__ __forceinline__ float wave_sum(float x) {
  return col_sum(over_row(x, [](float a, float b) { return a + b; }));
}

template <bool BF16>
__device__ __forceinline__ f32x4 mma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  return __builtin_bit_cast(uint32_t, cvt2x<BF16>(a, b));
}

// What pack2(a, b) = ab leaves out, rounded alike. fp16: words that the compiler
// does not see through, or it rounds a and b a second time.
template <bool BF16>
__device__ __forceinline__ uint32_t rest2(float a, float b, uint32_t ab) {
  if constexpr (BF16) {
    return pack2<true>(a - __uint_as_float(ab << 16), b - __uint_as_float(ab & 0xffff0000u));
  } else {
    asm("" : "+v"(ab));
    const f16x2 h = __builtin_bit_cast(f16x2, ab);
    return pack2<false>(a - (float)h[0], b - (float)h[1]);
  }
}

// K is loaded in whole 128-byte lines of eight tokens, and an operand has 64 bytes of
// sixteen. a has tokens 0 .. 7 and b tokens 8 .. 15, lanes 0 .. 7 of a row of 16 the
// first half of a line and lanes 8 .. 15 the second; after, a has the first half and b
// the second, of token lane % 16.
__device__ __forceinline__ void turn_k(u32x4& a, u32x4& b, bool upper) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t x = a[j], y = b[j];
    // row_ror:8: of lane ^ 8 within the row
    const uint32_t xo = __builtin_amdgcn_update_dpp(0, x, 0x128, 0xf, 0xf, false);
    const uint32_t yo = __builtin_amdgcn_update_dpp(0, y, 0x128, 0xf, 0xf, false);
    a[j] = upper ? yo : x;
    b[j] = upper ? y : xo;
  }
}

// LDS of a workgroup: its waves' parts, heads in different banks.
template <int D, int WAVES = kWaves>
struct Shared {
  __attribute__((aligned(16))) float o[WAVES][16][D + 4];
  float m[WAVES][16], l[WAVES][16];
  int bad[WAVES];
};

// Where the tokens are: the page id of place p in a list, and the tokens from its
// first on (of the last place, fewer than 16).
struct Pages {
  const int32_t* pt;
  int ctx;
  __device__ int id(int p) const { return pt[p]; }
  __device__ int tokens(int p) const { return ctx - p * kTokens; }
};
// The pages of a prefix, np of them, and then a sequence's own.
struct JoinedPages {
  const int32_t *prefix, *own;
  int np, P, ctx;
  __device__ int id(int p) const { return p < np ? prefix[p] : own[p - np]; }
  __device__ int tokens(int p) const { return p < np ? P - p * kTokens : ctx - (p - np) * kTokens; }
};

// Scores of a chunk that go to memory, K Q^T unscaled, a float a slot of the
// sequence: column 0's, and `stride` on those of the next of `heads` columns.
struct NoScores {
  static constexpr bool kThere = false;
};
struct ScoresOut {
  static constexpr bool kThere = true, kKept = false;
  float* to;
  int64_t stride;
  int heads;
};
// Scores that stay in LDS: rows of `stride` floats for the columns, places from 0 on.
struct ScoresKept {
  static constexpr bool kThere = true, kKept = true;
  float* rows;
  int stride;
};

// One chunk by WAVES waves, `wave` their number: places p0 .. p1 - 1 of the pages, for
// up to 16 query rows. Column col of the products is the query row at element qoff of
// q (live: there is one). At the end row(d, v) is called for its dims d .. d + 3,
// normalised, by some lane of the column, and stat(maximum, sum of the weights) by one:
// (-inf, 0) of no tokens, a NaN sum where a page or the length (bad) is invalid. NT:
// pages are read with the non-temporal hint. Has one barrier of the workgroup, so waves
// without a chunk call it too, with no pages and no live row.
template <int D, bool BF16, bool NT, int WAVES, typename Where, typename Scores, typename Row, typename Stat>
__device__ __forceinline__ void
chunk_body(Shared<D, WAVES>& sh, const int wave, const uint16_t* __restrict__ q,
           const char* __restrict__ k_pool, const char* __restrict__ v_pool, const Where& pages, int p0,
           int p1, bool bad, bool live, int64_t qoff, int hk, int Hkv, int num_pages, float c,
           const Scores& scores, Row&& row, Stat&& stat) {
  constexpr int BYTES = kTokens * D * 2;   // a page of one head
  constexpr int KS = D / 32;               // steps of S = K Q^T, K pieces of a lane
  constexpr int DB = D / 16;               // blocks of O^T
  constexpr int VW = D / 32;               // words of a lane's V piece of a token
  constexpr int kAux = NT ? 2 : 0;
  const int lane = threadIdx.x & 63;
  const int col = lane & 15, grp = lane >> 4;
  // This wave's pages, in whole batches but for the last wave's.
  const int per = ((p1 - p0 + kBatch - 1) / kBatch + WAVES - 1) / WAVES * kBatch;
  const int w0 = min(p0 + per * wave, p1), w1 = min(w0 + per, p1);

  // Ids of 64 pages a load, lane i that of page 64 j + i; first of all, as the
  // pages wait for them.
  int ids = 0;
  const auto load_ids = [&](int w) { ids = pages.id(min(w + lane, w1 - 1)); };
  if (w0 < w1) load_ids(w0);
  u32x4 qf[KS];   // column col, dims 32 kb + 8 grp .. + 7
#pragma unroll
  for (int kb = 0; kb < KS; ++kb) {
    qf[kb] = u32x4{};
    if (live) qf[kb] = *reinterpret_cast<const u32x4*>(q + qoff + 32 * kb + 8 * grp);
  }
  float m = -INFINITY, l = 0.f;
  f32x4 acc[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) acc[db] = f32x4{};

  // K: token col % 8 (+ 8), dims 32 (col / 8) + 8 grp of a 128-byte line; see turn_k.
  const uint32_t koff = (col & 7) * (2 * D) + 64 * (col >> 3) + 16 * grp;
  const bool upper = col >= 8;
  const uint32_t voff = 4 * grp * (2 * D) + col * (4 * VW);   // tokens 4 grp + r, dims D/16 col ..
  u32x4 xk[kBatch][KS];
  uint32_t xv[kBatch][4][VW];
  for (int w = w0; w < w1; w += kBatch) {
    if (((w - w0) & 63) == 0) {
      if (w != w0) load_ids(w);
      const bool no = ids < 0 || ids >= num_pages;
      bad |= no;
      ids = no ? 0 : ids;   // read in place of a page that is not there; the result is NaN
      // Used up here: after the branch the compiler would wait for the load on either
      // path, and with it, every batch, for the scores' stores.
      asm volatile("" : "+v"(ids));
    }
    // Past the wave's last page the last one again, masked below.
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const size_t rec = (size_t)__builtin_amdgcn_readlane(ids, (w - w0 + i) & 63) * Hkv + hk;
      const auto rk = make_rsrc(k_pool + rec * BYTES, BYTES);
      const auto rv = make_rsrc(v_pool + rec * BYTES, BYTES);
#pragma unroll
      for (int kb = 0; kb < KS; ++kb)   // line kb / 2 of tokens 8 (kb % 2) ..
        xk[i][kb] = __builtin_amdgcn_raw_buffer_load_b128(rk, koff, 128 * (kb / 2) + 16 * D * (kb % 2), kAux);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if constexpr (VW == 4) {
          const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(rv, voff, 2 * D * r, kAux);
#pragma unroll
          for (int j = 0; j < 4; ++j) xv[i][r][j] = x[j];
        } else {
          const u32x2 x = __builtin_amdgcn_raw_buffer_load_b64(rv, voff, 2 * D * r, kAux);
          xv[i][r][0] = x[0];
          xv[i][r][1] = x[1];
        }
      }
    }
    int n[kBatch];   // tokens of the pages
    bool tail = false;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      n[i] = w + i < w1 ? min(pages.tokens(w + i), kTokens) : 0;
      tail |= n[i] < kTokens;
    }
    f32x4 s[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      s[i] = f32x4{};
#pragma unroll
      for (int kb = 0; kb < KS; kb += 2) turn_k(xk[i][kb], xk[i][kb + 1], upper);
#pragma unroll
      for (int kb = 0; kb < KS; ++kb) s[i] = mma16<BF16>(xk[i][kb], qf[kb], s[i]);
    }
    if (tail) {           // wave-uniform
      asm volatile("");   // a branch: not selects in every batch
      // Rows past the context may hold NaN, and 0 NaN is NaN: V's become zeros.
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool in = 4 * grp + r < n[i];
          s[i][r] = in ? s[i][r] : -INFINITY;
#pragma unroll
          for (int j = 0; j < VW; ++j) xv[i][r][j] = in ? xv[i][r][j] : 0u;
        }
    }
    if constexpr (Scores::kThere) {
      if constexpr (Scores::kKept) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
          if (w + i < w1)
            *reinterpret_cast<f32x4*>(scores.rows + col * scores.stride + (w + i) * kTokens + 4 * grp) = s[i];
      } else {
        // They wait in the wave's part of sh.o, D/16 pages of them, and go out in long
        // rows, a head's 64 D/16 bytes at a time.
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
          *reinterpret_cast<f32x4*>(&sh.o[wave][col][((w - w0 + i) % DB) * kTokens + 4 * grp]) = s[i];
        if ((w - w0) % DB == DB - kBatch || w + kBatch >= w1) {
          const int from = w0 + (w - w0) / DB * DB, slots = (min(w + kBatch, w1) - from) * kTokens;
          constexpr int LANES = 4 * DB;   // of a row, 4 slots each
#pragma unroll
          for (int h = 0; h < 16; h += 64 / LANES) {
            const int g = h + lane / LANES, j = 4 * (lane % LANES);
            if (g < scores.heads && j < slots)
              *reinterpret_cast<f32x4*>(scores.to + g * scores.stride + (int64_t)from * kTokens + j) =
                  *reinterpret_cast<const f32x4*>(&sh.o[wave][g][j]);
          }
        }
      }
    }
    float top = s[0][0];
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) top = fmaxf(top, s[i][r]);
    const float m_new = fmaxf(m, col_max(top));
    if (__any(m_new != m)) {
      const float alpha = m_new == m ? 1.f : exp2_hw((m - m_new) * c);
      l *= alpha;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[db][r] *= alpha;
      m = m_new;
    }
    const float mu = m == -INFINITY ? 0.f : m;   // no score above -inf so far: weights of 0
    u32x2 ph[kBatch], pl[kBatch];                // P's two terms
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      float p[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        p[r] = exp2_hw((s[i][r] - mu) * c);
        l += p[r];
      }
      ph[i] = u32x2{pack2<BF16>(p[0], p[1]), pack2<BF16>(p[2], p[3])};
      pl[i] = u32x2{rest2<BF16>(p[0], p[1], ph[i][0]), rest2<BF16>(p[2], p[3], ph[i][1])};
    }
    // Slots 0 .. 3 of the lane's reduction are tokens 4 grp .. + 3 of the first
    // page, slots 4 .. 7 those of the second.
    const u32x4 bh = u32x4{ph[0][0], ph[0][1], ph[1][0], ph[1][1]};
    const u32x4 bl = u32x4{pl[0][0], pl[0][1], pl[1][0], pl[1][1]};
#pragma unroll
    for (int j = 0; j < VW; ++j) {
      u32x4 even, odd;   // dims 2 j and 2 j + 1 of the lane's sixteenth
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        even[2 * i] = __builtin_amdgcn_perm(xv[i][1][j], xv[i][0][j], 0x05040100u);
        even[2 * i + 1] = __builtin_amdgcn_perm(xv[i][3][j], xv[i][2][j], 0x05040100u);
        odd[2 * i] = __builtin_amdgcn_perm(xv[i][1][j], xv[i][0][j], 0x07060302u);
        odd[2 * i + 1] = __builtin_amdgcn_perm(xv[i][3][j], xv[i][2][j], 0x07060302u);
      }
      acc[2 * j] = mma16<BF16>(even, bh, acc[2 * j]);
      acc[2 * j + 1] = mma16<BF16>(odd, bh, acc[2 * j + 1]);
      acc[2 * j] = mma16<BF16>(even, bl, acc[2 * j]);
      acc[2 * j + 1] = mma16<BF16>(odd, bl, acc[2 * j + 1]);
    }
  }
  l = col_sum(l);

  // The waves' parts join in LDS. acc[db][r] is dim (4 grp + r) D/16 + db.
  const bool wave_bad = __any(bad);
  if (lane == 0) sh.bad[wave] = wave_bad;
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int db = 0; db < DB; ++db) sh.o[wave][col][(4 * grp + r) * DB + db] = acc[db][r];
  if (grp == 0) {
    sh.m[wave][col] = m;
    sh.l[wave][col] = l;
  }
  __syncthreads();
  bool any_bad = false;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) any_bad |= sh.bad[w] != 0;
  // A row's columns are written by its lane column: lanes (col, grp) of all waves.
  if (!live) return;
  float M = sh.m[0][col];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) M = fmaxf(M, sh.m[w][col]);
  float e[WAVES], z = 0.f;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    const float wl = sh.l[w][col];
    e[w] = wl == 0.f ? 0.f : exp2_hw((sh.m[w][col] - M) * c);   // without pages: m = -inf, sums 0
    z = fmaf(e[w], wl, z);
  }
  if (any_bad) z = NAN;
  const float inv = z == 0.f ? 0.f : 1.f / z;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) e[w] *= inv;   // before the sums: bf16's V reaches 2^127
  for (int d = 4 * (4 * wave + grp); d < D; d += 16 * WAVES) {
    f32x4 a = f32x4{};
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(&sh.o[w][col][d]);
#pragma unroll
      for (int j = 0; j < 4; ++j) a[j] = fmaf(e[w], v[j], a[j]);
    }
    row(d, a);
  }
  if (wave == 0 && grp == 0) stat(M, z);
}

// row and stat of chunk_body: partial number `part`, part_o[part * D ..] and
// part_ml[part]; or the result itself.
template <int D>
struct PartOut {
  float* o;
  float2* ml;
  int64_t part;
  __device__ void operator()(int d, f32x4 a) const { *reinterpret_cast<f32x4*>(o + part * D + d) = a; }
  __device__ void operator()(float m, float z) const { ml[part] = make_float2(m, z); }
};
// L from the maximum of the products K Q^T and the sum of the weights.
__device__ __forceinline__ float lse_of(float m, float z, float c) {
  return z == 0.f ? -INFINITY : fmaf(m, c, log2_hw(z)) * kLn2;
}
template <int D, bool BF16>
struct RowOut {
  uint16_t* o;
  float* lse;
  int64_t row;
  float c;
  __device__ void operator()(int d, f32x4 a) const {
    *reinterpret_cast<u32x2*>(o + row * D + d) = u32x2{pack2<BF16>(a[0], a[1]), pack2<BF16>(a[2], a[3])};
  }
  __device__ void operator()(float m, float z) const { lse[row] = lse_of(m, z, c); }
};

// Partials of one row: number at + i * stride, i < n.
struct Parts {
  const float* o;
  const float2* ml;
  int64_t at, stride;
  int n;
};

constexpr int kJoinThreads = 256;
constexpr int kJoinWeights = 512;   // parts whose weights are kept at a time

template <int D>
struct JoinShared {
  float w[kJoinWeights];
  float red[2 * kJoinThreads / 64];
  float acc[4 * kJoinThreads / D][D];
};

// Maximum and sum over a row's parts, for the whole wave: (-inf, 0) of empty
// ones, a NaN sum where one is.
__device__ __forceinline__ float2 join_wave(const Parts& p, float c) {
  const int lane = threadIdx.x & 63;
  float M = -INFINITY, z = 0.f;
  for (int i = lane; i < p.n; i += 64) {
    const float2 x = p.ml[p.at + i * p.stride];
    if (x.x > M) {
      z *= exp2_hw((M - x.x) * c);   // M = -inf: z is 0 or NaN
      M = x.x;
    }
    z += x.x == -INFINITY ? x.y : x.y * exp2_hw((x.x - M) * c);
  }
  const float top = wave_max(M);
  return make_float2(top, wave_sum(M == -INFINITY ? z : z * exp2_hw((M - top) * c)));
}

// Parts are joined by 2^-kJoinShift of their sums, which add up to as many as there are tokens (2^8
// times that of tiles): V near bf16's end that a part's own sums hold, of a 2^14th of the tokens at
// least, stay in range. At the lower end a V of 2^-118 is 2^-16 off. Weights that add up to 1
// would wait for their sum: 2048 rows 5.0 -> 5.9 us.
template <bool BF16>
constexpr float kJoinShift = BF16 ? 16.f : 0.f;

// O and L of one row out of two lists of parts, by one workgroup; sums in a fixed
// order. Bound by the chain of a launch, the parts' weights and the parts: 2048 rows of 10
// to 16 parts 5.2 us (5.7 with shuffles over LDS for the wave's maxima and sums). Parts
// asked for before their weights, one, two or four a thread: 5.5, 6.1, 6.6.
template <int D, bool BF16>
__device__ __forceinline__ void join_row(JoinShared<D>& sh, const Parts& a, const Parts& b, float c,
                                         uint16_t* __restrict__ o, float* __restrict__ lse) {
  constexpr int PER = D / 4, SIDE = kJoinThreads / PER, WAVES = kJoinThreads / 64;
  const int tid = threadIdx.x, wave = tid >> 6;
  const int n = a.n + b.n;
  const auto ml = [&](int i) { return i < a.n ? a.ml[a.at + i * a.stride] : b.ml[b.at + (i - a.n) * b.stride]; };
  const int d = 4 * (tid % PER), side = tid / PER;
  const auto part = [&](int k) {
    const float* p = k < a.n ? a.o + (a.at + k * a.stride) * D : b.o + (b.at + (k - a.n) * b.stride) * D;
    return *reinterpret_cast<const f32x4*>(p + d);
  };
  const float2 mine = tid < n ? ml(tid) : make_float2(-INFINITY, 0.f);
  float M = mine.x;
  for (int i = tid + kJoinThreads; i < n; i += kJoinThreads) M = fmaxf(M, ml(i).x);
  M = wave_max(M);
  if ((tid & 63) == 0) sh.red[wave] = M;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < WAVES; ++i) M = fmaxf(M, sh.red[i]);
  float z = 0.f;
  f32x4 v = f32x4{};
  for (int i0 = 0; i0 < n; i0 += kJoinWeights) {
    const int m = min(kJoinWeights, n - i0);
    if (i0 > 0) __syncthreads();
    for (int i = tid; i < m; i += kJoinThreads) {
      const float2 x = i0 + i < kJoinThreads ? mine : ml(i0 + i);   // an empty part: (-inf, 0), or NaN
      const float e = x.x == -INFINITY ? x.y : x.y * exp2_hw(fmaf(x.x - M, c, -kJoinShift<BF16>));
      sh.w[i] = e;
      z += e;
    }
    __syncthreads();
    int i = side;
#pragma unroll 4
    for (; i < m; i += SIDE) {
      const f32x4 x = part(i0 + i);
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = fmaf(sh.w[i], x[r], v[r]);
    }
  }
  z = wave_sum(z);
  if ((tid & 63) == 0) sh.red[WAVES + wave] = z;
#pragma unroll
  for (int r = 0; r < 4; ++r) sh.acc[side][d + r] = v[r];
  __syncthreads();
  if (side > 0) return;
  z = 0.f;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) z += sh.red[WAVES + i];
#pragma unroll
  for (int i = 1; i < SIDE; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] += sh.acc[i][d + r];
  const float inv = z == 0.f ? 0.f : 1.f / z;   // a NaN sum: NaN
  *reinterpret_cast<u32x2*>(o + d) = u32x2{pack2<BF16>(v[0] * inv, v[1] * inv), pack2<BF16>(v[2] * inv, v[3] * inv)};
  if (tid == 0) *lse = lse_of(M, z * exp2_hw(kJoinShift<BF16>), c);
}

}  // namespace stream
}  // namespace fa
