// fa_mx_decode.hip — paged decode over a KV cache in MX pages (fa_mx.hpp).
//
// No reference counterpart (the reference has no decode path). One query token
// per sequence; of the ctx tokens in the sequence's pages
//   s_t = q . k_t / sqrt(D),  L = log sum_t exp(s_t),  O = sum_t exp(s_t - L) v_t,
// one pass with a running maximum and sum, cut into chunks of pages that are
// joined by their maxima and sums.
//
// Bound by memory: a page of 16 tokens of one KV head is 16 D (bits / 8 + 1 / 32)
// bytes each of K and V, read once for up to 16 query heads. A wave loads whole
// pages straight into registers in operand layout (see fa_mx.hpp), converts
// them to 16 bits there (one instruction for two values, exact) and multiplies
//   S   = K Q^T     (16x16x32: 16 tokens x 16 heads; heads past the group are zero columns)
//   O^T += V^T P^T  (16x16x32 over two pages: rows c of block db are values
//                    c D/16 + db, P^T straight from the S accumulators)
// P^T goes in as two terms, so V's product is made twice.
// Lane l has head l % 16 in both products, so a head's maximum and sum stay in
// its lane column.
//
// Maxima are kept as K Q^T gives them, and differences are scaled: s - m is 0 for
// the largest score, so no weight passes 2^kShift however large the scores are.
// (Of scaled scores s c and a rounded maximum m c the fma s c - m c is not 0 but
// up to half a place of m c off: from 2^24 on, weights of 2 and more.) Chunks
// are joined by (maximum, sum) for the same reason, not by their logsumexp.
#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include "fa_mi355x.h"
#include "fa_mx.hpp"
#include "fa_probe.h"

namespace fa {
namespace mx {

constexpr int kXcds = 8;

// Pages that a wave takes at a time: their loads are in flight together. Four
// of up to 32 code bytes a lane (K and V), two of larger ones, whose registers
// would leave three waves a SIMD and not four (K8V4 at D = 128 bf16, 24
// sequences: 57.4 us with two, 58.2 with four; 4 bits, one sequence of 131072
// tokens over one KV head: 15.1 and 14.5). Times here are of the launches of one
// call in a captured graph; a call from the outside adds the host's.
template <int D, int KB, int VB>
constexpr int kBatchOf = Page<D, KB>::PIECE + Page<D, VB>::PIECE <= 32 ? 4 : 2;

// Chunks. The pages of all sequences, T in all, are cut into runs of about C
// pages, a sequence into equal ones: workgroups of like size whatever the
// lengths, from lengths that only the device knows. The grid has the most
// chunks that any lengths can give, and the rest end at once.
//
// C, for the batch's T pages (chunks are counted along the pages; a chunk is a
// workgroup for every head group):
//   kMinChunk pages while they make fewer than kFill workgroups (kMinFull where
//   the sequences alone give every CU one),
//   then what makes kFill of them, up to kMaxChunk pages,
//   then kMaxChunk pages, until they make kMost workgroups.
// kFill is the four workgroups that a CU holds; chunks past kMaxChunk pages are
// cut for balance, at little cost. Besides, at most kRowFill chunks a sequence
// (one of 131072 tokens over one KV head, in 512, 256 and 128 chunks: 12.9, 11.8
// and 12.9 us for 8 query heads, 17.6, 14.4 and 13.8 for 32).
//
// kMinChunk is a batch of four pages for each wave. Joining chunks costs a second
// launch, 4 us: it is not made, and nothing is cut, for tables of up to
// kOnePages pages (one sequence of 512 tokens 7.0 -> 5.0 us, 8 of them 7.9 ->
// 5.2; at 768 tokens one sequence is faster cut, 6.9 and 7.3, 8 are not, 8.0 and
// 7.9) or where no table entry could make a second chunk (kMinFull: 32 sequences
// of 768 tokens over 8 KV heads 12.8 -> 9.6 us, of 2048 20.8 -> 16.3; with fewer
// than 256 workgroups 8 sequences of 1024 would gain, 8.7 -> 8.0, 8 of 2048 lose,
// 10.9 -> 12.3). Both go by the table, which alone the host knows: a short context
// in a wide table pays the second launch (one of 130 tokens 3.4 us in a table of 9
// pages, 5.2 in one of 2048).
constexpr int kFill = 1024, kMost = 4096;
constexpr int kMinChunk = 16, kMaxChunk = 128, kMinFull = 96;
constexpr int kOnePages = 32;
constexpr int kRowFill = 256;

// Sequences up to which every wave finds its chunk by itself, a lane for up to
// four of them; more are planned by a launch of their own. In a table of 512
// pages, sequences of 50 to 300 tokens: over 8 KV heads (D = 128) 257 take 24.5
// us so and 34.8 planned by the waves with 16 a lane, 1024 take 69 and 137; over
// one (D = 64) 257 take 9.5 and 9.2 (256 with four a lane 7.6), 1024 16 and 46.
constexpr int kWavePlan = 256;

// Chunks a sequence from which the join gives a row a workgroup for each 32
// columns (one sequence over one KV head, 256 chunks: 17.9 -> 14.5 us; two
// sequences of 63 chunks 14.1 -> 13.7; four of 32 13.6 and 13.9, eight of 8 10.85
// and 11.2).
constexpr int kWideJoin = 48;

// Pools from this size on do not stay in the caches between two steps; their
// codes are read with the non-temporal hint. Of four batches in turn, each the
// whole of its pools: 2.5 GB 452 -> 404 us, 299 MB 64.7 -> 57.4, 165 MB 39.8 ->
// 36.2, 131 MB 33.5 -> 31.6, 65 MB 18.4 -> 19.8, 35 MB 13.3 -> 14.0. The rule goes
// by the pools, as a step reads other layers' between two of this one; a small
// batch in large pools that is read again at once loses by it (35 MB in 4 GB 12.0
// -> 12.3 us, 165 MB 33.3 -> 36.4). Scales are read without the hint: their lines
// are shared with the codes' ends and with the next page's.
constexpr int64_t kPassThrough = 64 << 20;

static int64_t head_groups(int64_t H, int64_t Hkv) { return Hkv * ((H / Hkv + 15) / 16); }

// Chunks along the pages that make kFill and kMost workgroups; least pages of one.
struct Plan {
  unsigned fill, most, least;
};
static Plan plan_of(int64_t B, int64_t H, int64_t Hkv) {
  const int64_t g = head_groups(H, Hkv);
  int64_t fill = (kFill + g - 1) / g;
  if (fill > kRowFill * B) fill = kRowFill * B;
  const unsigned least = B * g >= kFill / 4 ? kMinFull : kMinChunk;
  return {(unsigned)fill, (unsigned)((kMost + g - 1) / g), least};
}

// Whether every sequence is one chunk, whatever the lengths: none (kMinFull) has
// 3/2 chunks of the least length.
static bool never_cut(int64_t B, int64_t H, int64_t Hkv, int64_t max_pages) {
  return max_pages <= kOnePages || 2 * max_pages < 3 * (int64_t)plan_of(B, H, Hkv).least;
}

// Pages of a chunk where the batch has `total`.
__host__ __device__ inline int chunk_pages(int total, Plan plan) {
  const unsigned c = ((unsigned)total + plan.fill - 1) / plan.fill;
  if (c <= kMaxChunk) return (int)(c < plan.least ? plan.least : c);
  const unsigned d = ((unsigned)total + plan.most - 1) / plan.most;
  return d < kMaxChunk ? kMaxChunk : (int)d;
}

// total / chunk_pages(total) for any total up to B * max_pages, at most: all
// that the host knows. sum ceil(p / C) <= total / C + B, so the chunks are at
// most this many and one a sequence.
static int64_t most_chunks(int64_t B, int64_t H, int64_t Hkv, int64_t max_pages) {
  const int64_t total = B * max_pages;
  const int64_t fill = plan_of(B, H, Hkv).fill, most = plan_of(B, H, Hkv).most;
  const int64_t by_max = total / kMaxChunk < most ? total / kMaxChunk : most;
  const int64_t by_min = total / kMinChunk, n = fill > by_max ? fill : by_max;
  return (n < by_min ? n : by_min) + 1;
}
// Rows of the grid: most chunks and one a sequence, a chunk to each XCD.
static int64_t chunk_rows(int64_t B, int64_t most) { return (most + B + kXcds - 1) / kXcds; }

// Chunks of the sequences that are cut at all, more than one a sequence: such a
// sequence has more than C pages and less than 2 pages / C chunks.
static int64_t partial_chunks(int64_t B, int64_t most) { return most + (B < most ? B : most); }

// The workspace, in words of 4 bytes: the table of chunks where one is planned,
// partial O, their maxima and sums, and the cut sequences for the join.
struct Workspace {
  int64_t slots, part_o, part_ml, plan, words;
};
static Workspace workspace_of(int64_t B, int64_t H, int64_t D, int64_t most) {
  Workspace w;
  w.slots = partial_chunks(B, most);
  w.part_o = B > kWavePlan ? 4 * (1 + chunk_rows(B, most) * kXcds) : 0;
  w.part_ml = w.part_o + w.slots * H * D;
  w.plan = w.part_ml + 2 * w.slots * H;
  w.words = w.plan + 1 + 2 * (B < most ? B : most);
  return w;
}

// P goes into its product as two 16-bit terms, itself rounded and then what that
// leaves out: 22 bits in fp16, 16 in bf16, beside a sum of P that is not rounded
// at all. (One fp16 term leaves half a place of 11 bits in each weight: O off by
// up to six times the rest of its error. The second costs, in us, 1 % of large
// batches (32 sequences of up to 32768 tokens 398 -> 402, one of 32000 13.0 ->
// 13.15), 5 % where 16 heads have few pages a wave (one of 131072 over one KV
// head 13.75 -> 14.45) and 8 % of many short uncut ones (256 of 100 to 900,
// 16 heads over 4, 13.0 -> 14.0).) In fp16 P reaches 2^15 rather than 1, so that
// what lies 2^-29 below a row's largest weight still has 11 bits and its rest
// ends at 2^-39; bf16 has fp32's range.
template <bool BF16>
constexpr float kShift = BF16 ? 0.f : 15.f;

// A chunk's sum as the join takes it for its weight: of n tokens the weights add
// up to n 2^-12, less than a chunk's tokens in any context, so no value whose
// chunk's own sums are in range leaves it there, and none near the range's lower
// end either. Exact: powers of two, and a sum is 2^kShift at least.
template <bool BF16>
constexpr float kPartScale = BF16 ? 0x1p-12f : 0x1p-27f;
constexpr float kJoinScale = 0x1p12f;   // of the joined weights: back to sums of exponentials

// What a workgroup's chunk is.
struct Chunk {
  int b, ctx;           // sequence, -1: none; its length
  int split, splits;    // number of the chunk in the sequence, and how many there are
  int partial;          // of the chunk, among those of cut sequences
  int index, cuts;      // the sequence's number among those, and how many there are
};

__device__ __forceinline__ int pages_of(int ctx, int max_pages) {
  const int p = (int)(((unsigned)max(ctx, 0) + kTokens - 1) / kTokens);
  return p > max_pages ? 0 : p;   // of an invalid length: none
}

// Of a sequence of p pages: its chunks, and what it adds to the count of cut
// sequences (<< 16) and of their chunks, which are fewer than 2 kMost. p / C to
// the nearest, so that none is longer or shorter than C by half; of kMinChunk
// pages not to the nearest but up, as a longer one takes its waves a second
// batch (8 sequences of 200 to 4000 tokens 13.1 -> 12.2 us).
__device__ __forceinline__ int chunks_of(int p, int C, int* cut) {
  const unsigned c = (unsigned)C, up = C == kMinChunk ? 2 * c - 1 : c;
  const int s = max(1, (int)((2u * (unsigned)p + up) / (2u * c)));
  *cut = s > 1 ? (s | 1 << 16) : 0;
  return s;
}

// Chunk number x of a batch of up to kWavePlan sequences.
__device__ __forceinline__ Chunk chunk_of(const int32_t* __restrict__ ctx_lens, int B,
                                          int max_pages, Plan plan, int x) {
  Chunk r;
  if (B == 1) {
    r.ctx = ctx_lens[0];
    const int p = pages_of(r.ctx, max_pages);
    r.splits = chunks_of(p, chunk_pages(p, plan), &r.cuts);
    r.b = x < r.splits ? 0 : -1;
    r.split = r.partial = x;
    r.index = 0;
    r.cuts >>= 16;
    return r;
  }
  constexpr int MOST = kWavePlan / 64;
  const int per = (B + 63) / 64, i0 = (int)(threadIdx.x & 63) * per;
  int ctx[MOST], n[MOST], m[MOST], pages = 0, ns = 0, ms = 0;
#pragma unroll
  for (int k = 0; k < MOST; ++k) {
    ctx[k] = k < per && i0 + k < B ? ctx_lens[i0 + k] : 0;
    pages += pages_of(ctx[k], max_pages);
  }
  const int C = chunk_pages(__builtin_amdgcn_readlane(scan_sum(pages), 63), plan);
#pragma unroll
  for (int k = 0; k < MOST; ++k) {
    n[k] = m[k] = 0;
    if (k < per && i0 + k < B) n[k] = chunks_of(pages_of(ctx[k], max_pages), C, &m[k]);
    ns += n[k];
    ms += m[k];
  }
  const int im = scan_sum(ms);
  int e = scan_sum(ns) - ns, f = im - ms;   // of the lane's first sequence
  int b = -1, len = 0, split = 0, splits = 0, before = 0;
#pragma unroll
  for (int k = 0; k < MOST; ++k) {
    if (x >= e && x < e + n[k]) {
      b = i0 + k;
      len = ctx[k];
      split = x - e;
      splits = n[k];
      before = f;
    }
    e += n[k];
    f += m[k];
  }
  const uint64_t one = __ballot(b >= 0);
  if (one == 0) {
    r.b = -1;
    return r;
  }
  const int at = __builtin_ctzll(one);
  r.b = __builtin_amdgcn_readlane(b, at);
  r.ctx = __builtin_amdgcn_readlane(len, at);
  r.split = __builtin_amdgcn_readlane(split, at);
  r.splits = __builtin_amdgcn_readlane(splits, at);
  before = __builtin_amdgcn_readlane(before, at);
  r.partial = (before & 0xffff) + r.split;
  r.index = before >> 16;
  r.cuts = __builtin_amdgcn_readlane(im, 63) >> 16;
  return r;
}

// Exclusive prefixes of x and y over the workgroup's threads, and their sums.
template <int WAVES>
__device__ __forceinline__ void block_scan(int& x, int& y, int (&sh)[2][WAVES], int* sum_x,
                                           int* sum_y) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int ix = scan_sum(x), iy = scan_sum(y);
  __syncthreads();   // sh may still be read
  if (lane == 63) {
    sh[0][wave] = ix;
    sh[1][wave] = iy;
  }
  __syncthreads();
  int bx = 0, by = 0;
  *sum_x = *sum_y = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    bx += w < wave ? sh[0][w] : 0;
    by += w < wave ? sh[1][w] : 0;
    *sum_x += sh[0][w];
    *sum_y += sh[1][w];
  }
  x = bx + ix - x;
  y = by + iy - y;
}

// The chunks of a batch of any size: table[0] has their number, table[1 + x]
// chunk x as (sequence, its length, split | splits << 16, partial); plan as the
// join reads it. One workgroup, a run of sequences a thread; a sequence's
// entries are written by the whole wave.
constexpr int kPlanWaves = 16;
__global__ void __launch_bounds__(64 * kPlanWaves)
fa_decode_mx_plan_kernel(const int32_t* __restrict__ ctx_lens, int B, int max_pages,
                         Plan chunk_plan, int4* __restrict__ table, int32_t* __restrict__ plan) {
  __shared__ int sh[2][kPlanWaves];
  const int tid = threadIdx.x, lane = tid & 63;
  const int per = (B + 64 * kPlanWaves - 1) / (64 * kPlanWaves);
  const int i0 = min(tid * per, B), i1 = min(i0 + per, B);
  int mine = 0, zero = 0, total, none;
  for (int i = i0; i < i1; ++i) mine += pages_of(ctx_lens[i], max_pages);
  block_scan<kPlanWaves>(mine, zero, sh, &total, &none);
  const int C = chunk_pages(total, chunk_plan);
  int n = 0, m = 0, chunks, cuts;
  for (int i = i0; i < i1; ++i) {
    int cut;
    n += chunks_of(pages_of(ctx_lens[i], max_pages), C, &cut);
    m += cut;
  }
  block_scan<kPlanWaves>(n, m, sh, &chunks, &cuts);
  if (tid == 0) {
    table[0] = int4{chunks, 0, 0, 0};
    plan[0] = cuts >> 16;
  }
  for (int k = 0; k < per; ++k) {
    const int i = i0 + k;
    int cut = 0, s = 0, ctx = 0;
    if (i < i1) {
      ctx = ctx_lens[i];
      s = chunks_of(pages_of(ctx, max_pages), C, &cut);
      if (s > 1) {
        plan[1 + 2 * (m >> 16)] = i;
        plan[2 + 2 * (m >> 16)] = (m & 0xffff) | s << 16;
      }
    }
    if (s == 1) table[1 + n] = int4{i, ctx, 1 << 16, 0};
    for (uint64_t rest = __ballot(s > 1); rest != 0; rest &= rest - 1) {
      const int l = __builtin_ctzll(rest);
      const int b = __builtin_amdgcn_readlane(i, l), cl = __builtin_amdgcn_readlane(ctx, l);
      const int sl = __builtin_amdgcn_readlane(s, l);
      const int nl = __builtin_amdgcn_readlane(n, l), ml = __builtin_amdgcn_readlane(m, l) & 0xffff;
      for (int j = lane; j < sl; j += 64) table[1 + nl + j] = int4{b, cl, j | sl << 16, ml + j};
    }
    n += s;
    m += cut;
  }
}

// Max and sum over the four lane groups of a column.
__device__ __forceinline__ float col_max(float x) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float col_sum(float x) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
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

// What pack2(a, b) = ab leaves out, rounded alike. fp16: a factor of -1 and words
// that the compiler does not see through make each difference one mixed fma, and
// keep it from rounding a and b a second time.
template <bool BF16>
__device__ __forceinline__ uint32_t rest2(float a, float b, uint32_t ab) {
  if constexpr (BF16) {
    return pack2<true>(a - __uint_as_float(ab << 16), b - __uint_as_float(ab & 0xffff0000u));
  } else {
    float neg = -1.f;
    asm("" : "+s"(neg));
    asm("" : "+v"(ab));
    const f16x2 h = __builtin_bit_cast(f16x2, ab);
    return pack2<false>(fmaf((float)h[0], neg, a), fmaf((float)h[1], neg, b));
  }
}

// A lane's piece of a page.
template <bool NT, int WORDS>
__device__ __forceinline__ void load_piece(__amdgpu_buffer_rsrc_t r, uint32_t off, uint32_t (&w)[WORDS]) {
  constexpr int kAux = NT ? 2 : 0;
  if constexpr (WORDS == 2) {
    const u32x2 x = __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, kAux);
    w[0] = x[0];
    w[1] = x[1];
  } else {
#pragma unroll
    for (int j = 0; j < WORDS / 4; ++j) {
      const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(r, off, 1024 * j, kAux);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[4 * j + i] = x[i];
    }
  }
}

// Clears the codes of a V piece's tokens from n on.
template <int WORDS>
__device__ __forceinline__ void keep_tokens(uint32_t (&w)[WORDS], int n) {
#pragma unroll
  for (int j = 0; j < WORDS; ++j) {
    if constexpr (WORDS == 2)
      w[j] &= n >= 2 * j + 2 ? 0xffffffffu : n > 2 * j ? 0xffffu : 0u;
    else
      w[j] = j / (WORDS / 4) < n ? w[j] : 0u;
  }
}

// What a wave holds of a batch of pages before it is multiplied.
template <int D, int KB, int VB>
struct Batch {
  static constexpr int kBatch = kBatchOf<D, KB, VB>;
  uint32_t k[kBatch][Page<D, KB>::WORDS];
  uint32_t v[kBatch][Page<D, VB>::WORDS];
  uint32_t ks[kBatch], vs[kBatch];
};

// Values 2 i and 2 i + 1 of token r of a lane's V piece.
template <int D, int VB, bool BF16, int R, int I>
__device__ __forceinline__ uint32_t v_pair(const uint32_t (&w)[Page<D, VB>::WORDS], float scale) {
  constexpr int N = D / 16 * R + 2 * I;   // number of the value in the piece
  constexpr int PER = 32 / VB;            // values of a word
  return values2<VB, BF16, N % PER / 2>(w[N / PER], scale);
}

// NT: the pages are read with the non-temporal hint.
template <int D, int KB, int VB, bool BF16, bool NT, int WAVES>
__global__ void __launch_bounds__(64 * WAVES)
fa_decode_mx_kernel(const uint16_t* __restrict__ q, const char* __restrict__ k_pool,
                    const char* __restrict__ v_pool, const int32_t* __restrict__ page_table,
                    const int32_t* __restrict__ ctx_lens, float* __restrict__ part_o,
                    float2* __restrict__ part_ml, const int4* __restrict__ table,
                    int32_t* __restrict__ plan, uint16_t* __restrict__ o, float* __restrict__ lse,
                    int B, int H, int Hkv, int group, int ngrp, int max_pages, int num_pages,
                    int slots, Plan chunk_plan, float c) {
  using PK = Page<D, KB>;
  using PV = Page<D, VB>;
  constexpr int kBatch = kBatchOf<D, KB, VB>;
  constexpr int KS = D / 32;   // steps of S = K Q^T
  constexpr int DB = D / 16;   // blocks of O^T
  __shared__ __attribute__((aligned(16))) float sh_o[WAVES][16][D + 4];   // heads in different banks
  __shared__ float sh_m[WAVES][16], sh_l[WAVES][16];
  __shared__ int sh_bad[WAVES];

  // Workgroups go to the XCDs in turn: an XCD has every eighth chunk, and the
  // head groups of a chunk one after the other, so that what is read of a page
  // at about the same time by one L2 is contiguous.
  const int number = blockIdx.y * kXcds + blockIdx.x % kXcds, hg = blockIdx.x / kXcds;
  const int hk = ngrp == 1 ? hg : hg / ngrp, sub = ngrp == 1 ? 0 : hg % ngrp;
  const int h0 = hk * group + 16 * sub;   // first query head of this workgroup
  const int G = min(16, group - 16 * sub);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, grp = lane >> 4;

  Chunk ch;
  if (plan == nullptr) {   // nothing is cut: a chunk a sequence
    ch.b = number < B ? number : -1;
    ch.ctx = ctx_lens[min(number, B - 1)];
    ch.split = ch.partial = 0;
    ch.splits = 1;
  } else if (table != nullptr) {
    const int chunks = table[0].x;
    const int4 e = table[1 + number];
    ch.b = number < chunks ? e.x : -1;
    ch.ctx = e.y;
    ch.split = e.z & 0xffff;
    ch.splits = e.z >> 16;
    ch.partial = e.w;
  } else {
    ch = chunk_of(ctx_lens, B, max_pages, chunk_plan, number);
  }
  ch.b = __builtin_amdgcn_readfirstlane(ch.b);
  if (ch.b < 0) return;
  const int ctx = __builtin_amdgcn_readfirstlane(ch.ctx);
  const int pages = pages_of(ctx, max_pages);
  ch.split = __builtin_amdgcn_readfirstlane(ch.split);
  ch.splits = __builtin_amdgcn_readfirstlane(ch.splits);
  // The first pages % splits chunks have a page more: none is empty.
  const int each = (int)((unsigned)pages / (unsigned)ch.splits), more = pages - each * ch.splits;
  const int p0 = ch.split * each + min(ch.split, more), p1 = p0 + each + (ch.split < more);
  // This wave's pages.
  const int w0 = p0 + (p1 - p0) * wave / WAVES, w1 = p0 + (p1 - p0) * (wave + 1) / WAVES;
  bool bad = ctx < 0 || (ctx > 0 && pages == 0);

  const uint32_t koff = (4 * col + grp) * (PK::PIECE < 16 ? PK::PIECE : 16);
  const uint32_t voff = lane * (PV::PIECE < 16 ? PV::PIECE : 16);
  const uint32_t ksoff = k_scale<D, KB>(col, grp * PK::BLOCKS / 4);
  const uint32_t vsoff = v_scale<D, VB>(4 * grp, col * PV::BLOCKS / 16);
  const int32_t* pt = page_table + (size_t)ch.b * max_pages;

  float m = -INFINITY, l = 0.f;
  f32x4 acc[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) acc[db] = f32x4{};

  // Pages w .. + kBatch - 1, all loads at once; past the wave's last page they
  // repeat it (masked below). Four waves a SIMD hide each other's waits: a
  // second set of registers, loaded one batch ahead, leaves three and measured
  // slower (32 sequences of up to 32768 tokens by 1 %, one of 32000 by 8), and so
  // did loading K and V each as soon as their registers are free (6 and 8 %).
  int ids = 0;   // lane i: id of the wave's page 64 j + i
  Batch<D, KB, VB> x;
  const auto load_ids = [&](int w) { ids = pt[min(w + lane, w1 - 1)]; };
  if (w0 < w1) load_ids(w0);   // before Q, which is not waited for until the first scores
  // Q^T operand: column col = head h0 + col, step kb of the lane's quarter of D.
  u32x4 qf[KS];
#pragma unroll
  for (int kb = 0; kb < KS; ++kb) {
    qf[kb] = u32x4{};
    if (col < G)
      qf[kb] = *reinterpret_cast<const u32x4*>(q + ((size_t)ch.b * H + h0 + col) * D +
                                               grp * (D / 4) + 8 * kb);
  }

  const auto load = [&](int w) {
    if (((w - w0) & 63) == 0) {
      if (w != w0) load_ids(w);
      const bool no = ids < 0 || ids >= num_pages;
      bad |= no;
      ids = no ? 0 : ids;   // read in place of a page that is not there; the result is NaN
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const size_t rec = (size_t)__builtin_amdgcn_readlane(ids, (w - w0 + i) & 63) * Hkv + hk;
      const auto r = make_rsrc(k_pool + rec * PK::BYTES, PK::BYTES);
      load_piece<NT>(r, koff, x.k[i]);
      x.ks[i] = __builtin_amdgcn_raw_buffer_load_b8(r, ksoff, 0, 0);
      const auto t = make_rsrc(v_pool + rec * PV::BYTES, PV::BYTES);
      load_piece<NT>(t, voff, x.v[i]);
      x.vs[i] = __builtin_amdgcn_raw_buffer_load_b32(t, vsoff, 0, 0);
    }
  };
  for (int w = w0; w < w1; w += kBatch) {
    load(w);
    // Tokens of the batch that the wave has; from the lane's first.
    const int rem = min(ctx, w1 * kTokens) - w * kTokens, lim = rem - 4 * grp;
    const bool tail = rem < kBatch * kTokens;   // wave-uniform

    f32x4 s[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const float sc = scale_of(x.ks[i]);
      s[i] = f32x4{};
      static_for<0, KS>([&](auto kb) {
        u32x4 a;
        static_for<0, 4>([&](auto j) {
          constexpr int N = 8 * kb.value + 2 * j.value, PER = 32 / KB;
          a[j.value] = values2<KB, BF16, N % PER / 2>(x.k[i][N / PER], sc);
        });
        s[i] = mma16<BF16>(a, qf[kb.value], s[i]);
      });
    }
    if (tail) {
      asm volatile("");   // a branch: not selects in every batch
      // Rows past the context may hold NaN, and 0 NaN is NaN: V's become zeros.
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
#pragma unroll
        for (int r = 0; r < 4; ++r) s[i][r] = kTokens * i + r < lim ? s[i][r] : -INFINITY;
        const int n = min(max(lim - kTokens * i, 0), 4);   // of the lane's four tokens
        x.vs[i] &= (uint32_t)((1ull << (8 * n)) - 1);
        keep_tokens<PV::WORDS>(x.v[i], n);
      }
    }
    float top = s[0][0];
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) top = fmaxf(top, s[i][r]);
    const float m_new = fmaxf(m, col_max(top));
    if (__any(m_new != m)) {   // also where one of them is NaN
      const float alpha = m_new == m ? 1.f : exp2_hw((m - m_new) * c);
      l *= alpha;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[db][r] *= alpha;
      m = m_new;
    }
    u32x2 ph[kBatch], pl[kBatch];   // P's two terms
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      float p[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        p[r] = exp2_hw(fmaf(s[i][r] - m, c, kShift<BF16>));
        l += p[r];
      }
      ph[i] = u32x2{pack2<BF16>(p[0], p[1]), pack2<BF16>(p[2], p[3])};
      pl[i] = u32x2{rest2<BF16>(p[0], p[1], ph[i][0]), rest2<BF16>(p[2], p[3], ph[i][1])};
    }
    // Two pages a product: slots 0 .. 3 of the lane's reduction are tokens
    // 4 grp .. + 3 of the first, slots 4 .. 7 those of the second.
    static_for<0, kBatch / 2>([&](auto half) {
      constexpr int I0 = 2 * half.value;
      const u32x4 bh = u32x4{ph[I0][0], ph[I0][1], ph[I0 + 1][0], ph[I0 + 1][1]};
      const u32x4 bl = u32x4{pl[I0][0], pl[I0][1], pl[I0 + 1][0], pl[I0 + 1][1]};
      static_for<0, DB / 2>([&](auto qd) {
        u32x4 even, odd;   // values 2 qd and 2 qd + 1 of the lane's sixteenth
        static_for<0, 2>([&](auto j) {
          constexpr int I = I0 + j.value;
          uint32_t v[4];
          static_for<0, 4>([&](auto r) {
            v[r.value] = v_pair<D, VB, BF16, r.value, qd.value>(x.v[I], scale_at<r.value>(x.vs[I]));
          });
          even[2 * j.value] = __builtin_amdgcn_perm(v[1], v[0], 0x05040100u);
          even[2 * j.value + 1] = __builtin_amdgcn_perm(v[3], v[2], 0x05040100u);
          odd[2 * j.value] = __builtin_amdgcn_perm(v[1], v[0], 0x07060302u);
          odd[2 * j.value + 1] = __builtin_amdgcn_perm(v[3], v[2], 0x07060302u);
        });
        acc[2 * qd.value] = mma16<BF16>(even, bh, acc[2 * qd.value]);
        acc[2 * qd.value + 1] = mma16<BF16>(odd, bh, acc[2 * qd.value + 1]);
        acc[2 * qd.value] = mma16<BF16>(even, bl, acc[2 * qd.value]);
        acc[2 * qd.value + 1] = mma16<BF16>(odd, bl, acc[2 * qd.value + 1]);
      });
    });
  }
  l = col_sum(l);

  // The waves' parts join in LDS. acc[db][r] is value (4 grp + r) D/16 + db.
  const bool wave_bad = __any(bad);
  if (lane == 0) sh_bad[wave] = wave_bad;
  if (col < G) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int db = 0; db < DB; ++db) sh_o[wave][col][(4 * grp + r) * DB + db] = acc[db][r];
    if (grp == 0) {
      sh_m[wave][col] = m;
      sh_l[wave][col] = l;
    }
  }
  __syncthreads();
  bool any_bad = false;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) any_bad |= sh_bad[w] != 0;
  if (plan != nullptr && table == nullptr && hg == 0 && tid == 0) {   // for the pass that joins
    if (number == 0) plan[0] = ch.cuts;
    if (ch.splits > 1 && ch.split == 0) {
      plan[1 + 2 * ch.index] = ch.b;
      plan[2 + 2 * ch.index] = ch.partial | ch.splits << 16;
    }
  }
  // A thread has four columns of a head.
  for (int i = tid; i < G * (D / 4); i += 64 * WAVES) {
    const int g = i / (D / 4), d = 4 * (i % (D / 4));
    float wm[WAVES], wl[WAVES];
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      wm[w] = sh_m[w][g];
      wl[w] = sh_l[w][g];
    }
    float M = wm[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) M = fmaxf(M, wm[w]);
    f32x4 a = f32x4{};
    float z = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      // A wave without pages has m = -inf; its sums are 0.
      const float e = wl[w] == 0.f ? 0.f : exp2_hw((wm[w] - M) * c);
      const f32x4 v = *reinterpret_cast<const f32x4*>(&sh_o[w][g][d]);
      z = fmaf(e, wl[w], z);
#pragma unroll
      for (int j = 0; j < 4; ++j) a[j] = fmaf(e, v[j], a[j]);
    }
    if (any_bad) z = NAN;
    const float inv = z == 0.f ? 0.f : 1.f / z;
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] *= inv;
    if (ch.splits == 1) {
      const size_t row = (size_t)ch.b * H + h0 + g;
      *reinterpret_cast<u32x2*>(o + row * D + d) = u32x2{pack2<BF16>(a[0], a[1]), pack2<BF16>(a[2], a[3])};
      if (lse != nullptr && d == 0)
        lse[row] = z == 0.f ? -INFINITY : fmaf(M, c, log2_hw(z) - kShift<BF16>) * kLn2;
    } else {
      const size_t row = (size_t)(h0 + g) * slots + ch.partial;
      *reinterpret_cast<f32x4*>(part_o + row * D + d) = a;
      if (d == 0) part_ml[row] = float2{M, z * kPartScale<BF16>};
    }
  }
}

constexpr int kJoinWaves = 4;

// Joins the chunks of cut sequence blockIdx.x, head blockIdx.y: a wave has 32
// columns of the row (WAVES = 1) or kJoinWaves waves share them, eight lanes for
// four columns each in as many groups as there are, the chunks dealt out over
// the groups. One pass, with a running maximum.
template <int D, bool BF16, int WAVES>
__global__ void __launch_bounds__(WAVES == 1 ? 2 * D : 64 * kJoinWaves)
fa_decode_mx_join_kernel(const float* __restrict__ part_o, const float2* __restrict__ part_ml,
                         const int32_t* __restrict__ plan, uint16_t* __restrict__ o,
                         float* __restrict__ lse, int H, int slots, float c) {
  constexpr int GROUPS = 8 * WAVES, AHEAD = 4;
  __shared__ __attribute__((aligned(16))) f32x4 sh_a[kJoinWaves][8];
  __shared__ float sh_m[kJoinWaves], sh_z[kJoinWaves];
  const int cuts = plan[0], b = plan[1 + 2 * blockIdx.x], word = plan[2 + 2 * blockIdx.x];
  if ((int)blockIdx.x >= cuts) return;
  const int first = word & 0xffff, n = word >> 16;
  const int h = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int d = 32 * (WAVES == 1 ? wave : (int)blockIdx.z) + 4 * (lane & 7);
  const int g = WAVES == 1 ? lane >> 3 : 8 * wave + (lane >> 3);
  const float2* pl = part_ml + (size_t)h * slots + first;
  const float* po = part_o + ((size_t)h * slots + first) * D + d;

  float m = -INFINITY, z = 0.f;
  f32x4 a = f32x4{};
  for (int i = g; i < n; i += AHEAD * GROUPS) {
    float2 x[AHEAD];
    f32x4 v[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int k = min(i + j * GROUPS, n - 1);
      x[j] = i + j * GROUPS < n ? pl[k] : float2{-INFINITY, 0.f};
      v[j] = *reinterpret_cast<const f32x4*>(po + (size_t)k * D);
    }
    float top = m;   // finite or, with a NaN to come, -inf: a chunk of a cut sequence has tokens
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) top = fmaxf(top, x[j].x);
    const float e = exp2_hw((m - top) * c);
    z *= e;
#pragma unroll
    for (int k = 0; k < 4; ++k) a[k] *= e;
    m = top;
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const float w = x[j].y * exp2_hw((x[j].x - m) * c);
      z += w;
#pragma unroll
      for (int k = 0; k < 4; ++k) a[k] = fmaf(w, v[j][k], a[k]);
    }
  }
  // The groups of the wave, then the waves.
  float M = m;
#pragma unroll
  for (int k = 8; k < 64; k *= 2) M = fmaxf(M, __shfl_xor(M, k));
  const float e = m == M ? 1.f : exp2_hw((m - M) * c);   // a group without chunks: m = -inf, its sums 0
  z *= e;
#pragma unroll
  for (int j = 0; j < 4; ++j) a[j] *= e;
#pragma unroll
  for (int k = 8; k < 64; k *= 2) {
    z += __shfl_xor(z, k);
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] += __shfl_xor(a[j], k);
  }
  if constexpr (WAVES > 1) {
    if (lane < 8) sh_a[wave][lane] = a;
    if (lane == 0) {
      sh_m[wave] = M;
      sh_z[wave] = z;
    }
    __syncthreads();
    if (wave != 0) return;
    M = sh_m[0];
#pragma unroll
    for (int w = 1; w < kJoinWaves; ++w) M = fmaxf(M, sh_m[w]);
    z = 0.f;
    a = f32x4{};
#pragma unroll
    for (int w = 0; w < kJoinWaves; ++w) {
      const float f = sh_m[w] == M ? 1.f : exp2_hw((sh_m[w] - M) * c);
      const f32x4 v = sh_a[w][lane & 7];
      z = fmaf(f, sh_z[w], z);
#pragma unroll
      for (int j = 0; j < 4; ++j) a[j] = fmaf(f, v[j], a[j]);
    }
  }
  if (lane >= 8) return;
  const size_t row = (size_t)b * H + h;
  const float inv = 1.f / z;
  *reinterpret_cast<u32x2*>(o + row * D + d) =
      u32x2{pack2<BF16>(a[0] * inv, a[1] * inv), pack2<BF16>(a[2] * inv, a[3] * inv)};
  if (lse != nullptr && d == 0) lse[row] = fmaf(M, c, log2_hw(z * kJoinScale)) * kLn2;
}

template <int D, int KB, int VB, bool BF16>
static int decode(const void* q, const void* k_pool, const void* v_pool, const int32_t* page_table,
                  const int32_t* ctx_lens, int64_t B, int64_t H, int64_t Hkv, int64_t max_pages,
                  int64_t num_pages, float* workspace, void* o, float* lse, hipStream_t s) {
  const float c = (float)(1.0 / sqrt((double)D)) * kLog2e;
  const int64_t most = most_chunks(B, H, Hkv, max_pages);
  const bool one = never_cut(B, H, Hkv, max_pages);
  const Workspace w = workspace_of(B, H, D, most);
  float* part_o = one ? nullptr : workspace + w.part_o;
  float2* part_ml = one ? nullptr : reinterpret_cast<float2*>(workspace + w.part_ml);
  int32_t* plan = one ? nullptr : reinterpret_cast<int32_t*>(workspace + w.plan);
  int4* table = one || B <= kWavePlan ? nullptr : reinterpret_cast<int4*>(workspace);
  if (table != nullptr) {
    hipLaunchKernelGGL(fa_decode_mx_plan_kernel, dim3(1), dim3(64 * kPlanWaves), 0, s, ctx_lens, (int)B,
                       (int)max_pages, plan_of(B, H, Hkv), table, plan);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return -(int)e;
  }
  const dim3 grid((unsigned)(kXcds * head_groups(H, Hkv)),
                  (unsigned)chunk_rows(B, one ? 0 : most));
  const bool nt = num_pages * Hkv * (Page<D, KB>::BYTES + Page<D, VB>::BYTES) >= kPassThrough;
  // Eight waves where nothing is cut and a CU has one workgroup at most (32
  // sequences of 2048 tokens over 8 KV heads 20.5 -> 16.3 us, 8 of 512 5.3 ->
  // 5.2); four where there are more (32 of 768 over 32 heads, D = 64: 12.7 and
  // 17.0) or where four take a batch each (one of 130 tokens, D = 64: 3.4 and 4.3).
  const int64_t groups = head_groups(H, Hkv);
  const int waves = one && max_pages > kMinChunk && B * groups <= kFill / 4 ? 8 : 4;
  const auto kernel = waves == 8 ? (nt ? fa_decode_mx_kernel<D, KB, VB, BF16, true, 8>
                                       : fa_decode_mx_kernel<D, KB, VB, BF16, false, 8>)
                                 : (nt ? fa_decode_mx_kernel<D, KB, VB, BF16, true, 4>
                                       : fa_decode_mx_kernel<D, KB, VB, BF16, false, 4>);
  hipLaunchKernelGGL(kernel, grid, dim3(64 * waves), 0, s, (const uint16_t*)q, (const char*)k_pool,
                     (const char*)v_pool, page_table, ctx_lens, part_o, part_ml, table, plan,
                     (uint16_t*)o, lse, (int)B, (int)H, (int)Hkv, (int)(H / Hkv),
                     (int)(groups / Hkv), (int)max_pages, (int)num_pages, (int)w.slots,
                     plan_of(B, H, Hkv), c);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return -(int)e;
  if (one) return FA_OK;
  const unsigned cut = (unsigned)(B < most ? B : most);
  if (most > kWideJoin * B)
    hipLaunchKernelGGL((fa_decode_mx_join_kernel<D, BF16, kJoinWaves>), dim3(cut, (unsigned)H, D / 32),
                       dim3(64 * kJoinWaves), 0, s, part_o, part_ml, plan, (uint16_t*)o, lse, (int)H,
                       (int)w.slots, c);
  else
    hipLaunchKernelGGL((fa_decode_mx_join_kernel<D, BF16, 1>), dim3(cut, (unsigned)H), dim3(2 * D), 0,
                       s, part_o, part_ml, plan, (uint16_t*)o, lse, (int)H, (int)w.slots, c);
  e = hipGetLastError();
  return e == hipSuccess ? FA_OK : -(int)e;
}

}  // namespace mx
}  // namespace fa

extern "C" int64_t fa_decode_mx_workspace_floats(int64_t B, int64_t H, int64_t H_kv, int64_t D,
                                                 int64_t max_pages) {
  // the sizes that fa_validate_decode_mx refuses
  constexpr int64_t kIndexes = (int64_t(1) << 31) - 1;
  if (B <= 0 || B > 65535 || H <= 0 || H > 65535 || H_kv <= 0 || H % H_kv != 0 ||
      (D != 64 && D != 128) || max_pages <= 0 || max_pages > kIndexes / fa::mx::kTokens ||
      B > kIndexes / max_pages)
    return 0;
  if (fa::mx::never_cut(B, H, H_kv, max_pages)) return 0;
  return fa::mx::workspace_of(B, H, D, fa::mx::most_chunks(B, H, H_kv, max_pages)).words;
}

extern "C" int fa_decode_paged_mx(const void* q, const void* k_pool, const void* v_pool,
                                  const int32_t* page_table, const int32_t* ctx_lens, int64_t B,
                                  int64_t H, int64_t H_kv, int64_t D, int64_t k_bits,
                                  int64_t v_bits, int64_t page_size, int64_t max_pages,
                                  int64_t num_pages, float* workspace, void* o, float* lse,
                                  int bf16, void* stream) {
  const int st = fa_validate_decode_mx(q, k_pool, v_pool, page_table, ctx_lens, B, H, H_kv, D, k_bits,
                                       v_bits, page_size, max_pages, num_pages, workspace, o, lse);
  if (st != FA_OK) return st;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define FA_MX_DECODE(DD, KB, VB, BF)                                                               \
  return fa::mx::decode<DD, KB, VB, BF>(q, k_pool, v_pool, page_table, ctx_lens, B, H, H_kv,       \
                                        max_pages, num_pages, workspace, o, lse, s)
  FA_MX_DISPATCH(D, k_bits, v_bits, bf16, FA_MX_DECODE)
#undef FA_MX_DECODE
}

extern "C" int fa_probe_mx_chunks(int64_t B, int64_t H, int64_t H_kv, int64_t max_pages, int64_t total,
                                  int64_t* most) {
  if (B <= 0 || H <= 0 || H_kv <= 0 || H % H_kv != 0 || max_pages <= 0 || total < 0 ||
      B > ((int64_t(1) << 31) - 1) / max_pages || total > B * max_pages)
    return 0;
  if (fa::mx::never_cut(B, H, H_kv, max_pages)) {
    if (most != nullptr) *most = 0;
    return (int)(total > 0 ? total : 1);
  }
  if (most != nullptr) *most = fa::mx::most_chunks(B, H, H_kv, max_pages);
  return fa::mx::chunk_pages((int)total, fa::mx::plan_of(B, H, H_kv));
}
