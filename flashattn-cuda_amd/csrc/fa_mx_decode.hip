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
// Lane l has head l % 16 in both products, so a head's maximum and sum stay in
// its lane column.
#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include "fa_mi355x.h"
#include "fa_mx.hpp"

namespace fa {
namespace mx {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kBatch = 4;   // pages that a wave takes at a time

// Chunks. The pages of all sequences, T in all, are cut into runs of
// C = max(kMinChunk, T / kTargetChunks per head group) pages, a sequence into
// ceil(pages / C) nearly equal ones: workgroups of like size whatever the
// lengths, about kTargetChunks of them, from lengths that only the device
// knows. The grid has the most chunks that any lengths can give, and the rest
// end at once.
constexpr int kTargetChunks = 512;
constexpr int kMinChunk = 16;

static int64_t head_groups(int64_t H, int64_t Hkv) { return Hkv * ((H / Hkv + 15) / 16); }
// Chunks along the pages that each head group is cut into, at most this many
// and one a sequence: sum ceil(p / C) <= T / C + B.
static int64_t target_chunks(int64_t H, int64_t Hkv) {
  const int64_t g = head_groups(H, Hkv);
  return (kTargetChunks + g - 1) / g;
}
// Chunks of the sequences that are cut at all: ceil(p / C) < 2 p / C of each.
static int64_t partial_chunks(int64_t B, int64_t H, int64_t Hkv) {
  const int64_t w = target_chunks(H, Hkv);
  return w + (B < w ? B : w);
}

// What a workgroup's chunk is.
struct Chunk {
  int b;        // sequence, -1: none
  int split, splits;
  int partial;  // of the sequence's first chunk, among those of cut sequences
  int cut;      // the sequence's number among those
  int cuts;     // cut sequences in all
};

__device__ __forceinline__ int pages_of(int ctx, int max_pages) {
  const int64_t p = ((int64_t)ctx + kTokens - 1) / kTokens;
  return ctx <= 0 || p > max_pages ? 0 : (int)p;   // of an invalid length: none
}

// Exclusive prefix over the workgroup's threads, and the sum.
__device__ __forceinline__ int block_scan(int x, int* sh, int* total) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int inc = scan_sum(x);
  if (lane == 63) sh[wave] = inc;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const int t = sh[w];
    before += w < wave ? t : 0;
    all += t;
  }
  __syncthreads();
  *total = all;
  return before + inc - x;
}

// Chunk number x of the batch.
__device__ __forceinline__ Chunk chunk_of(const int32_t* __restrict__ ctx_lens, int B,
                                          int max_pages, int target, int x, int* sh) {
  Chunk r;
  if (B == 1) {
    const int p = pages_of(ctx_lens[0], max_pages);
    const int C = max(kMinChunk, (p + target - 1) / target);
    r.splits = max(1, (p + C - 1) / C);
    r.b = x < r.splits ? 0 : -1;
    r.split = x;
    r.partial = 0;
    r.cut = 0;
    r.cuts = r.splits > 1;
    return r;
  }
  const int per = (B + kThreads - 1) / kThreads;
  const int i0 = (int)threadIdx.x * per, i1 = min(i0 + per, B);
  int mine = 0, total;
  for (int i = i0; i < i1; ++i) mine += pages_of(ctx_lens[i], max_pages);
  block_scan(mine, sh, &total);
  const int C = max(kMinChunk, (total + target - 1) / target);
  // Chunks, and of the cut sequences (chunks, sequences) in one number: their
  // chunks are less than 2 target + 1.
  int n = 0, m = 0, all;
  for (int i = i0; i < i1; ++i) {
    const int s = (pages_of(ctx_lens[i], max_pages) + C - 1) / C;
    n += max(1, s);
    m += s > 1 ? (s | 1 << 16) : 0;
  }
  int e = block_scan(n, sh, &all);
  int f = block_scan(m, sh, &total);
  if (threadIdx.x == 0) sh[0] = -1;
  __syncthreads();
  if (x >= e && x < e + n) {   // one thread
    for (int i = i0; i < i1; ++i) {
      const int s = (pages_of(ctx_lens[i], max_pages) + C - 1) / C;
      if (x < e + max(1, s)) {
        sh[0] = i;
        sh[1] = x - e;
        sh[2] = max(1, s);
        sh[3] = f;
        break;
      }
      e += max(1, s);
      f += s > 1 ? (s | 1 << 16) : 0;
    }
  }
  __syncthreads();
  r.b = sh[0];
  r.split = sh[1];
  r.splits = sh[2];
  r.partial = sh[3] & 0xffff;
  r.cut = sh[3] >> 16;
  r.cuts = total >> 16;
  __syncthreads();
  return r;
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

// A lane's piece of a page.
template <int WORDS>
__device__ __forceinline__ void load_piece(const char* p, uint32_t (&w)[WORDS]) {
  if constexpr (WORDS == 2) {
    const u32x2 x = *reinterpret_cast<const u32x2*>(p);
    w[0] = x[0];
    w[1] = x[1];
  } else {
#pragma unroll
    for (int j = 0; j < WORDS / 4; ++j) {
      const u32x4 x = *reinterpret_cast<const u32x4*>(p + 1024 * j);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[4 * j + i] = x[i];
    }
  }
}

// What a wave holds of a batch of pages before it is multiplied.
template <int D, int KB, int VB>
struct Batch {
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

template <int D, int KB, int VB, bool BF16>
__global__ void __launch_bounds__(kThreads)
fa_decode_mx_kernel(const uint16_t* __restrict__ q, const char* __restrict__ k_pool,
                    const char* __restrict__ v_pool, const int32_t* __restrict__ page_table,
                    const int32_t* __restrict__ ctx_lens, float* __restrict__ part_o,
                    float* __restrict__ part_l, int32_t* __restrict__ plan,
                    uint16_t* __restrict__ o, float* __restrict__ lse, int B, int H, int Hkv,
                    int max_pages, int num_pages, int target, float c) {
  using PK = Page<D, KB>;
  using PV = Page<D, VB>;
  constexpr int KS = D / 32;   // steps of S = K Q^T
  constexpr int DB = D / 16;   // blocks of O^T
  // P reaches 2^15 in fp16 rather than 1, so that it keeps all its bits down to
  // 2^-29 of the row's largest (and some to 2^-39); bf16 has fp32's range.
  constexpr float kShift = BF16 ? 0.f : 15.f;
  __shared__ __attribute__((aligned(16))) float sh_o[kWaves][16][D + 4];   // heads in different banks
  __shared__ float sh_m[kWaves][16], sh_l[kWaves][16];
  __shared__ int sh_i[4];
  __shared__ int sh_bad;

  const int group = H / Hkv, ngrp = (group + 15) / 16;
  const int hk = blockIdx.y / ngrp;
  const int h0 = hk * group + 16 * (blockIdx.y % ngrp);   // first query head of this workgroup
  const int G = min(16, hk * group + group - h0);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, grp = lane >> 4;

  if (tid == 0) sh_bad = 0;
  Chunk ch = chunk_of(ctx_lens, B, max_pages, target, (int)blockIdx.x, sh_i);
  ch.b = __builtin_amdgcn_readfirstlane(ch.b);
  if (ch.b < 0) return;
  ch.split = __builtin_amdgcn_readfirstlane(ch.split);
  ch.splits = __builtin_amdgcn_readfirstlane(ch.splits);
  const int ctx = ctx_lens[ch.b];
  const int pages = __builtin_amdgcn_readfirstlane(pages_of(ctx, max_pages));
  const int len = (pages + ch.splits - 1) / ch.splits;
  const int p0 = min(ch.split * len, pages), p1 = min(p0 + len, pages);
  // This wave's pages.
  const int w0 = p0 + (p1 - p0) * wave / kWaves, w1 = p0 + (p1 - p0) * (wave + 1) / kWaves;
  bool bad = ctx < 0 || (ctx > 0 && pages == 0);

  // Q^T operand: column col = head h0 + col, step kb of the lane's quarter of D.
  u32x4 qf[KS];
#pragma unroll
  for (int kb = 0; kb < KS; ++kb) {
    qf[kb] = u32x4{};
    if (col < G)
      qf[kb] = *reinterpret_cast<const u32x4*>(q + ((size_t)ch.b * H + h0 + col) * D +
                                               grp * (D / 4) + 8 * kb);
  }

  const int koff = (4 * col + grp) * (PK::PIECE < 16 ? PK::PIECE : 16);
  const int voff = lane * (PV::PIECE < 16 ? PV::PIECE : 16);
  const int ksoff = k_scale<D, KB>(col, grp * PK::BLOCKS / 4);
  const int vsoff = v_scale<D, VB>(4 * grp, col * PV::BLOCKS / 16);
  const int32_t* pt = page_table + (size_t)ch.b * max_pages;

  float m = -INFINITY, l = 0.f;
  f32x4 acc[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) acc[db] = f32x4{};

  int ids = 0;   // lane i: page w0 + 64 j + i of the sequence
  for (int w = w0; w < w1; w += kBatch) {
    if (((w - w0) & 63) == 0) {
      ids = w + lane < w1 ? pt[w + lane] : 0;
      const bool no = ids < 0 || ids >= num_pages;
      bad |= no;
      ids = no ? 0 : ids;   // read in place of a page that is not there; the result is NaN
    }
    Batch<D, KB, VB> x;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {   // past w1: page 0, masked below
      const int pid = __builtin_amdgcn_readlane(ids, (w - w0 + i) & 63);
      const size_t rec = (size_t)pid * Hkv + hk;
      const char* kp = k_pool + rec * PK::BYTES;
      const char* vp = v_pool + rec * PV::BYTES;
      load_piece(kp + koff, x.k[i]);
      x.ks[i] = (uint8_t)kp[ksoff];
      load_piece(vp + voff, x.v[i]);
      x.vs[i] = *reinterpret_cast<const uint32_t*>(vp + vsoff);
    }
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
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[i][r] = kTokens * i + r < lim ? s[i][r] : -INFINITY;
    }
    float top = s[0][0];
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) top = fmaxf(top, s[i][r]);
    const float m_new = fmaxf(m, col_max(top) * c);
    if (__any(m_new != m)) {   // also where one of them is NaN
      const float alpha = m_new == m ? 1.f : exp2_hw(m - m_new);
      l *= alpha;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[db][r] *= alpha;
      m = m_new;
    }
    const float ref = m - kShift;
    u32x2 ph[kBatch], pl[kBatch];   // P as 16-bit operands, and in bf16 what the first leaves out
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      float p[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        p[r] = exp2_hw(fmaf(s[i][r], c, -ref));
        l += p[r];
      }
      ph[i] = u32x2{pack2<BF16>(p[0], p[1]), pack2<BF16>(p[2], p[3])};
      if constexpr (BF16) {
        // bf16 keeps 8 bits of P; a second product with the rounded remainder
        // makes them 16.
        const auto lo = [](uint32_t x) { return __uint_as_float(x << 16); };
        const auto hi = [](uint32_t x) { return __uint_as_float(x & 0xffff0000u); };
        pl[i] = u32x2{pack2<true>(p[0] - lo(ph[i][0]), p[1] - hi(ph[i][0])),
                      pack2<true>(p[2] - lo(ph[i][1]), p[3] - hi(ph[i][1]))};
      }
    }
    // Two pages a product: slots 0 .. 3 of the lane's reduction are tokens
    // 4 grp .. + 3 of the first, slots 4 .. 7 those of the second.
    static_for<0, kBatch / 2>([&](auto half) {
      constexpr int I0 = 2 * half.value;
      const u32x4 bh = u32x4{ph[I0][0], ph[I0][1], ph[I0 + 1][0], ph[I0 + 1][1]};
      static_for<0, DB / 2>([&](auto qd) {
        u32x4 even, odd;   // values 2 qd and 2 qd + 1 of the lane's sixteenth
        static_for<0, 2>([&](auto j) {
          constexpr int I = I0 + j.value;
          uint32_t v[4];
          static_for<0, 4>([&](auto r) {
            const uint32_t e = (x.vs[I] >> (8 * r.value)) & 0xffu;
            v[r.value] = v_pair<D, VB, BF16, r.value, qd.value>(x.v[I], scale_of(e));
            // Rows past the context may hold NaN, and 0 NaN is NaN.
            if (tail) v[r.value] = kTokens * I + r.value < lim ? v[r.value] : 0u;
          });
          even[2 * j.value] = __builtin_amdgcn_perm(v[1], v[0], 0x05040100u);
          even[2 * j.value + 1] = __builtin_amdgcn_perm(v[3], v[2], 0x05040100u);
          odd[2 * j.value] = __builtin_amdgcn_perm(v[1], v[0], 0x07060302u);
          odd[2 * j.value + 1] = __builtin_amdgcn_perm(v[3], v[2], 0x07060302u);
        });
        acc[2 * qd.value] = mma16<BF16>(even, bh, acc[2 * qd.value]);
        acc[2 * qd.value + 1] = mma16<BF16>(odd, bh, acc[2 * qd.value + 1]);
        if constexpr (BF16) {
          const u32x4 bl = u32x4{pl[I0][0], pl[I0][1], pl[I0 + 1][0], pl[I0 + 1][1]};
          acc[2 * qd.value] = mma16<true>(even, bl, acc[2 * qd.value]);
          acc[2 * qd.value + 1] = mma16<true>(odd, bl, acc[2 * qd.value + 1]);
        }
      });
    });
  }
  l = col_sum(l);

  // The waves' parts join in LDS. acc[db][r] is value (4 grp + r) D/16 + db.
  if (__any(bad) && lane == 0) sh_bad = 1;
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
  if (plan != nullptr && blockIdx.y == 0 && tid == 0) {   // for the pass that joins the chunks
    if (blockIdx.x == 0) plan[0] = ch.cuts;
    if (ch.splits > 1 && ch.split == 0) {
      plan[1 + 2 * ch.cut] = ch.b;
      plan[2 + 2 * ch.cut] = ch.partial | ch.splits << 16;
    }
  }
  for (int i = tid; i < G * D; i += kThreads) {
    const int g = i / D, d = i % D;
    float M = sh_m[0][g];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) M = fmaxf(M, sh_m[w][g]);
    float a = 0.f, z = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      // A wave without pages has m = -inf; its sum is 0.
      const float e = sh_l[w][g] == 0.f ? 0.f : exp2_hw(sh_m[w][g] - M);
      a = fmaf(e, sh_o[w][g][d], a);
      z = fmaf(e, sh_l[w][g], z);
    }
    float out = z == 0.f ? 0.f : a / z;
    float L = z == 0.f ? -INFINITY : M - kShift + log2_hw(z);   // in units of log 2
    if (sh_bad) out = L = NAN;
    if (ch.splits == 1) {
      const size_t row = (size_t)ch.b * H + h0 + g;
      const uint32_t bits = pack2<BF16>(out, 0.f);
      o[row * D + d] = (uint16_t)bits;
      if (lse != nullptr && d == 0) lse[row] = L * kLn2;
    } else {
      const size_t row = (size_t)(ch.partial + ch.split) * H + h0 + g;
      part_o[row * D + d] = out;
      if (d == 0) part_l[row] = L;
    }
  }
}

// Joins the chunks of cut sequence blockIdx.x: a workgroup per row (sequence,
// head), D / 4 threads for four values each, the chunks dealt out over
// kThreads / (D / 4) groups of them.
template <int D, bool BF16>
__global__ void __launch_bounds__(kThreads)
fa_decode_mx_join_kernel(const float* __restrict__ part_o, const float* __restrict__ part_l,
                         const int32_t* __restrict__ plan, uint16_t* __restrict__ o,
                         float* __restrict__ lse, int H) {
  constexpr int PER = D / 4, GROUPS = kThreads / PER;
  __shared__ float sh_m[kWaves], sh_z[GROUPS];
  __shared__ __attribute__((aligned(16))) float sh_o[GROUPS][D];
  if ((int)blockIdx.x >= plan[0]) return;
  const int b = plan[1 + 2 * blockIdx.x], word = plan[2 + 2 * blockIdx.x];
  const int first = word & 0xffff, n = word >> 16;
  const int h = blockIdx.y, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const float* pl = part_l + (size_t)first * H + h;
  const float* po = part_o + ((size_t)first * H + h) * D;

  float M = -INFINITY;
  bool nan = false;
  for (int i = tid; i < n; i += kThreads) {
    const float x = pl[(size_t)i * H];
    nan |= x != x;
    M = fmaxf(M, x);
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) M = fmaxf(M, __shfl_xor(M, d));
  if (lane == 0) sh_m[wave] = M;
  nan = __syncthreads_or(nan);
#pragma unroll
  for (int w = 0; w < kWaves; ++w) M = fmaxf(M, sh_m[w]);

  const int g = tid / PER, d = 4 * (tid % PER);
  f32x4 a = f32x4{};
  float z = 0.f;
  for (int i = g; i < n; i += GROUPS) {   // a chunk of a cut sequence has tokens: its L is finite or NaN
    const float e = exp2_hw(pl[(size_t)i * H] - M);
    const f32x4 x = *reinterpret_cast<const f32x4*>(po + (size_t)i * H * D + d);
    z += e;
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] = fmaf(e, x[j], a[j]);
  }
  *reinterpret_cast<f32x4*>(&sh_o[g][d]) = a;
  if (d == 0) sh_z[g] = z;
  __syncthreads();
  if (g != 0) return;
  a = f32x4{};
  z = 0.f;
#pragma unroll
  for (int i = 0; i < GROUPS; ++i) {
    const f32x4 x = *reinterpret_cast<const f32x4*>(&sh_o[i][d]);
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] += x[j];
    z += sh_z[i];
  }
  const size_t row = (size_t)b * H + h;
  const float inv = nan ? NAN : 1.f / z;
  *reinterpret_cast<u32x2*>(o + row * D + d) =
      u32x2{pack2<BF16>(a[0] * inv, a[1] * inv), pack2<BF16>(a[2] * inv, a[3] * inv)};
  if (lse != nullptr && d == 0) lse[row] = nan ? NAN : (M + log2_hw(z)) * kLn2;
}

template <int D, int KB, int VB, bool BF16>
static int decode(const void* q, const void* k_pool, const void* v_pool, const int32_t* page_table,
                  const int32_t* ctx_lens, int64_t B, int64_t H, int64_t Hkv, int64_t max_pages,
                  int64_t num_pages, float* workspace, void* o, float* lse, hipStream_t s) {
  const float c = (float)(1.0 / sqrt((double)D)) * kLog2e;
  const int64_t target = target_chunks(H, Hkv);
  // No sequence of up to kMinChunk pages is cut.
  const bool one = max_pages <= kMinChunk;
  const int64_t rows = partial_chunks(B, H, Hkv) * H;
  float* part_o = workspace;
  float* part_l = workspace + rows * D;
  int32_t* plan = one ? nullptr : reinterpret_cast<int32_t*>(part_l + rows);
  const dim3 grid((unsigned)(one ? B : target + B), (unsigned)head_groups(H, Hkv));
  hipLaunchKernelGGL((fa_decode_mx_kernel<D, KB, VB, BF16>), grid, dim3(kThreads), 0, s,
                     (const uint16_t*)q, (const char*)k_pool, (const char*)v_pool, page_table,
                     ctx_lens, part_o, part_l, plan, (uint16_t*)o, lse, (int)B, (int)H, (int)Hkv,
                     (int)max_pages, (int)num_pages, (int)target, c);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return -(int)e;
  if (one) return FA_OK;
  const dim3 rest((unsigned)(B < target ? B : target), (unsigned)H);
  hipLaunchKernelGGL((fa_decode_mx_join_kernel<D, BF16>), rest, dim3(kThreads), 0, s, part_o, part_l,
                     plan, (uint16_t*)o, lse, (int)H);
  e = hipGetLastError();
  return e == hipSuccess ? FA_OK : -(int)e;
}

}  // namespace mx
}  // namespace fa

extern "C" int64_t fa_decode_mx_workspace_floats(int64_t B, int64_t H, int64_t H_kv, int64_t D) {
  if (B <= 0 || H <= 0 || H_kv <= 0 || H % H_kv != 0 || D <= 0) return 0;
  const int64_t cut = fa::mx::target_chunks(H, H_kv);   // sequences that are cut, at most
  return fa::mx::partial_chunks(B, H, H_kv) * H * (D + 1) + 1 + 2 * (B < cut ? B : cut);
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
