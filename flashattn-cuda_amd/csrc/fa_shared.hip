// fa_shared.hip — paged decode of a batch that shares a prefix, for MI355X.
//
// No reference counterpart. Every sequence b attends to the keys of one shared
// prefix (one page list) and to its own pages:
//   O = softmax over both, L = logsumexp over both.
// The paged decode would read the prefix once per sequence. Here its keys are
// read once per KV head: the query rows of all sequences and of all heads that
// share a KV head, B * H / H_kv of them, form one product with them, as in a
// forward pass without a mask. Few rows (kFewRows) go through the chunks of
// fa_stream.hpp instead, as the own pages do, and in their launch. One launch joins
// the partials of both by their maxima and sums.
#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include "fa_mi355x.h"
#include "fa_stream.hpp"
#include "fa_tile.hpp"

namespace fa {
namespace shared {

using namespace stream;

// The cuts are made for the 256 CUs of a whole MI355X, whatever the device has: the
// workspace follows from the sizes alone. A partition of fewer CUs gets the same results by
// cuts that are not its own.
constexpr int kCus = 256, kMostUnits = 192;   // units: of the prefix pass in tiles

constexpr int kTile = 64;     // keys of a tile: 4 pages
constexpr int kStages = 4;    // tiles in LDS, three of them in flight
constexpr float kSlack = 8.f;   // of weights' exponents; see its use
// bf16's weights are 2^-kShift of those of the reference, up to 1: its V reach 2^127, which a
// weight above 1 would take out of range, while fp16's have no bits to lose at the lower end.
template <bool BF16>
constexpr float kShift = BF16 ? kSlack : 0.f;
constexpr float kFar = 4096.f;  // references, in units of log 2, from which on differences are scaled
constexpr int kKeyGroups = 2; // waves side by side over the keys of a tile
constexpr int kRowGroups = 4, kTileRows = 32 * kRowGroups;   // and over the query rows of a unit
constexpr int kTileWaves = kKeyGroups * kRowGroups;

// LDS of a workgroup that runs either a run of tiles or two chunks.
template <int D>
struct TileShared {
  static constexpr int kPage = kTokens * D * 2;
  static constexpr int kStage = 2 * (kTile / kTokens) * kPage;   // K, then V
  __attribute__((aligned(1024))) char ring[kStages * kStage];
  float m[kTileWaves][64], l[kTileWaves][64], over[kTileWaves][64];
  int bad;
};

// Prefix pass, unit g of all: (KV head, one of S runs of tiles, kTileRows query rows) by
// kRowGroups x 2 waves, wave (rm, kg) with rows 32 rm .. + 31 and the tile's keys 32
// kg .. + 31; rm the slow one, so that of a few rows every SIMD has some. Tiles are
// copied global -> LDS (buffer_load ... lds), the rows past the prefix as zeros (the
// copy's range ends there), and wait in a ring of kStages. Scores and products are
// those of the forward: S^T = K Q^T with Q in registers, O^T += V^T P^T with P^T
// straight from the accumulators (fa_tile.hpp), P rounded to the operands' type beside
// an unrounded sum, as the forward rounds it. O is then 1.35 times as far from 64 bits as
// its own rounding puts it; the chunks' second term would cost bf16 a second product and 40
// vector instructions a tile: 28.8 -> 34.5 us for 32 sequences of 50 to 1500 tokens under
// 7999, 68.4 -> 86.7 for 64 of 20 to 1000 under 32768 (H32 over 8, D = 128).
//
// Bound, with 128 rows a KV head, by memory: 256 units at D = 128 take 1.55 us a tile,
// 5.4 TB/s. With more, the row blocks of a tile find it in their L2 and a tile takes 1.2
// us of a CU, 0.9 PFLOP/s over the chip, the forward's rate, and no part of it by itself:
// 1.04 without the copies, 1.16 with half of the reads from LDS, 1.24 without the
// exponentials. Key groups that take turns at products and exponentials, or V in blocks
// of 32 columns, change it by 2 % at most. Beside the tiles a unit costs about 8 us, and
// 16.8 MB of partials 7 us at the end.
template <int D, bool BF16>
__device__ __forceinline__ void
tile_unit(TileShared<D>& sh, const int unit, const f16* __restrict__ q, const f16* __restrict__ kpool,
          const f16* __restrict__ vpool, const int32_t* __restrict__ prefix_table, int P, bool bad,
          float* __restrict__ part_o, float2* __restrict__ part_ml, int rows, int H, int Hkv, int num_pages,
          int S, int most, int row_blocks, int nxcd, float c) {
  constexpr int WM = kRowGroups, NW = kTileWaves;
  constexpr int PAGE = TileShared<D>::kPage, STAGE = TileShared<D>::kStage;
  constexpr int CPR = D / 8;
  constexpr int NC = PAGE / 1024;            // 1 KiB copies of a page
  constexpr int PAGES = kTile / kTokens;
  constexpr int NU = 2 * PAGES / NW;         // pages, of K or V, a wave copies of a tile
  constexpr int DB = D / 32;
  static_assert(NW * DB * 8 * 64 * 4 <= kStages * STAGE, "merge area within the ring");

  // Row blocks that read the same tiles are neighbours on one XCD.
  const int g = xcd_remap(unit, Hkv * S * row_blocks, nxcd);
  const int rb = g % row_blocks, s = (g / row_blocks) % S, hk = g / row_blocks / S;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rm = wave / kKeyGroups, kg = wave % kKeyGroups;
  const int G = H / Hkv;

  if (tid == 0) sh.bad = 0;
  __syncthreads();
  const int pages = (P + kTokens - 1) / kTokens;
  const int tiles = (pages + PAGES - 1) / PAGES;
  const int t0 = (int)((int64_t)tiles * s / S), t1 = (int)((int64_t)tiles * (s + 1) / S);

  // Query row of this lane: row r is head r % G of the group, sequence r / G.
  const int row = (rb * WM + rm) * 32 + (lane & 31);
  const bool live = row < rows;
  const bool some = (rb * WM + rm) * 32 < rows;   // of the wave's rows; without, it only copies
  const int64_t qrow = live ? (int64_t)(row / G) * H + hk * G + row % G : 0;
  f16x8 qf[D / 16];
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) {
    qf[kk] = f16x8{};
    if (live) qf[kk] = *reinterpret_cast<const f16x8*>(q + qrow * D + 16 * kk + 8 * (lane >> 5));
  }

  // Copies: lane l of copy i fills LDS chunk 64 i + l of a page with the chunk
  // that the swizzle puts there (t_swz repeats every 16 rows).
  uint32_t coff[NC];
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int L = 64 * i + lane, t = L / CPR;
    coff[i] = (uint32_t)((t * CPR + ((L % CPR) ^ t_swz<D>(t))) * 16);
  }
  const uint32_t lds0 = lds_addr(sh.ring);
  // Page ids of the wave's pages, 64 tiles at a time, read with readlane.
  int pidv[NU];
  auto issue = [&](int k) {   // tile t0 + k
#pragma unroll
    for (int x = 0; x < NU; ++x) {
      const int unit = wave + NW * x;   // K and V of page unit / 2
      if ((k & 63) == 0) {
        const int pi = (t0 + k + lane) * PAGES + unit / 2;
        pidv[x] = t0 + k + lane < t1 && pi < pages ? prefix_table[pi] : -1;
        // Used up here: after the branch the compiler would wait for the load on
        // either path, and with it, every tile, for all copies in flight.
        asm volatile("" : "+v"(pidv[x]));
      }
      const int pi = (t0 + k) * PAGES + unit / 2;
      const int pid = __builtin_amdgcn_readlane(pidv[x], k & 63);
      const bool in = t0 + k < t1 && pi < pages;
      const bool ok = in && pid >= 0 && pid < num_pages;
      bad |= in && !ok;
      const size_t off = ok ? ((size_t)pid * Hkv + hk) * (size_t)(kTokens * D) : 0;
      const auto r = make_rsrc_s(((unit & 1) ? vpool : kpool) + off, ok ? min(kTokens, P - pi * kTokens) * D * 2 : 0);
      const uint32_t dst = lds0 + (k % kStages) * STAGE + (unit & 1) * (PAGES * PAGE) + unit / 2 * PAGE;
#pragma unroll
      for (int i = 0; i < NC; ++i) dma16(r, dst + 1024 * i, coff[i]);
    }
  };

  // Reference of the weights, as K Q^T gives it (-inf: no score yet), and their sum. A weight is
  // 2^(s c - mu), mu the scaled reference and kShift, rounded: all of a row are off by the
  // same 2^rest, which the sums are freed of. Where a row of the wave has a scaled reference
  // of kFar or more, references are taken off the scores first, which holds however large
  // they are (a mu of 2^27 is rounded by 2^3, of 2^31 by 2^7, past all types); always done, a
  // tile pass of 28.8 us takes 29.4, and one of 46.3 at D = 64 49.3.
  float m = -INFINITY, l = 0.f, mu = 0.f;
  bool far = false;   // the same in the whole wave
  const auto rest = [&](float m, float mu, bool far) {
    return m == -INFINITY ? 0.f : (far ? -kShift<BF16> : fmaf(m, c, -mu));
  };
  f32x16 o[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) o[db] = f32x16{};
  f16x8 kf[D / 16];
  // K's operands of the wave's 32 keys of tile t0 + k.
  const auto load_k = [&](int k) {
    const uint32_t kb = row_base<D>(lds0 + (k % kStages) * STAGE + kg * (32 * 2 * D), lane);
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) kf[kk] = load_row_frag<D>(kb, 0, kk);
  };
  const auto scores = [&]() {
    f32x16 x = f32x16{};
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) x = mma32<BF16>(kf[kk], qf[kk], x);
    return x;
  };
  // The wave's keys of tile t0 + k, whose scores are sc; NEXT: and the scores of its
  // keys of the next tile, whose products run under this one's exponentials. LDS reads
  // go out a phase before their products: one after the other each product waited
  // for its own.
  const auto step = [&](int k, f32x16& sc, auto next) {
    if constexpr (decltype(next)::value) load_k(k + 1);
    const int key0 = (t0 + k) * kTile + 32 * kg;
    if (key0 + 32 > P) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (key0 + st_key(0, r, lane) >= P) sc[r] = -INFINITY;
    }
    float mx = sc[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) mx = fmaxf(mx, sc[r]);
    mx = max_xor32(mx);
    // The reference follows the maximum only where that is kSlack above it: of 32 rows
    // one has a new maximum in most steps (64 sequences under 32768: a call 83 us without,
    // 75 with). fp16's weights reach 2^kSlack, bf16's 1.
    if (__any((mx - m) * c > kSlack)) {   // of -inf and -inf a NaN: no
      const float m_new = fmaxf(m, mx);
      const bool far_new = __any(m_new != -INFINITY && fabsf(m_new) * c >= kFar);
      const float mu_new = far_new || m_new == -INFINITY ? kShift<BF16> : fmaf(m_new, c, kShift<BF16>);
      const float rests = rest(m_new, mu_new, far_new) - rest(m, mu, far);
      const float alpha = m == -INFINITY ? 1.f : exp2_hw((m - m_new) * c + rests);
      l *= alpha;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[db][r] *= alpha;
      m = m_new;
      mu = mu_new;
      far = far_new;
    }
    if (far) {            // wave-uniform
      asm volatile("");   // a branch: not selects in every step
      const float by = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[r] -= by;
    }
    __builtin_amdgcn_sched_barrier(0);
    const uint32_t vb = col_base<D>(lds0 + (k % kStages) * STAGE + PAGES * PAGE + kg * (32 * 2 * D), lane);
    f16x8 vf[2][DB];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int db = 0; db < DB; ++db) vf[j][db] = load_col_frag<D>(vb, 0, j, db);
    __builtin_amdgcn_sched_barrier(0);
    f32x16 sn;
    if constexpr (decltype(next)::value) sn = scores();
#pragma unroll
    for (int r = 0; r < 16; ++r) sc[r] = exp2_hw(fmaf(sc[r], c, -mu));   // of -inf, with no reference too: 0
    f16x8 p[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) p[j] = pack_px<BF16>(sc, j);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db] = mma32<BF16>(vf[j][db], p[j], o[db]);
    float ps[4] = {sc[0], sc[1], sc[2], sc[3]};
#pragma unroll
    for (int r = 4; r < 16; ++r) ps[r & 3] += sc[r];
    l += (ps[0] + ps[1]) + (ps[2] + ps[3]);
    if constexpr (decltype(next)::value) sc = sn;
  };

  const int n = t1 - t0;
  if (n > 0) {
#pragma unroll
    for (int k = 0; k < kStages - 1; ++k) issue(k);
    wait_vmcnt<(kStages - 2) * NU * NC>();   // this wave's copies of the first tile have landed
    __syncthreads();                         // and everyone's
    f32x16 sc;
    if (some) {
      load_k(0);
      sc = scores();
    }
    for (int k = 0; k < n - 1; ++k) {
      wait_vmcnt<(kStages - 3) * NU * NC>();   // tile k + 1
      __syncthreads();                         // everyone's, and tile k - 1 is used up
      issue(k + kStages - 1);
      if (some) step(k, sc, std::true_type{});
    }
    if (some) step(n - 1, sc, std::false_type{});
  }
  l = sum_xor32(l);
  const float over = exp2_hw(-rest(m, mu, far));   // of the weights that reach the sum and the products

  // Merge the two key groups through LDS, each for half of the columns: a wave
  // leaves the other's half register by register, lanes of the two hold the same
  // elements.
  wait_vmem();
  if (bad) sh.bad = 1;
  __syncthreads();
  constexpr int HB = DB / 2, XCH = HB * 16 * 64;   // words a wave leaves
  float* const area = reinterpret_cast<float*>(sh.ring);
  {
    float* to = area + (wave)*XCH;
#pragma unroll
    for (int h = 0; h < HB; ++h)
#pragma unroll
      for (int r = 0; r < 16; ++r) to[(h * 16 + r) * 64 + lane] = kg == 0 ? o[HB + h][r] : o[h][r];
    sh.m[wave][lane] = m;
    sh.l[wave][lane] = l;
    sh.over[wave][lane] = over;
  }
  __syncthreads();
  const int other = wave ^ 1;   // the same rows, the other keys
  const float m1 = sh.m[other][lane], M = fmaxf(m, m1);
  const float e0 = m == -INFINITY ? 0.f : exp2_hw((m - M) * c) * over;   // over: 2^(kSlack + 1/2) at most
  const float e1 = m1 == -INFINITY ? 0.f : exp2_hw((m1 - M) * c) * sh.over[other][lane];
  const float z = e0 * l + e1 * sh.l[other][lane];
  const bool nan = sh.bad || z != z;
  const float inv = nan ? NAN : (z > 0.f ? 1.f / z : 0.f);
  const float f0 = e0 * inv, f1 = e1 * inv;
  float v[HB][16];
  const float* theirs = area + other * XCH;
#pragma unroll
  for (int h = 0; h < HB; ++h)
#pragma unroll
    for (int r = 0; r < 16; ++r)
      v[h][r] = f0 * (kg == 0 ? o[h][r] : o[HB + h][r]) + f1 * theirs[(h * 16 + r) * 64 + lane];
  __syncthreads();
  // Through LDS once more, rows of the wave's half in a row: 32 rows of D / 2 (and 4
  // words, for the banks), stored a row's 2 D bytes at a time.
  constexpr int ROW = D / 2 + 4;
  static_assert(NW * 32 * ROW * 4 <= kStages * STAGE, "rows within the ring");
  float* const mine = area + wave * (32 * ROW);
#pragma unroll
  for (int h = 0; h < HB; ++h)
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4)
      *reinterpret_cast<f32x4*>(mine + (lane & 31) * ROW + 32 * h + 8 * r4 + 4 * (lane >> 5)) =
          f32x4{v[h][4 * r4], v[h][4 * r4 + 1], v[h][4 * r4 + 2], v[h][4 * r4 + 3]};
  if (kg == 0 && lane < 32 && live) part_ml[(size_t)qrow * most + s] = make_float2(M, nan ? NAN : z);
  constexpr int PER = D / 8;   // lanes of a row's half
#pragma unroll 4
  for (int i = 0; i < 32; i += 64 / PER) {
    const int x = i + lane / PER, r = (rb * WM + rm) * 32 + x, d = 4 * (lane % PER);
    if (r >= rows) continue;
    const size_t at = ((size_t)(r / G) * H + hk * G + r % G) * most + s;
    *reinterpret_cast<f32x4*>(part_o + at * D + kg * (D / 2) + d) = *reinterpret_cast<const f32x4*>(mine + x * ROW + d);
  }
}

// Splits of a short list of prefix pages in the chunk pass: SP at most.
__device__ __forceinline__ int prefix_splits(int P, int max_pages, int SP) {
  const int n = pages_of(P, max_pages) / kMinChunk;
  return n < 1 ? 1 : min(n, SP);
}

// Workgroups [0, pre_blocks): chunks of the prefix for 16 of the `rows` query rows
// of a KV head; partial number split * B * H + row. The others: chunks of the own
// pages, partial number chunk * H + h.
template <int D, bool BF16, bool NT>
__global__ void __launch_bounds__(stream::kThreads)
fa_shared_chunk_kernel(const uint16_t* __restrict__ q, const char* __restrict__ k_pool,
                       const char* __restrict__ v_pool, const int32_t* __restrict__ prefix_table,
                       const int32_t* __restrict__ prefix_len, const int32_t* __restrict__ page_table,
                       const int32_t* __restrict__ ctx_lens, const int4* __restrict__ table,
                       float* __restrict__ pre_o, float2* __restrict__ pre_ml, float* __restrict__ own_o,
                       float2* __restrict__ own_ml, int2* __restrict__ first, int B, int H, int Hkv,
                       int group, int ngrp, int rows, int pre_blocks, int pre_grp, int SP,
                       int prefix_pages, int max_pages, int num_pages, Plan plan, float c) {
  __shared__ Shared<D> sh;
  const int col = threadIdx.x & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if ((int)blockIdx.x < pre_blocks) {
    const Place at = place_of(blockIdx.x, Hkv * pre_grp);
    const int P = prefix_len[0], pages = pages_of(P, prefix_pages);
    const int n = prefix_splits(P, prefix_pages, SP);
    if (at.number >= n) return;
    const int hk = at.hg / pre_grp, r = 16 * (at.hg - hk * pre_grp) + col;
    const bool live = r < rows;
    const int64_t row = live ? (int64_t)(r / group) * H + hk * group + r % group : 0;
    const int p0 = (int)((int64_t)pages * at.number / n), p1 = (int)((int64_t)pages * (at.number + 1) / n);
    const PartOut<D> out{pre_o, pre_ml, (int64_t)at.number * B * H + row};
    chunk_body<D, BF16, NT>(sh, wave, q, k_pool, v_pool, Pages{prefix_table, P}, p0, p1,
                            P < 0 || (P > 0 && pages == 0), live, row * D, hk, Hkv, num_pages, c, NoScores{},
                            out, out);
    return;
  }
  const Place at = place_of((int)blockIdx.x - pre_blocks, Hkv * ngrp);
  const Run r = run_of(ctx_lens, table, B, max_pages, plan, at.number);
  if (r.b < 0) return;
  if (at.hg == 0 && r.split == 0 && threadIdx.x == 0) first[r.b] = make_int2(at.number, r.splits);
  const int hk = at.hg / ngrp, sub = at.hg - hk * ngrp;
  const int h = hk * group + 16 * sub + col;
  const bool live = 16 * sub + col < group;
  const PartOut<D> out{own_o, own_ml, (int64_t)at.number * H + h};
  chunk_body<D, BF16, NT>(sh, wave, q, k_pool, v_pool, Pages{page_table + (size_t)r.b * max_pages, r.ctx},
                          r.p0, r.p1, r.bad, live, ((int64_t)r.b * H + h) * D, hk, Hkv, num_pages, c,
                          NoScores{}, out, out);
}

// Splits of the prefix in the launch of tiles, from the lengths that only the device
// knows: as many units as make the prefix's share of the CUs that of its work, in us of a
// CU, so that the own pages are read beside the tiles and neither is left over; of
// kUnitTiles tiles at least, and kMostUnits at most (more, and the own pages of a short
// batch wait for a CU: 16 sequences of 50 to 200 under 8000 20 -> 23.5 us). `per` units a
// split, `pages` own pages. Against 160 units for any lengths, us a call, H32 over 8, D =
// 128: 32 sequences of 50 to 1500 tokens under 7999 38.6 -> 33.7, 128 of 20 to 500 under
// 32768 122 -> 115, 64 of 500 to 2000 107 -> 105, of 20 to 1000 75 and 75, 36 of 30 to 120
// under 2500 19.4 -> 22.2; 18 such sets in the mean 2 % less. In launches of their own
// the first took 17 + 20.4 and the fourth 48.5 + 24.7. kUnitTime 0.5, 3, 8 and 13: the mean
// 39.9, 39.1, 40.0, 39.8 (a unit's own time is 8); kUnitTiles 1, 2, 3, 4 and 6, 8 sets of
// short prefixes: 16.8, 16.6, 16.6, 17.0, 18.0.
template <int D>
__device__ __forceinline__ int tile_splits(int tiles, int per, int pages, int Hkv, int most) {
  constexpr float kTileTime = 1.15f * D / 128, kUnitTime = 3.f, kPageTime = 0.4f * D / 128;
  constexpr int kUnitTiles = 3;
  const float t = kTileTime * tiles * per, own = kPageTime * pages * Hkv;
  const float x = t + own - kCus * kUnitTime;   // kUnitTime u^2 + x u - kCus t = 0
  const float u = (__builtin_sqrtf(x * x + 4 * kUnitTime * kCus * t) - x) / (2 * kUnitTime);
  return max(min(min((int)(u / per + 0.5f), tiles / kUnitTiles), most), 1);
}

// Workgroups [0, units): runs of tiles of the prefix, at most SP a KV head and row block;
// those past the planned ones end at once. The others: two chunks of the
// own pages each, of neighbouring head groups (see place_of: here an XCD's chunks and
// head groups follow one another over its workgroups' halves). The own pages are bound
// by memory and the tiles by their products, so one launch has both under way.
template <int D, bool BF16, bool NT>
__global__ void __launch_bounds__(64 * kTileWaves)
fa_shared_tile_kernel(const uint16_t* __restrict__ q, const char* __restrict__ k_pool,
                      const char* __restrict__ v_pool, const int32_t* __restrict__ prefix_table,
                      const int32_t* __restrict__ prefix_len, const int32_t* __restrict__ page_table,
                      const int32_t* __restrict__ ctx_lens, const int4* __restrict__ table,
                      float* __restrict__ pre_o, float2* __restrict__ pre_ml, float* __restrict__ own_o,
                      float2* __restrict__ own_ml, int2* __restrict__ first, int B, int H, int Hkv,
                      int group, int ngrp, int rows, int units, int row_blocks, int SP,
                      int* __restrict__ splits, int prefix_pages, int max_pages, int num_pages, Plan plan,
                      int nxcd, float c) {
  constexpr int kHalves = kTileWaves / kWaves;
  __shared__ union Lds {
    TileShared<D> tile;
    Shared<D> chunk[kHalves];
    __device__ Lds() {}
  } sh;
  if ((int)blockIdx.x < units) {
    int P = prefix_len[0];
    const bool bad = P < 0 || P > prefix_pages * kTokens;
    if (bad) P = 0;
    const int S = tile_splits<D>((P + kTile - 1) / kTile, Hkv * row_blocks,
                                 total_pages(ctx_lens, table, B, max_pages), Hkv, SP);
    if (blockIdx.x == 0 && threadIdx.x == 0) *splits = S;
    if ((int)blockIdx.x >= Hkv * S * row_blocks) return;
    tile_unit<D, BF16>(sh.tile, blockIdx.x, (const f16*)q, (const f16*)k_pool, (const f16*)v_pool,
                       prefix_table, P, bad, pre_o, pre_ml, rows, H, Hkv, num_pages, S, SP, row_blocks, nxcd,
                       c);
    return;
  }
  const int w = (int)blockIdx.x - units, col = threadIdx.x & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = wave / kWaves;
  const int seq = kHalves * (w / kXcds) + half, groups = Hkv * ngrp;
  const int number = seq / groups * kXcds + w % kXcds, hg = seq % groups;
  const Run r = run_of(ctx_lens, table, B, max_pages, plan, number);
  if (r.b >= 0 && hg == 0 && r.split == 0 && threadIdx.x % (64 * kWaves) == 0)
    first[r.b] = make_int2(number, r.splits);
  const int hk = hg / ngrp, sub = hg - hk * ngrp;
  const int h = hk * group + 16 * sub + col;
  const bool live = r.b >= 0 && 16 * sub + col < group;
  const PartOut<D> out{own_o, own_ml, (int64_t)number * H + h};
  chunk_body<D, BF16, NT>(sh.chunk[half], wave % kWaves, q, k_pool, v_pool,
                          Pages{page_table + (size_t)max(r.b, 0) * max_pages, r.ctx}, r.p0, r.p1, r.bad, live,
                          ((int64_t)r.b * H + h) * D, hk, Hkv, num_pages, c, NoScores{}, out, out);
}

// Short calls in one launch, a workgroup of kOneWaves waves for a sequence and 16 heads of
// a KV head: it walks the prefix's pages and then its own.
constexpr int kOneWaves = 8;

template <int D, bool BF16>
__global__ void __launch_bounds__(64 * kOneWaves)
fa_shared_one_kernel(const uint16_t* __restrict__ q, const char* __restrict__ k_pool,
                     const char* __restrict__ v_pool, const int32_t* __restrict__ prefix_table,
                     const int32_t* __restrict__ prefix_len, const int32_t* __restrict__ page_table,
                     const int32_t* __restrict__ ctx_lens, uint16_t* __restrict__ o,
                     float* __restrict__ lse, int H, int Hkv, int group, int ngrp, int prefix_pages,
                     int max_pages, int num_pages, float c) {
  __shared__ Shared<D, kOneWaves> sh;
  const int hk = (int)blockIdx.x / ngrp, sub = (int)blockIdx.x - hk * ngrp, b = blockIdx.y;
  const int col = threadIdx.x & 15, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int P = __builtin_amdgcn_readfirstlane(prefix_len[0]);
  const int ctx = __builtin_amdgcn_readfirstlane(ctx_lens[b]);
  const int np = pages_of(P, prefix_pages), own = pages_of(ctx, max_pages);
  const bool bad = P < 0 || (P > 0 && np == 0) || ctx < 0 || (ctx > 0 && own == 0);
  const int64_t row = (int64_t)b * H + hk * group + 16 * sub + col;
  const RowOut<D, BF16> out{o, lse, row, c};
  chunk_body<D, BF16, false>(sh, wave, q, k_pool, v_pool,
                             JoinedPages{prefix_table, page_table + (size_t)b * max_pages, np, P, ctx}, 0,
                             np + own, bad, 16 * sub + col < group, row * D, hk, Hkv, num_pages, c,
                             NoScores{}, out, out);
}

// O and L of row blockIdx.x out of the partials of the prefix (of few rows, as many as
// the prefix's length gives, else *splits) and of the own pages.
template <int D, bool BF16>
__global__ void __launch_bounds__(kJoinThreads)
fa_shared_join_kernel(const float* __restrict__ pre_o, const float2* __restrict__ pre_ml,
                      const float* __restrict__ own_o, const float2* __restrict__ own_ml,
                      const int2* __restrict__ first, const int* __restrict__ splits,
                      const int32_t* __restrict__ prefix_len, uint16_t* __restrict__ o,
                      float* __restrict__ lse, int H, int rows, int SP, int few, int prefix_pages, float c) {
  __shared__ JoinShared<D> sh;
  const int row = blockIdx.x, b = row / H;
  const int2 f = first[b];
  const int n = few ? prefix_splits(prefix_len[0], prefix_pages, SP) : *splits;
  const Parts pre = few ? Parts{pre_o, pre_ml, row, rows, n} : Parts{pre_o, pre_ml, (int64_t)row * SP, 1, n};
  join_row<D, BF16>(sh, pre, Parts{own_o, own_ml, (int64_t)f.x * H + (row - b * H), H, f.y}, c,
                    o + (int64_t)row * D, lse + row);
}

// A call is one launch, a workgroup for a sequence and 16 heads, where little would be
// gained by cutting it: up to a workgroup a CU and kOneWork dims of the pages of both
// tables (36 pages of D = 128), or two and half of it. A call by itself, us, in one launch
// and cut: D = 64, 16 pages of 32 workgroups 4.8 and 8.3, 56 8.0 and 8.3, 72 9.4 and 8.3, of 128
// 9.2 and 14.7, of 256 10.0 and 17.4, 36 of 512 11.6 and 18.0; D = 128, 36 pages of 32 8.8 and
// 8.8, of 256 9.9 and 18.7, 18 of 512 12.4 and 18.7. One bound whatever the number of
// workgroups: few of them lose up to 1.1 us past 56 pages of D = 64.
constexpr int kOneWork = 36 * 128;
static bool in_one(int64_t blocks, int64_t pages, int64_t D) {
  return blocks <= 2 * kCus && pages * D * (blocks <= kCus ? 1 : 2) <= kOneWork;
}

// Query rows of a KV head up to which the prefix goes through the chunk pass, one or two
// workgroups of 16 rows for a chunk and kCus in all. A call, us, through chunks and tiles,
// H32 over 8, D = 128, 50 to 200 tokens under 8000 and 32000: 16 rows 15.1 28.4 and 20.5
// 36.7, 32 rows 15.7 35.6 and 21.2 37.8, 64 rows 21.1 59.1 and 19.5 39.8. The chunks of 32
// rows under 32000, for 256, 512 and 1024 workgroups: 35.6 38.9 42.5.
constexpr int kFewRows = 32;

// How a call is cut: the prefix pass and its splits, the own pages' chunks, and the
// workspace in floats.
struct Cut {
  bool one, few;
  int row_blocks, sp;
  Plan plan;   // of the own pages' chunks
  int64_t rows, own, pre_ml, own_o, own_ml, first, table, floats;
};

static Cut cut_of(int64_t B, int64_t H, int64_t Hkv, int64_t D, int64_t prefix_pages, int64_t max_pages) {
  Cut p;
  p.one = in_one(B * head_groups(H, Hkv), prefix_pages + max_pages, D);
  p.rows = B * (H / Hkv);
  p.few = p.rows <= kFewRows;
  const int64_t block = p.few ? 16 : kTileRows, part = p.few ? kMinChunk : kTile / kTokens;
  p.row_blocks = (int)((p.rows + block - 1) / block);
  int64_t sp = (p.few ? kCus : kMostUnits) / (Hkv * p.row_blocks);
  const int64_t most = (prefix_pages + part - 1) / part;
  sp = sp > most ? most : sp;
  p.sp = (int)(sp < 1 ? 1 : sp);
  p.plan = plan_of(head_groups(H, Hkv));
  p.own = most_chunks(B, max_pages, p.plan);
  p.own_o = B * H * p.sp * D;
  p.pre_ml = p.own_o + p.own * H * D;
  p.own_ml = p.pre_ml + 2 * B * H * p.sp;
  p.table = (p.own_ml + 2 * p.own * H + 3) / 4 * 4;   // entries of 16 bytes
  p.first = p.table + (B > kWavePlan ? 4 * (1 + p.own) : 0);
  p.floats = p.first + 2 * B + 1;
  return p;
}

template <int D, bool BF16>
static int launch(const Cut& p, const void* q, const void* k_pool, const void* v_pool,
                  const int32_t* prefix_table, const int32_t* prefix_len, const int32_t* page_table,
                  const int32_t* ctx_lens, int64_t B, int64_t H, int64_t Hkv, int64_t prefix_pages,
                  int64_t max_pages, int64_t num_pages, float* ws, void* o, float* lse, hipStream_t s) {
  const float c = (float)(1.0 / sqrt((double)D)) * kLog2e;
  const int64_t groups = head_groups(H, Hkv);
  if (p.one) {
    hipLaunchKernelGGL((fa_shared_one_kernel<D, BF16>), dim3((unsigned)groups, (unsigned)B),
                       dim3(64 * kOneWaves), 0, s, (const uint16_t*)q, (const char*)k_pool,
                       (const char*)v_pool, prefix_table, prefix_len, page_table, ctx_lens, (uint16_t*)o,
                       lse, (int)H, (int)Hkv, (int)(H / Hkv), (int)(groups / Hkv), (int)prefix_pages,
                       (int)max_pages, (int)num_pages, c);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? FA_OK : -(int)e;
  }
  const Plan plan = p.plan;
  float* own_o = ws + p.own_o;
  float2* pre_ml = (float2*)(ws + p.pre_ml);
  float2* own_ml = (float2*)(ws + p.own_ml);
  int2* first = (int2*)(ws + p.first);
  int* splits = (int*)(ws + p.first + 2 * B);
  int4* table = B > kWavePlan ? (int4*)(ws + p.table) : nullptr;
  if (table != nullptr)
    hipLaunchKernelGGL(fa_stream_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, ctx_lens, (int)B,
                       (int)max_pages, plan, table);
  const bool nt = pass_through(num_pages, Hkv, D);
  if (p.few) {
    const int64_t pre_blocks = chunk_blocks(p.sp, Hkv * p.row_blocks);
    const auto kernel = nt ? fa_shared_chunk_kernel<D, BF16, true> : fa_shared_chunk_kernel<D, BF16, false>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(pre_blocks + chunk_blocks(p.own, groups))),
                       dim3(stream::kThreads), 0, s, (const uint16_t*)q, (const char*)k_pool,
                       (const char*)v_pool, prefix_table, prefix_len, page_table, ctx_lens, table, ws,
                       pre_ml, own_o, own_ml, first, (int)B, (int)H, (int)Hkv, (int)(H / Hkv),
                       (int)(groups / Hkv), (int)p.rows, (int)pre_blocks, p.row_blocks, p.sp,
                       (int)prefix_pages, (int)max_pages, (int)num_pages, plan, c);
  } else {
    const int64_t units = Hkv * p.sp * p.row_blocks;
    const int64_t halves = kTileWaves / kWaves;
    const int64_t own = ((p.own + kXcds - 1) / kXcds * groups + halves - 1) / halves * kXcds;
    const auto kernel = nt ? fa_shared_tile_kernel<D, BF16, true> : fa_shared_tile_kernel<D, BF16, false>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(units + own)), dim3(64 * kTileWaves), 0, s,
                       (const uint16_t*)q, (const char*)k_pool, (const char*)v_pool, prefix_table,
                       prefix_len, page_table, ctx_lens, table, ws, pre_ml, own_o, own_ml, first, (int)B,
                       (int)H, (int)Hkv, (int)(H / Hkv), (int)(groups / Hkv), (int)p.rows, (int)units,
                       p.row_blocks, p.sp, splits, (int)prefix_pages, (int)max_pages, (int)num_pages,
                       plan, stream_topology(s).xcds, c);
  }
  hipLaunchKernelGGL((fa_shared_join_kernel<D, BF16>), dim3((unsigned)(B * H)), dim3(kJoinThreads), 0, s,
                     ws, pre_ml, own_o, own_ml, first, splits, prefix_len, (uint16_t*)o, lse, (int)H, (int)(B * H),
                     p.sp, (int)p.few, (int)prefix_pages, c);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? FA_OK : -(int)e;
}

}  // namespace shared
}  // namespace fa

extern "C" int64_t fa_decode_shared_workspace_floats(int64_t B, int64_t H, int64_t H_kv, int64_t D,
                                                     int64_t prefix_pages, int64_t max_pages) {
  // the sizes that fa_validate_decode_shared refuses
  constexpr int64_t kIndexes = (int64_t(1) << 31) - 1;
  if (B <= 0 || H <= 0 || H_kv <= 0 || H % H_kv != 0 || (D != 64 && D != 128) || prefix_pages <= 0 ||
      max_pages <= 0 || B > 65535 || H > 65535 || prefix_pages > (1 << 27) - 8 ||
      max_pages > kIndexes / 16 || B > kIndexes / max_pages)
    return 0;
  const fa::shared::Cut p = fa::shared::cut_of(B, H, H_kv, D, prefix_pages, max_pages);
  return p.one ? 0 : p.floats;
}

extern "C" int fa_decode_shared(const void* q, const void* k_pool, const void* v_pool,
                                const int32_t* prefix_table, const int32_t* prefix_len,
                                const int32_t* page_table, const int32_t* ctx_lens, int64_t B,
                                int64_t H, int64_t H_kv, int64_t D, int64_t page_size,
                                int64_t prefix_pages, int64_t max_pages, int64_t num_pages,
                                float* workspace, void* o, float* lse, int bf16, void* stream) {
  using namespace fa;
  using namespace fa::shared;
  const int st = fa_validate_decode_shared(q, k_pool, v_pool, prefix_table, prefix_len, page_table,
                                           ctx_lens, B, H, H_kv, D, page_size, prefix_pages,
                                           max_pages, num_pages, workspace, o, lse);
  if (st != FA_OK) return st;
  const Cut p = cut_of(B, H, H_kv, D, prefix_pages, max_pages);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const auto fn = D == 128 ? (bf16 ? launch<128, true> : launch<128, false>)
                           : (bf16 ? launch<64, true> : launch<64, false>);
  return fn(p, q, k_pool, v_pool, prefix_table, prefix_len, page_table, ctx_lens, B, H, H_kv,
            prefix_pages, max_pages, num_pages, workspace, o, lse, s);
}
