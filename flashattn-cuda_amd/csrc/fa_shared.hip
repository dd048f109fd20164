// fa_shared.hip — paged decode of a batch that shares a prefix, for MI355X.
//
// No reference counterpart. Every sequence b attends to the keys of one shared
// prefix (one page list) and to its own pages:
//   O = softmax over both, L = logsumexp over both.
// The paged decode would read the prefix once per sequence. Here its keys are
// read once per KV head: the query rows of all sequences and of all heads that
// share a KV head, B * H / H_kv of them, form one product with them, as in a
// forward pass without a mask. The own pages go through the split pass of the
// paged decode, and one launch joins the partials of both by their (maximum, sum).
#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include "fa_decode.hpp"
#include "fa_mi355x.h"
#include "fa_tile.hpp"

namespace fa {
namespace shared {

constexpr int kTile = 64;     // keys of a tile: 4 pages
constexpr int kStages = 4;    // tiles in LDS, three of them in flight
constexpr int kKeyGroups = 2; // waves side by side over the keys of a tile

// Prefix pass. One workgroup per (KV head, run of tiles, 32 WM query rows): WM x
// 2 waves, wave (rm, kg) with rows 32 rm .. + 31 and the tile's keys 32 kg .. +
// 31. Tiles are copied global -> LDS (buffer_load ... lds), the rows past the
// prefix as zeros (the copy's range ends there), and wait in a ring of kStages.
// Scores and products are those of the forward: S^T = K Q^T with Q in registers,
// O^T += V^T P^T with P^T straight from the accumulators (fa_tile.hpp), P rounded
// to the operands' type beside an unrounded sum, as the forward rounds it.
template <int D, bool BF16, int WM>
__global__ void __launch_bounds__(64 * WM * kKeyGroups)
fa_prefix_split_kernel(const f16* __restrict__ q, const f16* __restrict__ kpool,
                       const f16* __restrict__ vpool, const int32_t* __restrict__ prefix_table,
                       const int32_t* __restrict__ prefix_len, float* __restrict__ part_o,
                       float2* __restrict__ part_ml, int rows, int H, int Hkv, int max_pages,
                       int num_pages, int S, int row_blocks, int nxcd, float c) {
  constexpr int NW = WM * kKeyGroups;
  constexpr int PAGE = kPage * D * 2;
  constexpr int CPR = D / 8;
  constexpr int NC = PAGE / 1024;            // 1 KiB copies of a page
  constexpr int PAGES = kTile / kPage;
  constexpr int NU = 2 * PAGES / NW;         // pages, of K or V, a wave copies of a tile
  constexpr int STAGE = 2 * PAGES * PAGE;    // K, then V
  constexpr int DB = D / 32;
  static_assert(WM * DB * 16 * 64 * 4 <= kStages * STAGE, "merge area within the ring");
  __shared__ __attribute__((aligned(1024))) char smem[kStages * STAGE];
  __shared__ float sh_m[WM][64], sh_l[WM][64];
  __shared__ int sh_bad;

  // Row blocks that read the same tiles are neighbours on one XCD.
  const int g = xcd_remap(blockIdx.x, gridDim.x, nxcd);
  const int rb = g % row_blocks, s = (g / row_blocks) % S, hk = g / row_blocks / S;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rm = wave % WM, kg = wave / WM;
  const int G = H / Hkv;

  if (tid == 0) sh_bad = 0;
  __syncthreads();
  int P = prefix_len[0];
  bool bad = P < 0 || P > max_pages * kPage;
  if (bad) P = 0;
  const int pages = (P + kPage - 1) / kPage;
  const int tiles = (pages + PAGES - 1) / PAGES;
  const int t0 = (int)((int64_t)tiles * s / S), t1 = (int)((int64_t)tiles * (s + 1) / S);

  // Query row of this lane: row r is head r % G of the group, sequence r / G.
  const int row = (rb * WM + rm) * 32 + (lane & 31);
  const bool live = row < rows;
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
  const uint32_t lds0 = lds_addr(smem);
  // Page ids of the wave's pages, 64 tiles at a time, read with readlane.
  int pidv[NU];
  auto issue = [&](int k) {   // tile t0 + k
#pragma unroll
    for (int x = 0; x < NU; ++x) {
      const int unit = wave + NW * x;   // K and V of page unit / 2
      if ((k & 63) == 0) {
        const int pi = (t0 + k + lane) * PAGES + unit / 2;
        pidv[x] = t0 + k + lane < t1 && pi < pages ? prefix_table[pi] : -1;
      }
      const int pi = (t0 + k) * PAGES + unit / 2;
      const int pid = __builtin_amdgcn_readlane(pidv[x], k & 63);
      const bool in = t0 + k < t1 && pi < pages;
      const bool ok = in && pid >= 0 && pid < num_pages;
      bad |= in && !ok;
      const size_t off = ok ? ((size_t)pid * Hkv + hk) * (size_t)(kPage * D) : 0;
      const auto r = make_rsrc_s(((unit & 1) ? vpool : kpool) + off, ok ? min(kPage, P - pi * kPage) * D * 2 : 0);
      const uint32_t dst = lds0 + (k % kStages) * STAGE + (unit & 1) * (PAGES * PAGE) + unit / 2 * PAGE;
#pragma unroll
      for (int i = 0; i < NC; ++i) dma16(r, dst + 1024 * i, coff[i]);
    }
  };

  float m = -INFINITY, l = 0.f;
  f32x16 o[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) o[db] = f32x16{};

#pragma unroll
  for (int k = 0; k < kStages - 1; ++k) issue(k);
  for (int t = t0; t < t1; ++t) {
    const int k = t - t0;
    wait_vmcnt<(kStages - 2) * NU * NC>();   // this wave's copies of tile t have landed
    __syncthreads();                         // everyone's, and tile t - 1 is used up
    issue(k + kStages - 1);
    const int key0 = t * kTile + 32 * kg;
    if (key0 < P) {
      const uint32_t ks = lds0 + (k % kStages) * STAGE + kg * (32 * 2 * D);
      const uint32_t kb = row_base<D>(ks, lane), vb = col_base<D>(ks + PAGES * PAGE, lane);
      f32x16 sc = f32x16{};
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) sc = mma32<BF16>(load_row_frag<D>(kb, 0, kk), qf[kk], sc);
      float mx = -INFINITY;
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[r] *= c;
      if (key0 + 32 > P) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (key0 + st_key(0, r, lane) >= P) sc[r] = -INFINITY;
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, sc[r]);
      mx = max_xor32(mx);
      const float m_new = fmaxf(m, mx);
      if (__any(m_new != m)) {
        const float alpha = m == m_new ? 1.f : exp2_hw(m - m_new);
        l *= alpha;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[db][r] *= alpha;
        m = m_new;
      }
      const float mu = m == -INFINITY ? 0.f : m;   // no score above -inf so far: weights of 0
      float ps = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        sc[r] = exp2_hw(sc[r] - mu);
        ps += sc[r];
      }
      l += ps;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const f16x8 p = pack_px<BF16>(sc, j);
#pragma unroll
        for (int db = 0; db < DB; ++db) o[db] = mma32<BF16>(load_col_frag<D>(vb, 0, j, db), p, o[db]);
      }
    }
  }
  l = sum_xor32(l);

  // Merge the two key groups through LDS, register by register: lanes of the two
  // waves hold the same elements.
  wait_vmem();
  if (bad) sh_bad = 1;
  __syncthreads();
  float* sh_o = reinterpret_cast<float*>(smem) + rm * (DB * 16 * 64);
  if (kg == 1) {
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) sh_o[(db * 16 + r) * 64 + lane] = o[db][r];
    sh_m[rm][lane] = m;
    sh_l[rm][lane] = l;
  }
  __syncthreads();
  if (kg == 1 || !live) return;
  const float m1 = sh_m[rm][lane], M = fmaxf(m, m1);
  const float e0 = m == -INFINITY ? 0.f : exp2_hw(m - M), e1 = m1 == -INFINITY ? 0.f : exp2_hw(m1 - M);
  const float z = e0 * l + e1 * sh_l[rm][lane];
  const bool nan = sh_bad || z != z;
  const float inv = nan ? NAN : (z > 0.f ? 1.f / z : 0.f);
  const size_t at = (size_t)qrow * S + s;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) {
      f32x4 v;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        v[r] = (e0 * o[db][4 * r4 + r] + e1 * sh_o[(db * 16 + 4 * r4 + r) * 64 + lane]) * inv;
      *reinterpret_cast<f32x4*>(part_o + at * D + 32 * db + 8 * r4 + 4 * (lane >> 5)) = v;
    }
  if (lane < 32) part_ml[at] = make_float2(M, nan ? NAN : z);
}

// The split pass of the paged decode over the own pages, partials as it leaves them.
template <int D, bool BF16>
__global__ void __launch_bounds__(kDecThreads)
fa_own_split_kernel(const typename DecT<BF16>::e* __restrict__ q,
                    const typename DecT<BF16>::e* __restrict__ kpool,
                    const typename DecT<BF16>::e* __restrict__ vpool,
                    const int32_t* __restrict__ page_table, const int32_t* __restrict__ ctx_lens,
                    float* __restrict__ part_o, float* __restrict__ part_ml, int H, int Hkv,
                    int max_pages, int num_pages, int S, int ordered, float c) {
  __shared__ DecShared<D> sh;
  decode_split_body<D, BF16, true>(sh, blockIdx.x, blockIdx.y, blockIdx.z, gridDim.z, q, kpool, vpool,
                                   page_table, ctx_lens, part_o, part_ml, nullptr, nullptr, H, Hkv,
                                   max_pages, num_pages, S, ordered, c);
}

// O and L of a row out of the partials of both passes: one workgroup a row, D / 4
// threads a partial, the sums in a fixed order.
constexpr int kJoinThreads = 256;
constexpr int kMaxPrefixSplits = 256;
constexpr int kMaxOwnSplits = 16;

template <int D, bool BF16>
__global__ void __launch_bounds__(kJoinThreads)
fa_shared_join_kernel(const float* __restrict__ pre_o, const float2* __restrict__ pre_ml, int SP,
                      const float* __restrict__ own_o, const float2* __restrict__ own_ml, int SO,
                      typename DecT<BF16>::e* __restrict__ o, float* __restrict__ lse) {
  typedef typename DecT<BF16>::e e4 __attribute__((ext_vector_type(4)));
  constexpr int PER = D / 4, SIDE = kJoinThreads / PER, WAVES = kJoinThreads / 64;
  __shared__ float w[kMaxPrefixSplits + kMaxOwnSplits];
  __shared__ float red[2 * WAVES];
  __shared__ float acc[SIDE][D];
  const int tid = threadIdx.x, wave = tid >> 6;
  const int64_t row = blockIdx.x;
  const int S = SP + SO;
  const auto ml = [&](int i) { return i < SP ? pre_ml[row * SP + i] : own_ml[row * SO + i - SP]; };
  float M = -INFINITY;
  for (int i = tid; i < S; i += kJoinThreads) M = fmaxf(M, ml(i).x);
#pragma unroll
  for (int d = 1; d < 64; d *= 2) M = fmaxf(M, __shfl_xor(M, d));
  if ((tid & 63) == 0) red[wave] = M;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < WAVES; ++i) M = fmaxf(M, red[i]);
  float z = 0.f;
  for (int i = tid; i < S; i += kJoinThreads) {
    const float2 x = ml(i);   // an empty part: (-inf, 0), or NaN
    const float e = x.x == -INFINITY ? x.y : x.y * exp2_hw(x.x - M);
    w[i] = e;
    z += e;
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) z += __shfl_xor(z, d);
  if ((tid & 63) == 0) red[WAVES + wave] = z;
  __syncthreads();
  z = 0.f;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) z += red[WAVES + i];
  f32x4 v = f32x4{};
  const int d = 4 * (tid % PER), side = tid / PER;
#pragma unroll 4
  for (int i = side; i < S; i += SIDE) {
    const float* p = i < SP ? pre_o + (row * SP + i) * D : own_o + (row * SO + i - SP) * D;
    const f32x4 x = *reinterpret_cast<const f32x4*>(p + d);
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = fmaf(w[i], x[r], v[r]);
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) acc[side][d + r] = v[r];
  __syncthreads();
  if (side > 0) return;
  for (int i = 1; i < SIDE; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] += acc[i][d + r];
  const float inv = z == 0.f ? 0.f : 1.f / z;   // a NaN sum: NaN
  e4 out;
#pragma unroll
  for (int r = 0; r < 4; ++r) out[r] = (typename DecT<BF16>::e)(v[r] * inv);
  *reinterpret_cast<e4*>(o + row * D + d) = out;
  if (tid == 0) lse[row] = z == 0.f ? -INFINITY : (M + log2_hw(z)) * kLn2;
}

// How a call is cut: rows of a workgroup of the prefix pass, its runs of tiles,
// the splits of the own pages.
struct Plan {
  int wm, row_blocks, sp, so;
};

// Made for the 256 CUs of a whole MI355X, whatever the device has: the workspace
// follows from the sizes alone.
constexpr int kCus = 256;

static Plan plan(int64_t B, int64_t H, int64_t Hkv, int64_t prefix_pages, int64_t max_pages) {
  Plan p;
  const int64_t rows = B * (H / Hkv);
  p.wm = rows <= 32 ? 1 : (rows <= 64 ? 2 : 4);
  p.row_blocks = (int)((rows + 32 * p.wm - 1) / (32 * p.wm));
  const int64_t tiles = (prefix_pages * kPage + kTile - 1) / kTile;
  int64_t sp = kCus / (Hkv * p.row_blocks);
  sp = sp < 1 ? 1 : (sp > kMaxPrefixSplits ? kMaxPrefixSplits : sp);
  p.sp = (int)(sp > tiles ? tiles : sp);
  int64_t so = 2 * kCus / (B * decode_head_groups(H, Hkv));
  const int64_t most = (max_pages + 7) / 8;
  so = so > most ? most : so;
  p.so = (int)(so < 1 ? 1 : (so > kMaxOwnSplits ? kMaxOwnSplits : so));
  return p;
}

template <int D, bool BF16>
static int launch(const Plan& p, const void* q, const void* k_pool, const void* v_pool,
                  const int32_t* prefix_table, const int32_t* prefix_len, const int32_t* page_table,
                  const int32_t* ctx_lens, int64_t B, int64_t H, int64_t Hkv, int64_t prefix_pages,
                  int64_t max_pages, int64_t num_pages, const Topology& topo, float* ws, void* o,
                  float* lse, hipStream_t s) {
  using E = typename DecT<BF16>::e;
  const float c = (float)(1.0 / sqrt((double)D)) * kLog2e;
  const int64_t rows = B * H;
  float* pre_o = ws;
  float* own_o = pre_o + rows * p.sp * D;
  float* pre_ml = own_o + rows * p.so * D;
  float* own_ml = pre_ml + 2 * rows * p.sp;
  const dim3 grid((unsigned)(Hkv * p.sp * p.row_blocks));
#define FA_PREFIX(WM)                                                                              \
  hipLaunchKernelGGL((fa_prefix_split_kernel<D, BF16, WM>), grid, dim3(64 * WM * kKeyGroups), 0, s, \
                     (const f16*)q, (const f16*)k_pool, (const f16*)v_pool, prefix_table,          \
                     prefix_len, pre_o, (float2*)pre_ml, (int)(B * (H / Hkv)), (int)H, (int)Hkv,           \
                     (int)prefix_pages, (int)num_pages, p.sp, p.row_blocks, topo.xcds, c)
  if (p.wm == 1) FA_PREFIX(1);
  else if (p.wm == 2) FA_PREFIX(2);
  else FA_PREFIX(4);
#undef FA_PREFIX
  hipLaunchKernelGGL((fa_own_split_kernel<D, BF16>),
                     dim3((unsigned)p.so, (unsigned)decode_head_groups(H, Hkv), (unsigned)B),
                     dim3(kDecThreads), 0, s, (const E*)q, (const E*)k_pool, (const E*)v_pool,
                     page_table, ctx_lens, own_o, own_ml, (int)H, (int)Hkv, (int)max_pages,
                     (int)num_pages, p.so, (int)decode_ordered(B, H, Hkv, D, p.so, topo.cus), c);
  hipLaunchKernelGGL((fa_shared_join_kernel<D, BF16>), dim3((unsigned)rows), dim3(kJoinThreads), 0, s,
                     pre_o, (const float2*)pre_ml, p.sp, own_o, (const float2*)own_ml, p.so, (E*)o, lse);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? FA_OK : -(int)e;
}

}  // namespace shared
}  // namespace fa

extern "C" int64_t fa_decode_shared_workspace_floats(int64_t B, int64_t H, int64_t H_kv, int64_t D,
                                                     int64_t prefix_pages, int64_t max_pages) {
  if (B <= 0 || H <= 0 || H_kv <= 0 || H % H_kv != 0 || D <= 0 || prefix_pages <= 0 || max_pages <= 0)
    return 0;
  if (B > 65535 || H > 65535 || D > 128 || prefix_pages > (1 << 27) || max_pages > (1 << 27))
    return 0;   // sizes that the call refuses
  const fa::shared::Plan p = fa::shared::plan(B, H, H_kv, prefix_pages, max_pages);
  return B * H * (D + 2) * (p.sp + p.so);
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
  const Plan p = shared::plan(B, H, H_kv, prefix_pages, max_pages);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const auto fn = D == 128 ? (bf16 ? launch<128, true> : launch<128, false>)
                           : (bf16 ? launch<64, true> : launch<64, false>);
  return fn(p, q, k_pool, v_pool, prefix_table, prefix_len, page_table, ctx_lens, B, H, H_kv,
            prefix_pages, max_pages, num_pages, stream_topology(s), workspace, o, lse, s);
}
