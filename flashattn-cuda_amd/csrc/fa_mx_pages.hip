// fa_mx_pages.hip — writer and reader of the KV cache in MX pages (fa_mx.hpp):
// rows of 16-bit values quantised as they are written, and read back.
//
// No reference counterpart (the reference has no KV cache). Positions, page
// table and flags are the 16-bit writer's (fa_pages.hip).
//
// Both are bound by memory: 2 D bytes of a row on one side and
// D bits / 8 + D / 32 on the other, no reuse. A thread has 8 values of a row
// (16 bytes of it, its block shared with three neighbours), D / 8 threads a
// row; a workgroup has whole pages (one at D = 128, two at D = 64) of one head,
// so that its stores fill a page's codes without a gap wherever the call covers
// the page.
#include <hip/hip_runtime.h>

#include <stdint.h>

#include "fa_mi355x.h"
#include "fa_mx.hpp"
#include "fa_pages.hpp"

namespace fa {
namespace mx {

using pages::any_bad;
using pages::kThreads;

// Tokens of a workgroup.
template <int D>
constexpr int kRows = kThreads / (D / 8);

// Rows read back of this size and more are written past the caches. The read
// alone is faster by it at any size; a kernel after it that reads all rows at once
// then finds them in memory and is slower by as much or more, until they outgrow
// the caches (us, alone and with that kernel, one sequence over 8 heads, D = 128:
//   65 MB 19.4 -> 14.0, 33.1 -> 35.2;  102 MB 28.6 -> 20.4, 49.1 -> 51.7;
//   131 MB 35.5 -> 25.5, 63.6 -> 64.5; 205 MB 53.6 -> 38.4, 101.3 -> 104.3;
//   262 MB, two sequences, 63.4 -> 45.7, 138.7 -> 126.0).
// So a caller gains where more than a pass over memory comes between, or from
// 256 MB on; smaller rows are left where their reader finds them.
constexpr int64_t kPassThrough = 100 << 20;

// Workgroups along a sequence that cover T tokens from any position: whole
// pages, the first and the last of which may be covered in part.
template <int D>
static unsigned token_blocks(int64_t T) {
  if (T <= 0) return 1;
  const int64_t pages = (T - 1 + kTokens - 1) / kTokens + 1, per = kRows<D> / kTokens;
  return (unsigned)((pages + per - 1) / per);
}

// Which token and page slot a thread has.
struct Place {
  int64_t t;     // token of the call; outside [0, n): none
  int64_t page;  // of the sequence
  int slot, u;   // row of the page, eighth-value group of the row
};
template <int D>
__device__ __forceinline__ Place place_of(int start, unsigned block) {
  Place r;
  const int row = (int)threadIdx.x / (D / 8);
  const int64_t pos = (int64_t)(start & ~(kTokens - 1)) + (int64_t)block * kRows<D> + row;
  r.t = pos - start;
  r.page = pos >> 4;   // of a negative position: negative
  r.slot = (int)(pos & (kTokens - 1));
  r.u = (int)threadIdx.x % (D / 8);
  return r;
}

// Largest of the block's magnitudes: the four threads of a quad have a block.
__device__ __forceinline__ uint32_t quad_max(uint32_t x) {
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xB1, 0xf, 0xf, true));   // lane ^ 1
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4E, 0xf, 0xf, true));   // lane ^ 2
  return x;
}

// Eight 16-bit values to codes and their block's scale code. A block with a
// NaN or an infinity has scale code 255 and codes 0.
template <int BITS, bool BF16>
__device__ __forceinline__ uint32_t quantize(const u32x4 raw, uint32_t (&w)[BITS / 4]) {
  float x[8];
  uint32_t mag = 0;   // magnitudes compare as integers
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = raw[i] & 0xffffu, hi = raw[i] >> 16;
    mag = max(mag, max(lo & 0x7fffu, hi & 0x7fffu));
    if constexpr (BF16) {
      x[2 * i] = __uint_as_float(lo << 16);
      x[2 * i + 1] = __uint_as_float(hi << 16);
    } else {
      x[2 * i] = (float)__builtin_bit_cast(f16, (uint16_t)lo);
      x[2 * i + 1] = (float)__builtin_bit_cast(f16, (uint16_t)hi);
    }
  }
  mag = quad_max(mag);
  const bool finite = mag < (BF16 ? 0x7f80u : 0x7c00u);
  const float a = BF16 ? __uint_as_float(mag << 16) : (float)__builtin_bit_cast(f16, (uint16_t)mag);
  const int s = scale_code<BITS, BF16>(finite ? a : 0.f);
  codes8<BITS>(x, scale_of((uint32_t)s), w);
#pragma unroll
  for (int i = 0; i < BITS / 4; ++i) w[i] = finite ? w[i] : 0u;
  return finite ? (uint32_t)s : 255u;
}

// A thread's codes into K or V page `page`, at slot t.
template <int D, int BITS>
__device__ __forceinline__ void store_k(char* page, int t, int u, const uint32_t (&w)[BITS / 4]) {
  char* p = page + k_codes<D, BITS>(t, u);
  if constexpr (BITS == 4) *reinterpret_cast<uint32_t*>(p) = w[0];
  else *reinterpret_cast<u32x2*>(p) = u32x2{w[0], w[1]};
}
template <int D, int BITS>
__device__ __forceinline__ void store_v(char* page, int t, int u, const uint32_t (&w)[BITS / 4]) {
  if constexpr (D == 128) {
    char* p = page + v_codes<D, BITS>(t, u);
    if constexpr (BITS == 4) *reinterpret_cast<uint32_t*>(p) = w[0];
    else *reinterpret_cast<u32x2*>(p) = u32x2{w[0], w[1]};
  } else {
    char* p0 = page + v_codes<D, BITS>(t, 2 * u);
    char* p1 = page + v_codes<D, BITS>(t, 2 * u + 1);
    if constexpr (BITS == 4) {
      *reinterpret_cast<uint16_t*>(p0) = (uint16_t)w[0];
      *reinterpret_cast<uint16_t*>(p1) = (uint16_t)(w[0] >> 16);
    } else {
      *reinterpret_cast<uint32_t*>(p0) = w[0];
      *reinterpret_cast<uint32_t*>(p1) = w[1];
    }
  }
}

template <int D, int BITS>
__device__ __forceinline__ void load_k(const char* page, int t, int u, uint32_t (&w)[BITS / 4]) {
  const char* p = page + k_codes<D, BITS>(t, u);
  if constexpr (BITS == 4) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else {
    const u32x2 x = *reinterpret_cast<const u32x2*>(p);
    w[0] = x[0];
    w[1] = x[1];
  }
}
template <int D, int BITS>
__device__ __forceinline__ void load_v(const char* page, int t, int u, uint32_t (&w)[BITS / 4]) {
  if constexpr (D == 128) {
    const char* p = page + v_codes<D, BITS>(t, u);
    if constexpr (BITS == 4) {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
      const u32x2 x = *reinterpret_cast<const u32x2*>(p);
      w[0] = x[0];
      w[1] = x[1];
    }
  } else {
    const char* p0 = page + v_codes<D, BITS>(t, 2 * u);
    const char* p1 = page + v_codes<D, BITS>(t, 2 * u + 1);
    if constexpr (BITS == 4) {
      w[0] = (uint32_t)*reinterpret_cast<const uint16_t*>(p0) |
             (uint32_t)*reinterpret_cast<const uint16_t*>(p1) << 16;
    } else {
      w[0] = *reinterpret_cast<const uint32_t*>(p0);
      w[1] = *reinterpret_cast<const uint32_t*>(p1);
    }
  }
}

// Eight values of codes, as raw 16-bit pairs.
template <int BITS, bool BF16>
__device__ __forceinline__ u32x4 values8(const uint32_t (&w)[BITS / 4], float scale) {
  if constexpr (BITS == 4)
    return u32x4{values2<4, BF16, 0>(w[0], scale), values2<4, BF16, 1>(w[0], scale),
                 values2<4, BF16, 2>(w[0], scale), values2<4, BF16, 3>(w[0], scale)};
  else
    return u32x4{values2<8, BF16, 0>(w[0], scale), values2<8, BF16, 1>(w[0], scale),
                 values2<8, BF16, 0>(w[1], scale), values2<8, BF16, 1>(w[1], scale)};
}

template <int D, int KB, int VB, bool BF16>
__global__ void __launch_bounds__(kThreads)
fa_kv_append_mx_kernel(const u32x4* __restrict__ k_new, const u32x4* __restrict__ v_new,
                       const int32_t* __restrict__ page_table,
                       const int32_t* __restrict__ start_pos,
                       const int32_t* __restrict__ new_lens, char* __restrict__ k_pool,
                       char* __restrict__ v_pool, int32_t* __restrict__ bad, int H, int T,
                       int max_pages, int num_pages) {
  const int h = blockIdx.y, b = blockIdx.z;
  const int start = start_pos[b];
  const int32_t* pt = page_table + (size_t)b * max_pages;
  int n = T;
  if (new_lens) n = min(max(new_lens[b], 0), T);
  if (blockIdx.x == 0 && h == 0) {
    const bool any = any_bad(pt, start, n, max_pages, num_pages);
    if (threadIdx.x == 0) bad[b] = any;
  }
  const Place p = place_of<D>(start, blockIdx.x);
  // The four threads of a block leave together: their row is one.
  if (p.t < 0 || p.t >= n || p.page < 0 || p.page >= max_pages) return;
  const int pid = pt[p.page];
  if (pid < 0 || pid >= num_pages) return;
  const size_t src = (((size_t)b * H + h) * T + (size_t)p.t) * (D / 8) + p.u;
  const size_t dst = (size_t)pid * H + h;
  const u32x4 kx = k_new[src], vx = v_new[src];
  uint32_t kw[KB / 4], vw[VB / 4];
  const uint32_t ks = quantize<KB, BF16>(kx, kw);
  const uint32_t vs = quantize<VB, BF16>(vx, vw);
  char* kp = k_pool + dst * Page<D, KB>::BYTES;
  char* vp = v_pool + dst * Page<D, VB>::BYTES;
  store_k<D, KB>(kp, p.slot, p.u, kw);
  store_v<D, VB>(vp, p.slot, p.u, vw);
  if ((p.u & 3) == 0) {
    kp[k_scale<D, KB>(p.slot, p.u >> 2)] = (char)ks;
    vp[v_scale<D, VB>(p.slot, p.u >> 2)] = (char)vs;
  }
}

// NT: the rows are written with the non-temporal hint, and the heads of a page
// are read one after the other (16 heads of 4 x 4096 tokens with the hint alone
// 31.4 us, with the order alone 31.9, with both 23.0).
template <int D, int KB, int VB, bool BF16, bool NT>
__global__ void __launch_bounds__(kThreads)
fa_kv_read_mx_kernel(const char* __restrict__ k_pool, const char* __restrict__ v_pool,
                     const int32_t* __restrict__ page_table, const int32_t* __restrict__ start_pos,
                     const int32_t* __restrict__ lens, u32x4* __restrict__ k, u32x4* __restrict__ v,
                     int32_t* __restrict__ bad, int H, int T, int max_pages, int num_pages) {
  const int h = NT ? blockIdx.x % H : blockIdx.y, b = blockIdx.z;
  const unsigned block = NT ? blockIdx.x / H : blockIdx.x;
  const int start = start_pos[b];
  const int32_t* pt = page_table + (size_t)b * max_pages;
  int n = T;
  if (lens) n = min(max(lens[b], 0), T);
  if (block == 0 && h == 0) {
    const bool any = any_bad(pt, start, n, max_pages, num_pages);
    if (threadIdx.x == 0) bad[b] = any;
  }
  const Place p = place_of<D>(start, block);
  if (p.t < 0 || p.t >= T) return;
  u32x4 kx = u32x4{}, vx = u32x4{};   // rows past the sequence's own: zeros
  if (p.t < n) {
    const int pid = p.page >= 0 && p.page < max_pages ? pt[p.page] : -1;
    if (pid >= 0 && pid < num_pages) {
      const size_t src = (size_t)pid * H + h;
      const char* kp = k_pool + src * Page<D, KB>::BYTES;
      const char* vp = v_pool + src * Page<D, VB>::BYTES;
      uint32_t kw[KB / 4], vw[VB / 4];
      load_k<D, KB>(kp, p.slot, p.u, kw);
      load_v<D, VB>(vp, p.slot, p.u, vw);
      const uint32_t ks = (uint8_t)kp[k_scale<D, KB>(p.slot, p.u >> 2)];
      const uint32_t vs = (uint8_t)vp[v_scale<D, VB>(p.slot, p.u >> 2)];
      kx = values8<KB, BF16>(kw, scale_of(ks));
      vx = values8<VB, BF16>(vw, scale_of(vs));
    } else {
      constexpr uint32_t nan2 = BF16 ? 0x7fc07fc0u : 0x7e007e00u;
      kx = vx = u32x4{nan2, nan2, nan2, nan2};
    }
  }
  const size_t dst = (((size_t)b * H + h) * T + (size_t)p.t) * (D / 8) + p.u;
  if constexpr (NT) {
    __builtin_nontemporal_store(kx, &k[dst]);
    __builtin_nontemporal_store(vx, &v[dst]);
  } else {
    k[dst] = kx;
    v[dst] = vx;
  }
}

template <int D, int KB, int VB, bool BF16>
static int append(const void* k_new, const void* v_new, const int32_t* page_table,
                  const int32_t* start_pos, const int32_t* new_lens, void* k_pool, void* v_pool,
                  int32_t* bad, int64_t B, int64_t H, int64_t T, int64_t max_pages,
                  int64_t num_pages, hipStream_t s) {
  const dim3 grid(token_blocks<D>(T), (unsigned)H, (unsigned)B);
  hipLaunchKernelGGL((fa_kv_append_mx_kernel<D, KB, VB, BF16>), grid, dim3(kThreads), 0, s,
                     (const u32x4*)k_new, (const u32x4*)v_new, page_table, start_pos, new_lens,
                     (char*)k_pool, (char*)v_pool, bad, (int)H, (int)T, (int)max_pages,
                     (int)num_pages);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? FA_OK : -(int)e;
}

template <int D, int KB, int VB, bool BF16>
static int read(const void* k_pool, const void* v_pool, const int32_t* page_table,
                const int32_t* start_pos, const int32_t* lens, void* k, void* v, int32_t* bad,
                int64_t B, int64_t H, int64_t T, int64_t max_pages, int64_t num_pages,
                hipStream_t s) {
  const int64_t blocks = token_blocks<D>(T);
  // (a grid holds fewer than 2^32 threads along x)
  const bool nt = B * H * T >= kPassThrough / (4 * D) && blocks * H < (1 << 24);
  const dim3 grid((unsigned)(nt ? blocks * H : blocks), nt ? 1u : (unsigned)H, (unsigned)B);
  const auto kernel = nt ? fa_kv_read_mx_kernel<D, KB, VB, BF16, true>
                         : fa_kv_read_mx_kernel<D, KB, VB, BF16, false>;
  hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, s, (const char*)k_pool, (const char*)v_pool,
                     page_table, start_pos, lens, (u32x4*)k, (u32x4*)v, bad, (int)H, (int)T,
                     (int)max_pages, (int)num_pages);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? FA_OK : -(int)e;
}

}  // namespace mx
}  // namespace fa

extern "C" int fa_kv_append_mx(const void* k_new, const void* v_new, const int32_t* page_table,
                               const int32_t* start_pos, const int32_t* new_lens, void* k_pool,
                               void* v_pool, int32_t* bad, int64_t B, int64_t H, int64_t T,
                               int64_t D, int64_t k_bits, int64_t v_bits, int64_t page_size,
                               int64_t max_pages, int64_t num_pages, int bf16, void* stream) {
  const int st = fa_validate_kv_append_mx(k_new, v_new, page_table, start_pos, new_lens, k_pool,
                                          v_pool, bad, B, H, T, D, k_bits, v_bits, page_size,
                                          max_pages, num_pages);
  if (st != FA_OK) return st;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define FA_MX_APPEND(DD, KB, VB, BF)                                                               \
  return fa::mx::append<DD, KB, VB, BF>(k_new, v_new, page_table, start_pos, new_lens, k_pool,     \
                                        v_pool, bad, B, H, T, max_pages, num_pages, s)
  FA_MX_DISPATCH(D, k_bits, v_bits, bf16, FA_MX_APPEND)
#undef FA_MX_APPEND
}

extern "C" int fa_kv_read_mx(const void* k_pool, const void* v_pool, const int32_t* page_table,
                             const int32_t* start_pos, const int32_t* lens, void* k, void* v,
                             int32_t* bad, int64_t B, int64_t H, int64_t T, int64_t D,
                             int64_t k_bits, int64_t v_bits, int64_t page_size, int64_t max_pages,
                             int64_t num_pages, int bf16, void* stream) {
  const int st = fa_validate_kv_append_mx(k, v, page_table, start_pos, lens, k_pool, v_pool, bad, B,
                                          H, T, D, k_bits, v_bits, page_size, max_pages, num_pages);
  if (st != FA_OK) return st;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define FA_MX_READ(DD, KB, VB, BF)                                                                 \
  return fa::mx::read<DD, KB, VB, BF>(k_pool, v_pool, page_table, start_pos, lens, k, v, bad, B, H, \
                                      T, max_pages, num_pages, s)
  FA_MX_DISPATCH(D, k_bits, v_bits, bf16, FA_MX_READ)
#undef FA_MX_READ
}
