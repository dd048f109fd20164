// fa_decode.hip — split-KV paged decode and its logsumexp combine for MI355X.
//
// No reference counterpart: the reference has no decode path. The math is
// attention of one query token over the keys of its sequence, read through a
// page table, computed per (sequence, head, split) as a normalised partial
// (O_s, L_s), then merged by L = log sum_s exp(L_s), O = sum_s exp(L_s - L) O_s.
//
// Pool layout: [num_pages, H_kv, 16, D] fp16 or bf16 (H_kv = H, or fewer KV heads
// shared by groups of H / H_kv query heads), so the 16 tokens of one head in a
// page are 16*D*2 contiguous bytes (4 KiB at D=128), copied into LDS as
// contiguous 1 KiB requests.
//
// Split kernel: one workgroup (4 waves) per (split, KV head, up to 16 query
// heads of its group, sequence); wave w walks pages p0+w, p0+w+4, ... and
// computes the scores of every head of the workgroup and their PV products
// on the matrix cores, so a page is read once per KV head. Each wave keeps
// its own running max/sum and fp32 partial output per head; the waves merge
// through LDS at the end. With one split the kernel writes O and L itself.
#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include <mutex>

#include "fa_decode.hpp"
#include "fa_mi355x.h"
#include "fa_probe.h"
#include "fa_tile.hpp"

namespace fa {

template <int D, bool BF16>
__global__ void __launch_bounds__(kDecThreads)
fa_decode_split_kernel(const typename DecT<BF16>::e* __restrict__ q,
                       const typename DecT<BF16>::e* __restrict__ kpool,
                       const typename DecT<BF16>::e* __restrict__ vpool,
                       const int32_t* __restrict__ page_table,
                       const int32_t* __restrict__ ctx_lens, float* __restrict__ part_o,
                       float* __restrict__ part_lse, typename DecT<BF16>::e* __restrict__ o_out,
                       float* __restrict__ lse_out, int H, int Hkv, int max_pages,
                       int num_pages, int S, int ordered, float c) {
  __shared__ DecShared<D> sh;
  decode_split_body<D, BF16>(sh, blockIdx.x, blockIdx.y, blockIdx.z, gridDim.z, q, kpool, vpool,
                             page_table, ctx_lens, part_o, part_lse, o_out, lse_out, H, Hkv, max_pages,
                             num_pages, S, ordered, c);
}

// Combine: D / 4 threads per row (b, h), four columns each. All of a row's
// loads (its S logsumexps and the thread's S partials) are issued before the
// first is used, so the pass waits for memory once (a thread per column with
// loops over S waited three times and more: B1 H32, 16 splits, decode 47.3 ->
// 43.2 us, B8 28.5 -> 24.5); the sums run in split order.
constexpr int kMaxSplits = 16;
constexpr int kCombThreads = 256;

template <int D, bool BF16>
__global__ void __launch_bounds__(kCombThreads)
fa_lse_combine_kernel(const float* __restrict__ part_o, const float* __restrict__ part_lse,
                      typename DecT<BF16>::e* __restrict__ o, float* __restrict__ lse, int S,
                      int rows) {
  // Element alignment only, as the pointers promise no more (one wide access
  // all the same: the target takes unaligned ones).
  typedef typename DecT<BF16>::e e4v __attribute__((ext_vector_type(4)));
  typedef e4v e4 __attribute__((aligned(2)));
  typedef f32x4 f4 __attribute__((aligned(4)));
  constexpr int PER = D / 4;   // threads of a row
  const int row = blockIdx.x * (kCombThreads / PER) + (int)threadIdx.x / PER;
  if (row >= rows) return;
  const int d = 4 * ((int)threadIdx.x % PER);
  const float* pl = part_lse + (size_t)row * S;
  const float* po = part_o + (size_t)row * S * D + d;
  float ls[kMaxSplits];
  f32x4 ps[kMaxSplits];
#pragma unroll
  for (int s = 0; s < kMaxSplits; ++s) {
    ls[s] = -INFINITY;
    ps[s] = f32x4{};
    if (s < S) {
      ls[s] = pl[s];
      ps[s] = *reinterpret_cast<const f4*>(po + (size_t)s * D);
    }
  }
  float M = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int s = 0; s < kMaxSplits; ++s) {
    nan |= (ls[s] != ls[s]);
    M = fmaxf(M, ls[s]);
  }
  f32x4 out = f32x4{};
  float L;
  if (nan) {
    out = f32x4{NAN, NAN, NAN, NAN};
    L = NAN;
  } else if (M == -INFINITY) {
    L = -INFINITY;
  } else {
    float z = 0.f;
#pragma unroll
    for (int s = 0; s < kMaxSplits; ++s)
      if (s < S) z += exp2_hw((ls[s] - M) * kLog2e);
    L = M + log2_hw(z) * kLn2;
#pragma unroll
    for (int s = 0; s < kMaxSplits; ++s) {
      if (s < S) {
        const float w = exp2_hw((ls[s] - L) * kLog2e);
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = fmaf(w, ps[s][i], out[i]);
      }
    }
  }
  e4v v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = (typename DecT<BF16>::e)out[i];
  *reinterpret_cast<e4*>(o + (size_t)row * D + d) = v;
  if (lse != nullptr && d == 0) lse[row] = L;
}

}  // namespace fa

namespace fa {
// Split pass with query heads h reading pool head h / (H / Hkv); arguments
// already validated. With o (num_splits 1) the kernel writes the result
// itself and the partials are not used.
template <bool BF16>
static int decode_split(const void* q, const void* k_pool, const void* v_pool,
                        const int32_t* page_table, const int32_t* ctx_lens, int64_t B, int64_t H,
                        int64_t Hkv, int64_t D, int64_t max_pages, int64_t num_pages,
                        int64_t num_splits, float* part_o, float* part_lse, void* o, float* lse,
                        void* stream) {
  using E = typename DecT<BF16>::e;
  if (o == nullptr && (!part_o || !part_lse)) return FA_ERR_NULL_POINTER;
  const float c = (float)(1.0 / sqrt((double)D)) * kLog2e;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  // One workgroup per (split, KV head, 16 of its query heads, sequence).
  const dim3 grid((unsigned)num_splits, (unsigned)decode_head_groups(H, Hkv), (unsigned)B);
  const int ordered = decode_ordered(B, H, Hkv, D, num_splits, stream_topology(s).cus);
#define FA_DECODE_SPLIT(DD)                                                                        \
  hipLaunchKernelGGL((fa_decode_split_kernel<DD, BF16>), grid, dim3(kDecThreads), 0, s,            \
                     (const E*)q, (const E*)k_pool, (const E*)v_pool, page_table, ctx_lens, part_o, \
                     part_lse, (E*)o, lse, (int)H, (int)Hkv, (int)max_pages, (int)num_pages,       \
                     (int)num_splits, ordered, c)
  if (D == 128) FA_DECODE_SPLIT(128);
  else FA_DECODE_SPLIT(64);
#undef FA_DECODE_SPLIT
  hipError_t e = hipGetLastError();
  return e == hipSuccess ? FA_OK : -(int)e;
}

// LSE combine of [B, H, num_splits] partials into O [B, H, D] (fp16 or bf16)
// and L fp32 [B, H] (may be null).
template <bool BF16>
static int lse_combine(const float* part_o, const float* part_lse, int64_t B, int64_t H,
                       int64_t D, int64_t num_splits, void* o, float* lse, void* stream) {
  using E = typename DecT<BF16>::e;
  if (!part_o || !part_lse || !o) return FA_ERR_NULL_POINTER;
  if (D != 64 && D != 128) return FA_ERR_HEAD_DIM;
  if (B <= 0 || H <= 0) return FA_ERR_BATCH_HEADS;
  if (num_splits < 1 || num_splits > 16) return FA_ERR_NUM_SPLITS;
  if (B * H > (int64_t(1) << 31) - 1) return FA_ERR_TOO_LARGE;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int rows = (int)(B * H), per_wg = kCombThreads / (int)(D / 4);
  const dim3 grid((unsigned)((rows - 1) / per_wg + 1));
  if (D == 128) {
    hipLaunchKernelGGL((fa_lse_combine_kernel<128, BF16>), grid, dim3(kCombThreads), 0, s, part_o,
                       part_lse, (E*)o, lse, (int)num_splits, rows);
  } else {
    hipLaunchKernelGGL((fa_lse_combine_kernel<64, BF16>), grid, dim3(kCombThreads), 0, s, part_o,
                       part_lse, (E*)o, lse, (int)num_splits, rows);
  }
  hipError_t e = hipGetLastError();
  return e == hipSuccess ? FA_OK : -(int)e;
}
}  // namespace fa

extern "C" int fa_probe_decode_ordered(int64_t B, int64_t H, int64_t H_kv, int64_t D,
                                       int64_t num_splits, int cus) {
  if (B <= 0 || H <= 0 || H_kv <= 0 || H % H_kv != 0 || cus <= 0) return 0;
  return B <= fa::kDecThreads && fa::decode_ordered(B, H, H_kv, D, num_splits, cus);
}

extern "C" int fa_decode_split_f16(const void* q, const void* k_pool, const void* v_pool,
                                   const int32_t* page_table, const int32_t* ctx_lens,
                                   int64_t B, int64_t H, int64_t D, int64_t page_size,
                                   int64_t max_pages, int64_t num_pages, int64_t num_splits,
                                   float* part_o, float* part_lse, void* stream) {
  int st = fa_validate_decode(q, k_pool, v_pool, page_table, ctx_lens, B, H, D, page_size,
                              max_pages, num_pages, num_splits);
  if (st != FA_OK) return st;
  return fa::decode_split<false>(q, k_pool, v_pool, page_table, ctx_lens, B, H, H, D, max_pages,
                                 num_pages, num_splits, part_o, part_lse, nullptr, nullptr, stream);
}

extern "C" int fa_lse_combine_f32(const float* part_o, const float* part_lse, int64_t B,
                                  int64_t H, int64_t D, int64_t num_splits, void* o,
                                  float* lse, void* stream) {
  return fa::lse_combine<false>(part_o, part_lse, B, H, D, num_splits, o, lse, stream);
}

namespace fa {
template <bool BF16>
static int decode_paged_gqa(const void* q, const void* k_pool, const void* v_pool,
                            const int32_t* page_table, const int32_t* ctx_lens, int64_t B,
                            int64_t H, int64_t H_kv, int64_t D, int64_t page_size,
                            int64_t max_pages, int64_t num_pages, int64_t num_splits,
                            float* part_o, float* part_lse, void* o, float* lse, void* stream) {
  int st = fa_validate_decode(q, k_pool, v_pool, page_table, ctx_lens, B, H, D, page_size,
                              max_pages, num_pages, num_splits);
  if (st != FA_OK) return st;
  if (H_kv <= 0 || H % H_kv != 0) return FA_ERR_KV_HEADS;
  if (!part_o || !part_lse || !o) return FA_ERR_NULL_POINTER;
  if (B * H > (int64_t(1) << 31) - 1) return FA_ERR_TOO_LARGE;
  if (num_splits == 1)
    return decode_split<BF16>(q, k_pool, v_pool, page_table, ctx_lens, B, H, H_kv, D, max_pages,
                              num_pages, 1, part_o, part_lse, o, lse, stream);
  st = decode_split<BF16>(q, k_pool, v_pool, page_table, ctx_lens, B, H, H_kv, D, max_pages,
                          num_pages, num_splits, part_o, part_lse, nullptr, nullptr, stream);
  if (st != FA_OK) return st;
  return lse_combine<BF16>(part_o, part_lse, B, H, D, num_splits, o, lse, stream);
}
}  // namespace fa

extern "C" int fa_decode_paged_f16(const void* q, const void* k_pool, const void* v_pool,
                                   const int32_t* page_table, const int32_t* ctx_lens,
                                   int64_t B, int64_t H, int64_t D, int64_t page_size,
                                   int64_t max_pages, int64_t num_pages, int64_t num_splits,
                                   float* part_o, float* part_lse, void* o, float* lse,
                                   void* stream) {
  return fa::decode_paged_gqa<false>(q, k_pool, v_pool, page_table, ctx_lens, B, H, H, D,
                                     page_size, max_pages, num_pages, num_splits, part_o,
                                     part_lse, o, lse, stream);
}

extern "C" int fa_decode_paged_gqa_f16(const void* q, const void* k_pool, const void* v_pool,
                                       const int32_t* page_table, const int32_t* ctx_lens,
                                       int64_t B, int64_t H, int64_t H_kv, int64_t D,
                                       int64_t page_size, int64_t max_pages, int64_t num_pages,
                                       int64_t num_splits, float* part_o, float* part_lse,
                                       void* o, float* lse, void* stream) {
  return fa::decode_paged_gqa<false>(q, k_pool, v_pool, page_table, ctx_lens, B, H, H_kv, D,
                                     page_size, max_pages, num_pages, num_splits, part_o,
                                     part_lse, o, lse, stream);
}

extern "C" int fa_decode_paged_bf16(const void* q, const void* k_pool, const void* v_pool,
                                    const int32_t* page_table, const int32_t* ctx_lens,
                                    int64_t B, int64_t H, int64_t H_kv, int64_t D,
                                    int64_t page_size, int64_t max_pages, int64_t num_pages,
                                    int64_t num_splits, float* part_o, float* part_lse, void* o,
                                    float* lse, void* stream) {
  return fa::decode_paged_gqa<true>(q, k_pool, v_pool, page_table, ctx_lens, B, H, H_kv, D,
                                    page_size, max_pages, num_pages, num_splits, part_o,
                                    part_lse, o, lse, stream);
}

// ---------------------------------------------------------------------------
// Allocation-free paged decode: the split partials (part_o, then part_lse)
// live in a file-scope device array instead of a caller workspace, for
// callers that cannot allocate device memory. The split pass writes every
// partial it owns (an empty split writes 0 and -inf), so nothing in the array
// needs clearing between calls.
namespace fa {
// One copy per GPU that loads this library, held until the process ends. In
// host code `scratch` names a host-side stand-in: only the address returned
// by hipGetSymbolAddress for the current device may reach a kernel.
static __device__ __align__(256) float scratch[FA_DECODE_SCRATCH_FLOATS];

constexpr int kScratchDevices = 64;
static std::mutex g_scratch_mu;
static float* g_scratch_addr[kScratchDevices];   // per device, null until resolved

// Device address of `scratch` on device `dev`, resolved on first use with
// `dev` current (then the previous current device is restored).
static int scratch_addr(int dev, float** out) {
  if (dev < 0 || dev >= kScratchDevices) return -(int)hipErrorInvalidDevice;
  std::lock_guard<std::mutex> lock(g_scratch_mu);
  if (g_scratch_addr[dev] == nullptr) {
    int cur = 0;
    hipError_t e = hipGetDevice(&cur);
    if (e != hipSuccess) return -(int)e;
    if (cur != dev && (e = hipSetDevice(dev)) != hipSuccess) return -(int)e;
    void* p = nullptr;
    e = hipGetSymbolAddress(&p, HIP_SYMBOL(scratch));
    const hipError_t e2 = cur != dev ? hipSetDevice(cur) : hipSuccess;
    if (e != hipSuccess) return -(int)e;
    if (e2 != hipSuccess) return -(int)e2;
    if (p == nullptr) return -(int)hipErrorInvalidSymbol;
    g_scratch_addr[dev] = static_cast<float*>(p);
  }
  *out = g_scratch_addr[dev];
  return FA_OK;
}
}  // namespace fa

extern "C" int fa_decode_paged_noalloc_f16(const void* q, const void* k_pool,
                                           const void* v_pool, const int32_t* page_table,
                                           const int32_t* ctx_lens, int64_t B, int64_t H,
                                           int64_t H_kv, int64_t D, int64_t page_size,
                                           int64_t max_pages, int64_t num_pages,
                                           int64_t num_splits, void* o, float* lse,
                                           void* stream) {
  int st = fa_validate_decode(q, k_pool, v_pool, page_table, ctx_lens, B, H, D, page_size,
                              max_pages, num_pages, num_splits);
  if (st != FA_OK) return st;
  if (o == nullptr) return FA_ERR_NULL_POINTER;
  if (H_kv <= 0 || H % H_kv != 0) return FA_ERR_KV_HEADS;
  // B, H, D and num_splits are bounded by the validation above, so the
  // product cannot overflow.
  if (B * H * num_splits * (D + 1) > FA_DECODE_SCRATCH_FLOATS) return FA_ERR_SCRATCH_SIZE;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  int dev = 0;
  hipError_t e = s != nullptr ? hipStreamGetDevice(s, &dev) : hipGetDevice(&dev);
  if (e != hipSuccess) return -(int)e;
  float* part_o = nullptr;
  st = fa::scratch_addr(dev, &part_o);
  if (st != FA_OK) return st;
  float* part_lse = part_o + B * H * num_splits * D;
  return fa::decode_paged_gqa<false>(q, k_pool, v_pool, page_table, ctx_lens, B, H, H_kv, D,
                                     page_size, max_pages, num_pages, num_splits, part_o,
                                     part_lse, o, lse, stream);
}
