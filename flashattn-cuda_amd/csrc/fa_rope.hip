// fa_rope.hip — rotary positions for MI355X: Q and K rotated (or gradients
// rotated back) in one launch, and the same fused with the KV page writer.
//
// No reference counterpart. Of the first R dims of a row at position p, pair i
// (x1, x2) becomes, with a = p f_i,
//   y1 = s (x1 cos a - x2 sin a),   y2 = s (x2 cos a + x1 sin a);
// pairs are dims (i, i + R/2), or neighbours (2i, 2i + 1). The way back is the
// transpose: -a for a. Dims from R on are copied.
//
// Bound: memory, each row read and written once. A thread keeps 8 pairs of one
// token (two 16-byte pieces of a 16-bit row), works out their 8 angles once and
// walks over heads of q, k (and v) with them, so the trigonometry is shared by
// the heads and needs no table in memory. Rows are addressed by strides: the
// [B, N, H, D] a projection leaves is read as it is and written head-major.
//
// Kernel times, us: 4 x 4096 tokens, 16 + 16 heads of D = 128, bf16: 42.6, 6.3 TB/s (a
// plain copy of 256 MB 5.4; calls in turn on other rows 52). Gradients of 2 x 2000 tokens,
// 32 + 8 heads of D = 128, fp32 to bf16: 21.3, 5.8 TB/s. The append of two prompts of up to
// 1777 tokens, 32 heads over 8, D = 128: 16.3. One token of 8 sequences: 4.2; 1024 tokens,
// 8 + 8 heads of D = 64: 3.4, with the library's sine and cosine half a us more. Rows asked
// for after the angles: 51.4, 24.7, 17.3, 4.6 and 3.7. Loads and stores with the
// non-temporal hint: 25 -> 36, 17.4 -> 20.5.
#include <hip/hip_runtime.h>

#include <stdint.h>

#include "fa_mi355x.h"
#include "fa_pages.hpp"
#include "fa_tile.hpp"

namespace fa {
namespace rope {

using pages::kPageSize;
using pages::kThreads;

// Eight consecutive values of a row as they lie in memory.
template <int TYPE>
struct Vec {   // FA_F16, FA_BF16
  f16x8 x;
};
template <>
struct Vec<FA_F32> {
  f32x4 x, y;
};
template <int TYPE>
struct Elem {
  using t = f16;
};
template <>
struct Elem<FA_F32> {
  using t = float;
};

template <int TYPE>
__device__ __forceinline__ Vec<TYPE> load8(const typename Elem<TYPE>::t* p) {
  return *reinterpret_cast<const Vec<TYPE>*>(p);
}

template <int TYPE>
__device__ __forceinline__ void widen(const Vec<TYPE>& v, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (TYPE == FA_F32) {
      f[i] = i < 4 ? v.x[i & 3] : v.y[i & 3];
    } else {
      const f16 h = v.x[i];   // a value: a bit cast of the element itself reads element 0
      if constexpr (TYPE == FA_BF16) f[i] = __uint_as_float((uint32_t)__builtin_bit_cast(uint16_t, h) << 16);
      else f[i] = (float)h;
    }
  }
}

// The one rounding of a value: to nearest even.
template <int TYPE>
__device__ __forceinline__ Vec<TYPE> narrow(const float (&f)[8]) {
  Vec<TYPE> v;
  if constexpr (TYPE == FA_F32) {
    v.x = f32x4{f[0], f[1], f[2], f[3]};
    v.y = f32x4{f[4], f[5], f[6], f[7]};
  } else {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const f16x2 p = cvt2x<TYPE == FA_BF16>(f[i], f[i + 1]);
      v.x[i] = p[0];
      v.x[i + 1] = p[1];
    }
  }
  return v;
}

// Rows of one input: element strides of sequence, head and token.
struct Rows {
  const void* p;
  int64_t sb, sh, sn;
};

struct Args {
  Rows in[3];              // q, k, v (v: the append only)
  void* out[2];            // rotated q, k, contiguous [B, h, N, D]; k's may be null in the append
  const double* freqs;     // radians a position, R / 2 of them
  const int32_t* pos;      // rope: [B, N] (pos_stride N, 0: one row for all) or null
  int64_t pos_stride;      // append: positions of the first tokens [B]
  int N, H, Hkv, D, R;
  float scale;
  int back;                // rotate by -a
  int tt_log2, per_wg;     // tokens of a workgroup (a power of two); heads a thread takes
  // the append
  const int32_t* table;
  const int32_t* start;
  const int32_t* lens;
  void* pool[2];
  int32_t* bad;
  int max_pages, num_pages;
};

constexpr int kBatch = 2;   // heads whose loads a thread has in flight (1, 2, 4, 8: 44.0 42.6 43.9 45.6 us of
                            // the first call above, 21.1 21.3 22.5 32.8 of the second)

// Thread (hs, tok, u): 8 pairs u of token tok, heads hs, hs + HS, ...: HS =
// 256 / (tokens * D/16) heads side by side, so that a call of single tokens
// still fills its waves.
template <int IN, int OUT, bool INTER, bool APPEND>
__global__ void __launch_bounds__(kThreads) fa_rope_kernel(const Args a) {
  using EI = typename Elem<IN>::t;
  using EO = typename Elem<OUT>::t;
  const int units = a.D / 16;   // threads of a row: 4 or 8
  const int u_log2 = units == 8 ? 3 : 2;
  const int tid = threadIdx.x;
  const int u = tid & (units - 1);
  const int tok = (tid >> u_log2) & ((1 << a.tt_log2) - 1);
  const int hs = tid >> (u_log2 + a.tt_log2);
  const int HS = kThreads >> (u_log2 + a.tt_log2);
  const int b = blockIdx.z;
  const int t = ((int)blockIdx.x << a.tt_log2) + tok;
  int n = a.N;
  int64_t slot = 0;
  if constexpr (APPEND) {
    if (a.lens) n = min(max(a.lens[b], 0), a.N);
    const int first = a.start[b];
    slot = (int64_t)first + t;
    if (blockIdx.x == 0 && blockIdx.y == 0) {
      const bool any = pages::any_bad(a.table + (size_t)b * a.max_pages, first, n, a.max_pages, a.num_pages);
      if (tid == 0) a.bad[b] = any;
    }
  }
  if (t >= a.N) return;
  const bool live = t < n;
  const int heads = a.H + a.Hkv + (APPEND ? a.Hkv : 0);
  int h = (int)blockIdx.y * a.per_wg * HS + hs;
  if (h >= heads) return;

  // Page of the token, the append's destination of k and v.
  int64_t page_row = -1;   // pool row of head 0, in rows of D; -1: none
  if constexpr (APPEND) {
    if (live && slot >= 0 && slot < (int64_t)a.max_pages * kPageSize) {
      const int pid = a.table[(size_t)b * a.max_pages + (size_t)(slot / kPageSize)];
      if (pid >= 0 && pid < a.num_pages)
        page_row = (int64_t)pid * a.Hkv * kPageSize + slot % kPageSize;
    }
  }

  // Dims of the unit: two pieces of eight, ea and eb. Rotated units come first.
  const bool turn = u < a.R / 16;
  const int ea = turn && !INTER ? 8 * u : 16 * u;
  const int eb = turn && !INTER ? a.R / 2 + 8 * u : 16 * u + 8;
  // Rows are asked for before the angles are worked out.
  Vec<IN> xa[kBatch], xb[kBatch];
  const auto load = [&](int i) {
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int hj = h + j * HS;
      xa[j] = Vec<IN>{};
      xb[j] = Vec<IN>{};
      if (i + j < a.per_wg && hj < heads && live) {
        const Rows& r = hj < a.H ? a.in[0] : (!APPEND || hj < a.H + a.Hkv ? a.in[1] : a.in[2]);
        const int hh = hj < a.H ? hj : (hj < a.H + a.Hkv ? hj - a.H : hj - a.H - a.Hkv);
        const EI* src = (const EI*)r.p + b * r.sb + hh * r.sh + t * r.sn;
        xa[j] = load8<IN>(src + ea);
        xb[j] = load8<IN>(src + eb);
      }
    }
  };
  load(0);
  float cs[8], sn[8];
  if (turn && h < a.H + a.Hkv) {
    int64_t p;
    if constexpr (APPEND) p = (a.pos ? (int64_t)a.pos[b] : (int64_t)a.start[b]) + t;
    else p = a.pos ? a.pos[b * a.pos_stride + t] : t;
    // In turns and 64 bits up to the fraction of a turn: 32 would leave the
    // angle of position 100000 off by 0.004. v_sin_f32 and v_cos_f32 take turns;
    // they are off by 2^-22.9 at most (measured over 2^26 values of [-1/2, 1/2]).
    constexpr double kTurn = 0.15915494309189533577;
    const double pd = (double)p;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const double x = pd * (a.freqs[8 * u + j] * kTurn);
      const float f = (float)(x - rint(x));
      const float s = __builtin_amdgcn_sinf(f), c = __builtin_amdgcn_cosf(f);
      cs[j] = c * a.scale;
      sn[j] = (a.back ? -s : s) * a.scale;
    }
  }

  for (int i = 0; i < a.per_wg; i += kBatch, h += kBatch * HS) {
    if (i > 0) load(i);
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int hj = h + j * HS;
      if (i + j >= a.per_wg || hj >= heads) break;
      const bool is_q = hj < a.H, is_v = APPEND && hj >= a.H + a.Hkv;
      Vec<OUT> ya, yb;
      bool copy = !turn || is_v;
      if constexpr (IN == OUT) {
        ya = xa[j];
        yb = xb[j];
      } else {
        copy = false;
      }
      if (!copy) {
        float fa[8], fb[8], ga[8], gb[8];
        widen<IN>(xa[j], fa);
        widen<IN>(xb[j], fb);
        if (turn) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            if constexpr (INTER) {   // pairs (2j, 2j + 1) of the 16 values
              const float x1 = e < 4 ? fa[2 * (e & 3)] : fb[2 * (e & 3)];
              const float x2 = e < 4 ? fa[2 * (e & 3) + 1] : fb[2 * (e & 3) + 1];
              const float y1 = x1 * cs[e] - x2 * sn[e], y2 = x2 * cs[e] + x1 * sn[e];
              (e < 4 ? ga : gb)[2 * (e & 3)] = y1;
              (e < 4 ? ga : gb)[2 * (e & 3) + 1] = y2;
            } else {
              ga[e] = fa[e] * cs[e] - fb[e] * sn[e];
              gb[e] = fb[e] * cs[e] + fa[e] * sn[e];
            }
          }
          ya = narrow<OUT>(ga);
          yb = narrow<OUT>(gb);
        } else {
          ya = narrow<OUT>(fa);
          yb = narrow<OUT>(fb);
        }
      }
      const int hh = is_q ? hj : (is_v ? hj - a.H - a.Hkv : hj - a.H);
      if (!is_v) {
        EO* dst = (EO*)a.out[is_q ? 0 : 1];
        if (!APPEND || dst != nullptr) {
          dst += (((int64_t)b * (is_q ? a.H : a.Hkv) + hh) * a.N + t) * a.D;
          *reinterpret_cast<Vec<OUT>*>(dst + ea) = ya;
          *reinterpret_cast<Vec<OUT>*>(dst + eb) = yb;
        }
      }
      if constexpr (APPEND) {
        if (!is_q && page_row >= 0) {
          EO* dst = (EO*)a.pool[is_v ? 1 : 0] + (page_row + (int64_t)hh * kPageSize) * a.D;
          *reinterpret_cast<Vec<OUT>*>(dst + ea) = ya;
          *reinterpret_cast<Vec<OUT>*>(dst + eb) = yb;
        }
      }
    }
  }
}

// Tokens of a workgroup, the heads a thread walks over and the grid: about 2048
// workgroups, where the angles are shared by as many heads as leave the chip full. The
// first three calls above, us, for 2048 and 4096: 42.6 43.9; 21.3 21.1; 16.3 17.2; four
// heads in flight and 512, 1024, 2048, 4096: 51.6 51.8 43.9 44.0.
static dim3 plan(Args& a, int64_t B, bool append) {
  const int units = a.D / 16;
  int tt = 0;
  while ((units << (tt + 1)) <= kThreads && (1 << tt) < a.N) ++tt;
  a.tt_log2 = tt;
  const int64_t side = kThreads / (units << tt);   // heads side by side
  const int64_t heads = a.H + a.Hkv + (append ? a.Hkv : 0);
  const int64_t slots = (heads + side - 1) / side;
  const int64_t blocks = a.N > 0 ? ((int64_t)a.N + (1 << tt) - 1) >> tt : 1;   // no tokens: the flags
  int64_t per = blocks * B * slots / 2048;
  per = per < 1 ? 1 : (per > slots ? slots : per);
  a.per_wg = (int)per;
  return dim3((unsigned)blocks, (unsigned)((slots + per - 1) / per), (unsigned)B);
}

template <int IN, int OUT, bool APPEND>
static int launch(Args& a, int64_t B, int interleaved, void* stream) {
  const dim3 grid = plan(a, B, APPEND);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (interleaved) hipLaunchKernelGGL((fa_rope_kernel<IN, OUT, true, APPEND>), grid, dim3(kThreads), 0, s, a);
  else hipLaunchKernelGGL((fa_rope_kernel<IN, OUT, false, APPEND>), grid, dim3(kThreads), 0, s, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? FA_OK : -(int)e;
}

static Rows rows(const void* p, const int64_t* st) {
  return p ? Rows{p, st[0], st[1], st[2]} : Rows{nullptr, 0, 0, 0};
}

}  // namespace rope
}  // namespace fa

extern "C" int fa_rope(const void* q, const int64_t q_strides[3], const void* k,
                       const int64_t k_strides[3], const double* freqs, const int32_t* positions,
                       int64_t pos_stride, void* q_out, void* k_out, int64_t B, int64_t H,
                       int64_t H_kv, int64_t N, int64_t D, int64_t rot_dim, float scale,
                       int interleaved, int back, int in_type, int out_type, void* stream) {
  const int st = fa_validate_rope(q, q_strides, k, k_strides, freqs, positions, pos_stride, q_out,
                                  k_out, B, H, H_kv, N, D, rot_dim, in_type, out_type);
  if (st != FA_OK) return st;
  using namespace fa::rope;
  Args a{};
  a.in[0] = rows(q, q_strides);
  a.in[1] = rows(k, k_strides);
  a.out[0] = q_out;
  a.out[1] = k_out;
  a.freqs = freqs;
  a.pos = positions;
  a.pos_stride = pos_stride;
  a.N = (int)N, a.H = (int)H, a.Hkv = (int)H_kv, a.D = (int)D, a.R = (int)rot_dim;
  a.scale = scale;
  a.back = back != 0;
  if (in_type == FA_F16) return launch<FA_F16, FA_F16, false>(a, B, interleaved, stream);
  if (in_type == FA_BF16) return launch<FA_BF16, FA_BF16, false>(a, B, interleaved, stream);
  if (out_type == FA_F16) return launch<FA_F32, FA_F16, false>(a, B, interleaved, stream);
  if (out_type == FA_BF16) return launch<FA_F32, FA_BF16, false>(a, B, interleaved, stream);
  return launch<FA_F32, FA_F32, false>(a, B, interleaved, stream);
}

extern "C" int fa_kv_append_rope(const void* q, const int64_t q_strides[3], const void* k,
                                 const int64_t k_strides[3], const void* v,
                                 const int64_t v_strides[3], const double* freqs,
                                 const int32_t* page_table, const int32_t* start_pos,
                                 const int32_t* positions, const int32_t* new_lens, void* k_pool,
                                 void* v_pool, void* q_out, void* k_out, int32_t* bad, int64_t B,
                                 int64_t H, int64_t H_kv, int64_t T, int64_t D, int64_t rot_dim,
                                 float scale, int interleaved, int64_t page_size, int64_t max_pages,
                                 int64_t num_pages, int bf16, void* stream) {
  const int st = fa_validate_kv_append_rope(q, q_strides, k, k_strides, v, v_strides, freqs,
                                            page_table, start_pos, positions, new_lens, k_pool,
                                            v_pool, q_out, k_out, bad, B, H, H_kv, T, D, rot_dim,
                                            page_size, max_pages, num_pages);
  if (st != FA_OK) return st;
  using namespace fa::rope;
  Args a{};
  a.in[0] = rows(q, q_strides);
  a.in[1] = rows(k, k_strides);
  a.in[2] = rows(v, v_strides);
  a.out[0] = q_out;
  a.out[1] = k_out;
  a.freqs = freqs;
  a.pos = positions;
  a.N = (int)T, a.H = (int)H, a.Hkv = (int)H_kv, a.D = (int)D, a.R = (int)rot_dim;
  a.scale = scale;
  a.table = page_table;
  a.start = start_pos;
  a.lens = new_lens;
  a.pool[0] = k_pool;
  a.pool[1] = v_pool;
  a.bad = bad;
  a.max_pages = (int)max_pages, a.num_pages = (int)num_pages;
  return bf16 ? launch<FA_BF16, FA_BF16, true>(a, B, interleaved, stream)
              : launch<FA_F16, FA_F16, true>(a, B, interleaved, stream);
}
