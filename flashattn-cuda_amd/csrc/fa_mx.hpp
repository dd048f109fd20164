// fa_mx.hpp — pages of the KV cache in microscaling (MX) formats: geometry and
// conversions shared by the writer, the reader and the decode.
//
// A row (one token's K or V of one head) is D values in blocks of 32 along D.
// A block has a scale 2^(s - 127), s one byte (E8M0; 255 stands for NaN), and
// its values are E2M1 (4 bits: 0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives)
// or E4M3 (8 bits, up to 448). A page is 16 tokens of one head: their codes,
// then their scales.
//
// The codes lie as the decode's lanes take them, so that a page is one (two
// at 128 bytes a row) contiguous load of the wave, straight into registers in
// the operand layout of the matrix products:
//   K  lane (t, g), t = lane % 16 a token, g = lane / 16: values
//      g D/4 .. + D/4 - 1 of row t. Its piece is number 4 t + g, so K codes
//      are plain rows.
//   V  lane (c, a), c = lane % 16, a = lane / 16: values c D/16 .. + D/16 - 1
//      of tokens 4 a .. 4 a + 3, token by token. Its piece is number lane.
// Pieces are 16 consecutive bytes (8 at 4 bits and D = 64); the 32-byte pieces
// of 8 bits and D = 128 are kept as two planes of 16-byte halves. In a byte of
// two 4-bit values the even one is the low half.
//
// Scales: K [token][block] (a lane of K has one), V [block][token] (a lane of
// V takes those of its four tokens as one word).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fa_tile.hpp"

namespace fa {
namespace mx {

constexpr int kTokens = 16;   // of a page

template <int D, int BITS>
struct Page {
  static constexpr int ROW = D * BITS / 8;          // code bytes of a row
  static constexpr int CODES = kTokens * ROW;
  static constexpr int BLOCKS = D / 32;             // of a row
  static constexpr int BYTES = CODES + kTokens * BLOCKS;
  static constexpr int PIECE = CODES / 64;          // code bytes of a lane: 8, 16 or 32
  static constexpr int WORDS = PIECE / 4;
};

// Offset of the codes of values 8 u .. 8 u + 7 (BITS bytes) of K row t.
template <int D, int BITS>
__device__ __forceinline__ int k_codes(int t, int u) {
  if constexpr (Page<D, BITS>::ROW == 128)
    return ((u & 3) >> 1) * 1024 + (t * 4 + (u >> 2)) * 16 + (u & 1) * 8;
  else
    return t * Page<D, BITS>::ROW + u * BITS;
}

// Offset of the codes of values c D/16 .. + D/16 - 1 (D BITS / 128 bytes) of V row t.
template <int D, int BITS>
__device__ __forceinline__ int v_codes(int t, int c) {
  constexpr int W = D * BITS / 128;
  const int cell = (t >> 2) * 16 + c, r = t & 3;
  if constexpr (W == 8)
    return (r >> 1) * 1024 + cell * 16 + (r & 1) * 8;
  else
    return cell * 4 * W + r * W;
}

template <int D, int BITS>
__device__ __forceinline__ int k_scale(int t, int block) {
  return Page<D, BITS>::CODES + t * Page<D, BITS>::BLOCKS + block;
}

template <int D, int BITS>
__device__ __forceinline__ int v_scale(int t, int block) {
  return Page<D, BITS>::CODES + block * kTokens + t;
}

// ---------------------------------------------------------------------------
// Conversions, with the instructions that take the scale as an operand: they
// round to nearest even, use the exponent bits of the scale alone, and give
// NaN for exponent 255 (checked over every code and every scale, and every
// 16-bit value).
// ---------------------------------------------------------------------------

// 2^(s - 127), or what the conversions take for NaN.
__device__ __forceinline__ float scale_of(uint32_t s) { return __uint_as_float(s << 23); }

// The scale in byte R of a word, the other bytes in its sign and fraction,
// which the conversions from codes do not look at (checked over every scale).
template <int R>
__device__ __forceinline__ float scale_at(uint32_t w) {
  return __uint_as_float(R == 3 ? w >> 1 : w << (23 - 8 * R));
}

// Values 2 I and 2 I + 1 of a word of codes (I < 4 at 4 bits, < 2 at 8), as
// raw 16-bit pairs. Exact wherever the type has the value.
template <int BITS, bool BF16, int I>
__device__ __forceinline__ uint32_t values2(uint32_t w, float scale) {
  if constexpr (BITS == 4) {
    if constexpr (BF16)
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, I));
    else
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, I));
  } else {
    if constexpr (BF16)
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, I != 0));
    else
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, I != 0));
  }
}

// The scale code of a block whose largest magnitude is a (finite): the
// smallest s >= 1 with a <= lim 2^(s - 127), lim = 7 = 1.75 2^2 or
// 464 = 1.8125 2^8, half a step past the format's largest (6, 448), to which
// values up to there go (464 by its tie, 7 by saturation: its tie is 8). The
// fraction of a above that of lim carries into the exponent. At most the code
// for which the format's largest value is finite in the rows' type: values past
// it saturate, which leaves them more than half a step off (of fp16 rows 65504
// becomes 49152 in 4 bits, 57344 in 8).
template <int BITS, bool BF16>
__device__ __forceinline__ int scale_code(float a) {
  constexpr uint32_t carry = BITS == 4 ? 0x7fffffu - 0x600000u : 0x7fffffu - 0x680000u;
  constexpr int lim_exp = BITS == 4 ? 2 : 8;
  constexpr int top = BF16 ? (BITS == 4 ? 252 : 246) : (BITS == 4 ? 140 : 134);
  const int s = (int)((__float_as_uint(a) + carry) >> 23) - lim_exp;
  return min(max(s, 1), top);
}

// Codes of eight finite values with the block's scale: BITS bytes, in order.
template <int BITS>
__device__ __forceinline__ void codes8(const float (&x)[8], float scale, uint32_t (&w)[BITS / 4]) {
  if constexpr (BITS == 4) {
    uint32_t r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[0], x[1], scale, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[2], x[3], scale, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[4], x[5], scale, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[6], x[7], scale, 3);
    w[0] = r;
  } else {
    typedef short s16x2 __attribute__((ext_vector_type(2)));
    // This conversion makes values past 464 NaN: saturated first.
    const float top = 448.f * scale;
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = fminf(fmaxf(x[i], -top), top);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      s16x2 r = s16x2{0, 0};
      r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, y[4 * i], y[4 * i + 1], scale, false);
      r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, y[4 * i + 2], y[4 * i + 3], scale, true);
      w[i] = __builtin_bit_cast(uint32_t, r);
    }
  }
}

}  // namespace mx
}  // namespace fa

// M(D, KB, VB, BF16) for the run-time head dimension, widths and type.
#define FA_MX_DISPATCH_B(DD, kb, vb, BF, M)             \
  {                                                     \
    if ((kb) == 4 && (vb) == 4) { M(DD, 4, 4, BF); }    \
    if ((kb) == 4) { M(DD, 4, 8, BF); }                 \
    if ((vb) == 4) { M(DD, 8, 4, BF); }                 \
    M(DD, 8, 8, BF);                                    \
  }
#define FA_MX_DISPATCH(D, kb, vb, bf16, M)                                       \
  if ((D) == 128) {                                                              \
    if (bf16) FA_MX_DISPATCH_B(128, kb, vb, true, M)                             \
    FA_MX_DISPATCH_B(128, kb, vb, false, M)                                      \
  }                                                                              \
  if (bf16) FA_MX_DISPATCH_B(64, kb, vb, true, M)                                \
  FA_MX_DISPATCH_B(64, kb, vb, false, M)
