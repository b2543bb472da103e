// MXFP4 (OCP microscaling, e2m1 elements, E8M0 block scales) building blocks.
//
// Format of a quantized matrix [rows, K]:
//   codes   uint8 [rows, 16 ceil(K / 32)]: two elements per byte, the even
//           one in the low half; a last partial block is zero-filled;
//   scales  uint8 [ceil(K / 512), rows, 16]: one byte per block of 32, e +
//           127 for the scale 2^e, 255 = NaN.  Of the 16 blocks of 512
//           elements, block 8 t + 2 g + s sits at byte 4 g + 2 t + s; bytes
//           of blocks past K are 0.
// The layout follows the matrix instruction: v_mfma_scale_f32_16x16x128
// takes 32 elements (one block, 16 code bytes) and one scale byte per lane;
// lane group g (of 4) multiplies block 8 t + 2 g + s in step (t, s), so one
// dword per lane holds its scales of four instructions (selected by opsel),
// 16 rows of a 512-element tile are 256 contiguous bytes, and the chunk
// order 2 g + s within 128 bytes is the one whose LDS reads run at the
// rate of a linear read.
//
// Quantization of a block (section 6.3 of the OCP MX specification v1.0):
// e = floor(log2(amax)) - 2 clamped to [-127, 127] (amax = 0: -127), code =
// e2m1(v 2^-e), round to nearest even, saturating at +-6; a block that holds
// NaN or an infinity gets scale byte 255 and codes 0, which the matrix
// instruction turns into NaN.
#pragma once

#include "mw8_common.h"
#include "row_overlap.h"

namespace mw8 {

constexpr int kMxBlock = 32;        // elements per scale
constexpr int kMxTile = 512;        // elements per 16-byte group of scales
constexpr int kMxTileBlocks = 16;

MW8_HD int64_t mx_blocks(int64_t k) { return (k + kMxBlock - 1) / kMxBlock; }
MW8_HD int64_t mx_tiles(int64_t k) { return (k + kMxTile - 1) / kMxTile; }
// code and scale bytes of a quantized matrix as memory
inline RowSet mx_codes_mem(const void* p, int64_t rows, int64_t k) { return one_row(p, rows * mx_blocks(k) * 16); }
inline RowSet mx_scales_mem(const void* p, int64_t rows, int64_t k) { return one_row(p, rows * mx_tiles(k) * kMxTileBlocks); }
// byte of block b (0..15) of a 512-element tile within its 16 scale bytes
MW8_HD int mx_scale_pos(int b) { return ((b >> 1) & 3) * 4 + (b >> 3) * 2 + (b & 1); }

// Scale byte from the largest sign-cleared bf16 bit pattern of a block: the
// biased exponent less 2 (floor(log2(amax)) - 2 + 127), 0 from below; the
// subnormals' true exponents lie below the clamp too.
MW8_HD uint32_t mx_scale_byte(uint32_t amax_bits) {
  const uint32_t e = amax_bits >> 7;
  return e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
}

// 2^(byte - 127) as fp32 (byte 0: the subnormal 2^-127), byte < 255
MW8_HD float mx_scale_value(uint32_t byte) {
  return __builtin_bit_cast(float, byte == 0 ? 0x00400000u : byte << 23);
}

#if !defined(MW8_HOST_ONLY)
#if defined(__HIP_DEVICE_COMPILE__)
typedef __bf16 mx_bf16x2 __attribute__((ext_vector_type(2)));

// 8 bf16 values -> 8 codes of value / scale (the conversion rounds to
// nearest even and saturates; checked for every bf16 value and scale)
__device__ __forceinline__ uint32_t mx_codes8(const U16x8& v, float scale) {
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(mx_bf16x2, v.w[0]), scale, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(mx_bf16x2, v.w[1]), scale, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(mx_bf16x2, v.w[2]), scale, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(mx_bf16x2, v.w[3]), scale, 3);
  return r;
}

__device__ __forceinline__ uint32_t mx_absmax8(const U16x8& v) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t lo = v.w[j] & 0x7FFFu, hi = (v.w[j] >> 16) & 0x7FFFu;
    m = lo > m ? lo : m;
    m = hi > m ? hi : m;
  }
  return m;
}

// Largest value over the quad of lanes that holds a block (8 elements each)
__device__ __forceinline__ uint32_t mx_quad_max(uint32_t m) {
  const uint32_t a = static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(m), 0xB1, 0xF, 0xF, false));
  m = a > m ? a : m;
  const uint32_t b = static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(m), 0x4E, 0xF, 0xF, false));
  return b > m ? b : m;
}

// The gated activation before a block quantizer.  Every block of 32 has a scale
// of its own, so the values keep their relative accuracy down to the smallest:
// 1 + erf would cancel (at g = -5 4% off, 0 from -5.6 down).  With a = |g|,
//   gelu(g) = max(g, 0) - a e^(-a^2 / 2) h(a),  h(a) = e^(a^2 / 2) erfc(a / sqrt 2) / 2,
// a^2 is exact (g holds a bf16 value) and h(a) = t Q(t) with t = 1 / (1 + 0.3 a): Q is
// the polynomial of degree 7 with the least relative error on 0 <= a <= 13.5 (2^-22.9;
// past it the product leaves fp32's range).  MI355X, 8192 x 17408 activations:
// 130 us; with erfcf 215, with 1 + erff 166; silu 105.
template <int ACT>
__device__ __forceinline__ float mx_act_fn(float g) {
  // silu: to zero from g = -87.3 down (below 2^-119; the reciprocal of e^87.3 is
  // subnormal.  Halving the exponent there kept it, for 2 to 17% more time: 2080 x
  // 25600 40.0 -> 46.9 us, in the product's epilogue 290 -> 298)
  if constexpr (ACT == 0) return act_fn<0>(g);
  const float a = __builtin_fabsf(g), t = __builtin_amdgcn_rcpf(__builtin_fmaf(a, 0.3f, 1.0f));
  float q = 0.0359320343f;
  q = __builtin_fmaf(q, t, -0.158277139f);
  q = __builtin_fmaf(q, t, 0.208208382f);
  q = __builtin_fmaf(q, t, -0.0553953275f);
  q = __builtin_fmaf(q, t, 0.129469901f);
  q = __builtin_fmaf(q, t, 0.0996372998f);
  q = __builtin_fmaf(q, t, 0.120798387f);
  q = __builtin_fmaf(q, t, 0.119626388f);
  const float e = __builtin_amdgcn_exp2f(g * g * -0.72134752044448170368f);  // / (2 ln 2)
  return __builtin_fmaxf(g, -0.0f) - a * t * (q * e);  // (-0: a zero keeps g's sign)
}

// Quantizes the block of which this lane of a quad holds 8 elements; every
// lane of the quad is active.  Returns the lane's codes, sets the block's byte.
__device__ __forceinline__ uint32_t mx_quant_quad(const U16x8& v, uint32_t& byte) {
  byte = mx_scale_byte(mx_quad_max(mx_absmax8(v)));
  return byte == 255u ? 0u : mx_codes8(v, mx_scale_value(byte));
}
#endif
#endif

}  // namespace mw8
