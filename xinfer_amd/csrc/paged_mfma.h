// Matrix-core helpers of attention over the paged 4-bit cache.
//
// Scores: a key's codes and scales go to the scaled matrix instructions as they lie in the cache (A operand, e2m1 with
// a scale a block of 32).  A query's bf16 features go as the sum of two e4m3 terms (B operand, scales of their own):
// a bf16 number has 8 significant bits, the first term takes the upper 4 and what is left, at most 4 bits, is the
// second term exactly.  So q is exact for features within 2^-14 of their block's largest, and off by at most 2^-23 of
// that below.  The two products take the time of one in bf16 and spare the keys' conversion and three quarters
// of their LDS traffic.  The instruction keeps about 2^-17 of a sum's largest term (measured: operands of random
// exponents over 2^30 against float64).
//
// Layouts (checked against float64 on the device): 16x16x128 with lane l: A row l % 16, k = 32 (l / 16) + 0..31, the
// scale that of this block; B column l % 16, k = 16 (l / 16) + 0..15 and 64 + 16 (l / 16) + 0..15, but the scale that
// of block l / 16; C column l % 16, rows 4 (l / 16) + 0..3.  32x32x64: A row l % 32, k = 32 (l / 32) + 0..31; B
// k = 16 (l / 32) + 0..15 and 32 + 16 (l / 32) + 0..15; C column l % 32, row 8 (r / 4) + 4 (l / 32) + r % 4 of
// register r.
#pragma once

#include "kv4_device.h"

namespace xattn {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef short i16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// Two weights as bf16 in one instruction (pack_bf16x2 takes four).
__device__ __forceinline__ uint32_t pack_weights(float lo, float hi) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, bf16x2));
}

// Adds two packed weights to a sum.  The instruction is off by up to 1.5 ulp of the result, on average 0.03 downwards
// (measured: weights and sums of random exponents against float64), so it is for sums of a few words.
__device__ __forceinline__ float add_weights(uint32_t word, float sum) {
  return __builtin_amdgcn_fdot2_f32_bf16(as_bf16x2(word), as_bf16x2(0x3f803f80u), sum, false);
}

template <int OPA, int OPB>
__device__ __forceinline__ f32x4 mfma16_fp4(const u32x4 &a, const u32x4 (&b)[2], f32x4 c, int scale_a, int scale_b) {
  const i32x8 x{(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
  const i32x8 y{(int)b[0][0], (int)b[0][1], (int)b[0][2], (int)b[0][3], (int)b[1][0], (int)b[1][1], (int)b[1][2], (int)b[1][3]};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 4, 0, OPA, scale_a, OPB, scale_b);
}
template <int OPA, int OPB>
__device__ __forceinline__ f32x16 mfma32_fp4(const u32x4 &a, const u32x4 (&b)[2], f32x16 c, int scale_a, int scale_b) {
  const i32x8 x{(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
  const i32x8 y{(int)b[0][0], (int)b[0][1], (int)b[0][2], (int)b[0][3], (int)b[1][0], (int)b[1][1], (int)b[1][2], (int)b[1][3]};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x, y, c, 4, 0, OPA, scale_a, OPB, scale_b);
}

// Scale byte of a query block's first term, from its largest magnitude's bits: the term's values stay below 256.
// The second term's is 4 lower.  255 (NaN) for a block with an infinity or a NaN: its query's output is NaN.
__device__ __forceinline__ int query_scale(uint32_t bits) {
  return bits >= 0x7f800000u ? 255 : max((int)(bits >> 23) - 7, 8);
}
__device__ __forceinline__ uint32_t largest(const u32x4 &x, uint32_t top) {
#pragma unroll
  for (int e = 0; e < 4; ++e) top = max(top, max((x[e] << 16) & 0x7fffffffu, x[e] & 0x7fff0000u));
  return top;
}
// Eight features (bf16) as the two terms, for a block of scale byte `scale`.
__device__ __forceinline__ void split_query(const u32x4 &x, int scale, u32x2 &first, u32x2 &second) {
  const float unit = kv4_scale_value(min(scale, 254)), small = unit * 0.0625f;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const float f[4] = {bf16_lo(x[2 * w]), bf16_hi(x[2 * w]), bf16_lo(x[2 * w + 1]), bf16_hi(x[2 * w + 1])};
    i16x2 p{0, 0}, r{0, 0};
    p = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(p, f[0], f[1], unit, false);
    p = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(p, f[2], f[3], unit, true);
    const uint32_t word = __builtin_bit_cast(uint32_t, p);
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(word, unit, false);
    const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(word, unit, true);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, f[0] - a[0], f[1] - a[1], small, false);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, f[2] - b[0], f[3] - b[1], small, true);
    first[w] = word;
    second[w] = __builtin_bit_cast(uint32_t, r);
  }
}
// Sixteen (two chunks).
__device__ __forceinline__ void split_query(const u32x4 &x0, const u32x4 &x1, int scale, u32x4 &first, u32x4 &second) {
  u32x2 f[2], r[2];
  split_query(x0, scale, f[0], r[0]);
  split_query(x1, scale, f[1], r[1]);
  first = u32x4{f[0].x, f[0].y, f[1].x, f[1].y};
  second = u32x4{r[0].x, r[0].y, r[1].x, r[1].y};
}

}  // namespace xattn
