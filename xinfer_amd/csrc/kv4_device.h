// Device helpers of the 4-bit KV cache (format: kv4_common.h).
#pragma once

#include "device_common.h"
#include "kv4_common.h"

namespace xattn {

// Block-uniform loads through the scalar unit.
__device__ __forceinline__ int64_t scalar_load(const int64_t *p, int64_t i) {
  typedef const __attribute__((address_space(4))) int64_t *ptr;
  return ((ptr)p)[i];
}

// Lane l's largest of x over its aligned group of four lanes.
__device__ __forceinline__ uint32_t quad_max(uint32_t x) {
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, kDppXor1, 0xF, 0xF, false));
  return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, kDppXor2, 0xF, 0xF, false));
}

// Scale byte of a block whose largest magnitude has the (finite) fp32 bits `bits`.
__device__ __forceinline__ int kv4_scale(uint32_t bits) {
  const int e = (int)(bits >> 23) - 2 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, kKv4MinScale), kKv4MaxScale);
}
__device__ __forceinline__ float kv4_scale_value(int scale) { return __uint_as_float((uint32_t)scale << 23); }

// Eight features as codes (the scaled conversion divides by the scale and rounds to the nearest, ties to even,
// saturating at 6).
__device__ __forceinline__ uint32_t kv4_codes(const float (&x)[8], float scale) {
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], scale, 3);
}
// Eight codes as bf16 values (exact).
__device__ __forceinline__ u32x4 kv4_values(uint32_t w, float scale) {
  return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3))};
}

// Places of a slot's vector of KV head h: codes of lane chunk c (8 features, 4 bytes) and the scale of its block.
struct Kv4Place {
  int64_t codes, scale;
};
__device__ __forceinline__ Kv4Place kv4_place(const Kv4Cache &cache, int64_t slot, int h, int c) {
  const int64_t page = slot >> cache.page_shift;
  const int at = (int)(slot & ((1 << cache.page_shift) - 1)), size = 1 << cache.page_shift;
  const int64_t head = page * cache.Hkv + h;
  return Kv4Place{(head * size + at) * (cache.D / 2) + 4 * c, (head * (cache.D / kKv4Block) + c / 4) * size + at};
}
__device__ __forceinline__ bool kv4_holds(const Kv4Cache &cache, int64_t slot) {
  return slot >= 0 && slot < (cache.pages << cache.page_shift);
}

// Quantises and stores a (slot, KV head)'s key and value, 8 features of each per lane, D/8 lanes together.  live:
// whether this lane's row is stored; every lane of the wave calls it.
template <int LPR>
__device__ __forceinline__ void kv4_store(const Kv4Cache &cache, int64_t slot, int h, int c, const float (&k)[8],
                                          const float (&v)[8], bool live) {
  uint32_t kmax = 0, vmax = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    kmax = max(kmax, __float_as_uint(k[e]) & 0x7fffffffu);  // NaNs are above infinity, infinity above all others
    vmax = max(vmax, __float_as_uint(v[e]) & 0x7fffffffu);
  }
  const uint64_t odd = __ballot(max(kmax, vmax) >= 0x7f800000u);
  const int lane = threadIdx.x & 63;
  const uint64_t row = (LPR == 64 ? ~0ull : (1ull << LPR) - 1) << (lane & ~(LPR - 1));
  const bool finite = (odd & row) == 0;
  const int ks = kv4_scale(quad_max(kmax)), vs = kv4_scale(quad_max(vmax));
  const uint32_t kw = finite ? kv4_codes(k, kv4_scale_value(ks)) : 0u, vw = finite ? kv4_codes(v, kv4_scale_value(vs)) : 0u;
  if (!live) return;
  const Kv4Place p = kv4_place(cache, slot, h, c);
  *as_global(reinterpret_cast<uint32_t *>(cache.key + p.codes)) = kw;
  *as_global(reinterpret_cast<uint32_t *>(cache.value + p.codes)) = vw;
  if ((c & 3) == 0) {
    *as_global(cache.key_scale + p.scale) = (uint8_t)(finite ? ks : kKv4NanScale);
    *as_global(cache.value_scale + p.scale) = (uint8_t)(finite ? vs : kKv4MinScale);
  }
}

__device__ __forceinline__ void unpack_floats(const u32x4 &x, float (&f)[8]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    f[2 * e] = bf16_lo(x[e]);
    f[2 * e + 1] = bf16_hi(x[e]);
  }
}

}  // namespace xattn
