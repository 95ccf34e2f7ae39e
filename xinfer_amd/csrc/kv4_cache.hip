// Writing and reading the paged 4-bit KV cache (format: kv4_common.h): the append, the query/key norm and rotation
// with the append in one launch, and the read-back.
//
// A row is a (token, head); LPR = D/8 lanes hold it, 8 features each, so a block's largest magnitude is one
// exchange among four lanes.  A lane takes the same features of the token's key and of its value, because a token
// is stored as not finite if either is.
//
// What bounds them: memory, and latency for few tokens.  2963 tokens of 8 x 512 places, 4 KV heads of 256 features: append
// 6.3 us (15 MB, 2.4 TB/s; half of it is the launch and one memory round trip), read-back 5.7 us (20 MB, 3.5 TB/s), norm
// with 16 query heads 21.5 us (82 MB, 3.8 TB/s; a large copy moves 4.9 TB/s).  8 single tokens, 8 heads of 128: append
// 2.2 us, read-back 2.2, norm 3.6.
#include "kv4_device.h"
#include "launch.h"

namespace xattn {

template <int LPR>
__global__ void __launch_bounds__(256) append_kv4_kernel(const Kv4AppendArgs a) {
  const uint32_t i = blockIdx.x * (256 / LPR) + threadIdx.x / LPR, Hkv = a.cache.Hkv;
  const int c = threadIdx.x % LPR;
  const bool row = i < (uint32_t)a.B * a.T * Hkv;
  const uint32_t token = row ? i / Hkv : 0;
  const int h = row ? (int)(i - token * Hkv) : 0, b = (int)(token / (uint32_t)a.T), t = (int)(token - b * (uint32_t)a.T);
  const int64_t slot = a.slots[b * a.slot_sb + t * a.slot_st];
  float k[8], v[8];
  unpack_floats(load16(a.key.p + b * a.key.sb + h * a.key.sh + t * a.key.st + 8 * c), k);
  unpack_floats(load16(a.value.p + b * a.value.sb + h * a.value.sh + t * a.value.st + 8 * c), v);
  kv4_store<LPR>(a.cache, slot, h, c, k, v, row && kv4_holds(a.cache, slot));
}

template <int LPR>
__global__ void __launch_bounds__(256) read_kv4_kernel(const Kv4ReadArgs a) {
  const uint32_t i = blockIdx.x * (256 / LPR) + threadIdx.x / LPR, Hkv = a.cache.Hkv;
  const int c = threadIdx.x % LPR;
  if (i >= (uint32_t)a.B * a.T * Hkv) return;
  // Output order: [B, Hkv, T].
  const uint32_t bh = i / (uint32_t)a.T;
  const int t = (int)(i - bh * a.T), b = (int)(bh / Hkv), h = (int)(bh - b * Hkv);
  const int64_t slot = a.slots[b * a.slot_sb + t * a.slot_st];
  u32x4 k{0, 0, 0, 0}, v{0, 0, 0, 0};
  if (kv4_holds(a.cache, slot)) {
    const Kv4Place p = kv4_place(a.cache, slot, h, c);
    const int ks = *as_global(a.cache.key_scale + p.scale), vs = *as_global(a.cache.value_scale + p.scale);
    k = kv4_values(*as_global(reinterpret_cast<const uint32_t *>(a.cache.key + p.codes)), kv4_scale_value(ks));
    v = kv4_values(*as_global(reinterpret_cast<const uint32_t *>(a.cache.value + p.codes)),
                   kv4_scale_value(min(vs, kKv4MaxScale)));
    if (ks == kKv4NanScale) k = u32x4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};
  }
  store16(a.key + (int64_t)i * (8 * LPR) + 8 * c, k);
  store16(a.value + (int64_t)i * (8 * LPR) + 8 * c, v);
}

// y = x * rsqrt(mean(x^2) + eps) * (weight + offset); of its first R features, the first half turns to
// y_i cos_i - y_{i + R/2} sin_i and the second to y_i cos_i + y_{i - R/2} sin_i, all in F.  The rotation's other half is
// read from memory again (a line this wave reads anyway) and normalised here, which takes no exchange between lanes.
template <int LPR>
struct NormRopeRow {
  u32x4 x, x_other, w, w_other, cos, sin;
  bool turned, low;
  __device__ __forceinline__ void load(const uint16_t *row, const uint16_t *weight, const uint16_t *c, const uint16_t *s,
                                       int R, int chunk) {
    const int half = R / 16;  // chunks of half the rotated features
    low = chunk < half;
    turned = chunk < 2 * half;
    const int other = low ? chunk + half : (turned ? chunk - half : chunk);
    x = load16(row + 8 * chunk);
    x_other = load16(row + 8 * other);
    w = load16(weight + 8 * chunk);
    w_other = load16(weight + 8 * other);
    cos = load16(c + 8 * (turned ? chunk : 0));
    sin = load16(s + 8 * (turned ? chunk : 0));
  }
  static __device__ __forceinline__ double row_sum(double v) {
    for (int mask = 1; mask < LPR; mask *= 2)
      v += __hiloint2double(__shfl_xor(__double2hiint(v), mask), __shfl_xor(__double2loint(v), mask));
    return v;
  }
  static __device__ __forceinline__ float row_sum(float v) { return group_sum<LPR>(v); }
  static __device__ __forceinline__ float root(float v) { return rsqrtf(v); }
  // Newton's step on the fp32 root: 2^-22 squares to 2^-44.  Where that root is infinite, so is the definition's.
  static __device__ __forceinline__ double root(double v) {
    const double r = (double)rsqrtf((float)v);
    return v > 0 && isfinite((float)r) ? r * (1.5 - 0.5 * v * r * r) : r;
  }
  template <typename F>
  __device__ __forceinline__ void compute(float eps, float offset, float (&y)[8]) const {
    float a[8], b[8], wa[8], wb[8], cs[8], sn[8];
    unpack_floats(x, a);
    unpack_floats(x_other, b);
    unpack_floats(w, wa);
    unpack_floats(w_other, wb);
    unpack_floats(cos, cs);
    unpack_floats(sin, sn);
    F ss = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += (F)(a[e] * a[e]);  // x^2 is exact in fp32
    const F inv = root(row_sum(ss) * (F)(1.0 / (8 * LPR)) + (F)eps);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const F p = (F)a[e] * inv * ((F)wa[e] + (F)offset), q = (F)b[e] * inv * ((F)wb[e] + (F)offset);
      y[e] = (float)(turned ? p * (F)cs[e] + (low ? -q : q) * (F)sn[e] : p);
    }
  }
};

// Whether a key's codes could be others if its values were off by 2^-20 of the row's largest, which bounds the fp32
// arithmetic above: a value next to a border of the grid, or a block's largest next to one of the scale.
template <int LPR>
__device__ __forceinline__ bool near_border(const float (&y)[8]) {
  float top = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(y[e]));
  const uint32_t block = quad_max(__float_as_uint(top));
  float row = __uint_as_float(block);
  row = fmaxf(row, dpp_move<kDppHalfMirror>(row));
  if constexpr (LPR >= 16) row = fmaxf(row, dpp_move<kDppMirror>(row));
  if constexpr (LPR >= 32) row = pair_max16(row);
  const float margin = row * 0x1p-20f, largest = __uint_as_float(block);
  const int scale = kv4_scale(__float_as_uint(largest + margin));
  float up[8], down[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    up[e] = fabsf(y[e]) + margin;
    down[e] = fmaxf(fabsf(y[e]) - margin, 0.0f);
  }
  return kv4_scale(__float_as_uint(fmaxf(largest - margin, 0.0f))) != scale ||
         kv4_codes(up, kv4_scale_value(scale)) != kv4_codes(down, kv4_scale_value(scale));
}

template <int LPR>
__global__ void __launch_bounds__(256) norm_rope_kv4_kernel(const Kv4NormRopeArgs a) {
  constexpr int HEADS = 64 / LPR;  // heads a wave takes together
  const int Hkv = a.cache.Hkv;
  const int q_tasks = (a.Hq + HEADS - 1) / HEADS, tasks = q_tasks + (Hkv + HEADS - 1) / HEADS;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  const uint32_t token = wave / (uint32_t)tasks;
  if (token >= (uint32_t)a.B * a.T) return;
  const int task = (int)(wave - token * tasks), b = (int)(token / (uint32_t)a.T), t = (int)(token - b * (uint32_t)a.T);
  const int lane = threadIdx.x & 63, c = lane % LPR;
  const bool query = task < q_tasks;
  const int heads = query ? a.Hq : Hkv, h = (task - (query ? 0 : q_tasks)) * HEADS + lane / LPR;
  const int hc = min(h, heads - 1);  // lanes past the last head repeat it and write nothing
  const uint16_t *const cos = a.cos.p + b * a.cos.sb + t * a.cos.st, *const sin = a.sin.p + b * a.sin.sb + t * a.sin.st;
  NormRopeRow<LPR> row;
  float y[8];
  if (query) {
    // Rounded once, from fp32 to bf16.
    row.load(a.q.p + b * a.q.sb + hc * a.q.sh + t * a.q.st, a.q_weight, cos, sin, a.R, c);
    row.template compute<float>(a.eps, a.offset, y);
    if (h < heads)
      store16(a.q_out + (((int64_t)b * a.Hq + h) * a.T + t) * (8 * LPR) + 8 * c,
              u32x4{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]), pack_bf16x2(y[6], y[7])});
  } else {
    const int64_t slot = scalar_load(a.slots, b * a.slot_sb + t * a.slot_st);
    if (!kv4_holds(a.cache, slot)) return;
    float v[8];
    unpack_floats(load16(a.v.p + b * a.v.sb + hc * a.v.sh + t * a.v.st + 8 * c), v);
    const uint16_t *key = a.k.p + b * a.k.sb + hc * a.k.sh + t * a.k.st;
    row.load(key, a.k_weight, cos, sin, a.R, c);
    row.template compute<float>(a.eps, a.offset, y);
    // The codes are those of the definition: a wave with a value near a border (under one in a hundred) reads and
    // computes its rows again in 64 bits.
    if (__builtin_expect(__any(near_border<LPR>(y)), 0)) {
      asm volatile("" : "+v"(key));  // not kept in registers for this
      row.load(key, a.k_weight, cos, sin, a.R, c);
      row.template compute<double>(a.eps, a.offset, y);
    }
    kv4_store<LPR>(a.cache, slot, h, c, y, v, h < heads);
  }
}

#define XATTN_BY_DIM(D, launch)      \
  switch (D) {                       \
    case 64: launch(8); break;       \
    case 128: launch(16); break;     \
    default: launch(32); break;      \
  }

hipError_t launch_append_kv4(const Kv4AppendArgs &a, hipStream_t stream) {
  const int64_t rows = (int64_t)a.B * a.T * a.cache.Hkv;
#define LAUNCH(LPR) \
  hipLaunchKernelGGL((append_kv4_kernel<LPR>), dim3((rows + 256 / LPR - 1) / (256 / LPR)), dim3(256), 0, stream, a)
  XATTN_BY_DIM(a.cache.D, LAUNCH)
#undef LAUNCH
  return hipGetLastError();
}

hipError_t launch_read_kv4(const Kv4ReadArgs &a, hipStream_t stream) {
  const int64_t rows = (int64_t)a.B * a.T * a.cache.Hkv;
#define LAUNCH(LPR) \
  hipLaunchKernelGGL((read_kv4_kernel<LPR>), dim3((rows + 256 / LPR - 1) / (256 / LPR)), dim3(256), 0, stream, a)
  XATTN_BY_DIM(a.cache.D, LAUNCH)
#undef LAUNCH
  return hipGetLastError();
}

hipError_t launch_norm_rope_kv4(const Kv4NormRopeArgs &a, hipStream_t stream) {
#define LAUNCH(LPR)                                                                                          \
  {                                                                                                          \
    constexpr int HEADS = 64 / LPR;                                                                          \
    const int64_t waves = (int64_t)a.B * a.T * ((a.Hq + HEADS - 1) / HEADS + (a.cache.Hkv + HEADS - 1) / HEADS); \
    hipLaunchKernelGGL((norm_rope_kv4_kernel<LPR>), dim3((waves + 3) / 4), dim3(256), 0, stream, a);         \
  }
  XATTN_BY_DIM(a.cache.D, LAUNCH)
#undef LAUNCH
  return hipGetLastError();
}

}  // namespace xattn
