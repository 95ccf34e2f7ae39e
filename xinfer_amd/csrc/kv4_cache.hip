// Writing and reading the paged 4-bit KV cache (format: kv4_common.h): the append, the query/key norm and rotation
// with the append in one launch, and the read-back.
//
// A row is a (token, head); LPR = D/8 lanes hold it, 8 features each, so a block's largest magnitude is one
// exchange among four lanes.  A lane takes the same features of the token's key and of its value, because a token
// is stored as not finite if either is.
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
// y_i cos_i - y_{i + R/2} sin_i and the second to y_i cos_i + y_{i - R/2} sin_i.  A query is rounded once, from fp32 to
// bf16.  A key goes to its codes, where a value next to a border changes by a whole step of the grid: it is computed in
// 64 bits, so that the codes are those of the definition.  The rotation's other half is read from memory again (a line
// this wave reads anyway) and normalised here, which takes no exchange between lanes.
__device__ __forceinline__ double wide_shuffle(double x, int mask) {
  return __hiloint2double(__shfl_xor(__double2hiint(x), mask), __shfl_xor(__double2loint(x), mask));
}
template <int LPR, typename F>
__device__ __forceinline__ void norm_rope_row(const uint16_t *x, const uint16_t *weight, const uint16_t *cos,
                                              const uint16_t *sin, float eps, float offset, int R, int c,
                                              float (&y)[8]) {
  const int half = R / 16;  // chunks of half the rotated features
  const bool turned = c < 2 * half;
  const int other = c < half ? c + half : (turned ? c - half : c);
  float x0[8], x1[8], w[8], wo[8], cs[8], sn[8];
  unpack_floats(load16(x + 8 * c), x0);
  unpack_floats(load16(x + 8 * other), x1);
  unpack_floats(load16(weight + 8 * c), w);
  unpack_floats(load16(weight + 8 * other), wo);
  unpack_floats(load16(cos + 8 * (turned ? c : 0)), cs);
  unpack_floats(load16(sin + 8 * (turned ? c : 0)), sn);
  F ss = 0, inv;
#pragma unroll
  for (int e = 0; e < 8; ++e) ss += (F)(x0[e] * x0[e]);  // x^2 is exact in fp32
  if constexpr (sizeof(F) == 8) {
#pragma unroll
    for (int mask = 1; mask < LPR; mask *= 2) ss += wide_shuffle(ss, mask);
    const F mean = ss * (F)(1.0 / (8 * LPR)) + (F)eps;
    inv = (F)rsqrtf((float)mean);
    // Newton's step on the fp32 root: 2^-22 squares to 2^-44.  Where that root overflows, so does the definition's.
    inv = mean > (F)0 && isfinite((float)inv) ? inv * (1.5 - 0.5 * mean * inv * inv) : inv;
  } else {
    inv = rsqrtf(group_sum<LPR>(ss) * (F)(1.0f / (8 * LPR)) + eps);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const F a = (F)x0[e] * inv * ((F)w[e] + (F)offset), b = (F)x1[e] * inv * ((F)wo[e] + (F)offset);
    y[e] = (float)(turned ? a * (F)cs[e] + (c < half ? -b : b) * (F)sn[e] : a);
  }
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
  float y[8];
  if (query) {
    norm_rope_row<LPR, float>(a.q.p + b * a.q.sb + hc * a.q.sh + t * a.q.st, a.q_weight, cos, sin, a.eps, a.offset, a.R, c, y);
    if (h < heads)
      store16(a.q_out + (((int64_t)b * a.Hq + h) * a.T + t) * (8 * LPR) + 8 * c,
              u32x4{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]), pack_bf16x2(y[6], y[7])});
  } else {
    const int64_t slot = scalar_load(a.slots, b * a.slot_sb + t * a.slot_st);
    if (!kv4_holds(a.cache, slot)) return;
    float v[8];
    unpack_floats(load16(a.v.p + b * a.v.sb + hc * a.v.sh + t * a.v.st + 8 * c), v);
    norm_rope_row<LPR, double>(a.k.p + b * a.k.sb + hc * a.k.sh + t * a.k.st, a.k_weight, cos, sin, a.eps, a.offset, a.R, c, y);
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
