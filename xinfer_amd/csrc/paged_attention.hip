// Attention over the paged 4-bit KV cache (format: kv4_common.h), in its simplest form: a wave takes one query
// vector, a lane one key of 64 for the scores, and then D/64 features for the output.  One pass over the keys with
// the running maximum and sum of the softmax, in fp32.
#include "kv4_device.h"
#include "launch.h"

namespace xattn {

template <int D>
__global__ void __launch_bounds__(64) paged_attention_kernel(const PagedArgs a) {
  constexpr int F = D / 64;
  const int lane = threadIdx.x, t = blockIdx.x, head = blockIdx.y, b = blockIdx.z;
  const int count = min(max(a.lengths[b], 0), min(a.T, a.max_length)), length = min(max(a.lengths[a.B + b], count), a.max_length);
  uint16_t *const out = a.out + (((int64_t)b * a.T + t) * a.Hq + head) * D;
  const int h = head / a.G, keys = t < count ? length - count + t + 1 : 0;
  const int shift = a.cache.page_shift, size = 1 << shift;
  __shared__ float q[D];
  const uint16_t *const qp = a.q.p + b * a.q.sb + head * a.q.sh + t * a.q.st;
  for (int d = lane; d < D; d += 64) q[d] = __uint_as_float((uint32_t)qp[d] << 16) * a.scale_log2;
  __syncthreads();
  float m = -INFINITY, l = 0.0f, o[F] = {};
  for (int first = 0; first < keys; first += 64) {
    const int page = a.table[(int64_t)b * a.width + (first >> shift)];
    if (page < 0 || page >= a.cache.pages) continue;
    const int64_t base = (int64_t)page * a.cache.Hkv + h;
    const int at = first & (size - 1), key = at + lane;
    const uint8_t *const codes = a.cache.key + (base * size + key) * (D / 2);
    float s = 0.0f;
    for (int block = 0; block < D / 32; ++block) {
      const int scale = a.cache.key_scale[(base * (D / 32) + block) * size + key];
      float sum = 0.0f;
      for (int w = 0; w < 4; ++w) {
        float x[8];
        unpack_floats(kv4_values(reinterpret_cast<const uint32_t *>(codes)[block * 4 + w], 1.0f), x);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fmaf(x[e], q[32 * block + 8 * w + e], sum);
      }
      s += scale == kKv4NanScale ? __uint_as_float(0x7fc00000u) : sum * kv4_scale_value(scale);
    }
    if (first + lane >= keys) s = -INFINITY;
    float top = s;
    for (int x = 32; x > 0; x /= 2) {
      const float other = __shfl_xor(top, x);
      top = top > other || top != top ? top : other;
    }
    const float now = fmaxf(m, top), old = exp2f(m - now), p = exp2f(s - now);
    m = now;
    l = l * old + group_sum<64>(p);
#pragma unroll
    for (int f = 0; f < F; ++f) o[f] *= old;
    for (int j = 0; j < min(64, keys - first); ++j) {
      const float pj = __shfl(p, j);
      const uint8_t *const v = a.cache.value + (base * size + at + j) * (D / 2);
#pragma unroll
      for (int f = 0; f < F; ++f) {
        const int d = lane + 64 * f;
        const int scale = min((int)a.cache.value_scale[(base * (D / 32) + d / 32) * size + at + j], kKv4MaxScale);
        const uint32_t code = (uint32_t)(v[d / 2] >> (4 * (d & 1))) & 15u;
        o[f] = fmaf(pj, bf16_lo(kv4_values(code, kv4_scale_value(scale))[0]), o[f]);
      }
    }
  }
#pragma unroll
  for (int f = 0; f < F; ++f) out[lane + 64 * f] = (uint16_t)f32_to_bf16_bits(l == 0.0f ? 0.0f : o[f] / l);
}

hipError_t launch_paged_attention(const PagedArgs &a, hipStream_t stream) {
  const dim3 grid(a.T, a.Hq, a.B);
  switch (a.cache.D) {
    case 64: hipLaunchKernelGGL((paged_attention_kernel<64>), grid, dim3(64), 0, stream, a); break;
    case 128: hipLaunchKernelGGL((paged_attention_kernel<128>), grid, dim3(64), 0, stream, a); break;
    default: hipLaunchKernelGGL((paged_attention_kernel<256>), grid, dim3(64), 0, stream, a); break;
  }
  return hipGetLastError();
}

}  // namespace xattn
