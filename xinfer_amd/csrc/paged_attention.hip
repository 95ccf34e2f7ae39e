// Kernels of attention over the paged 4-bit cache: rows of few query vectors a KV head (paged_decode.h), rows of many
// (paged_prefill.h), both in one launch for batches that may hold both, and the merge of rows cut into runs.
#include "paged_prefill.h"
#include "launch.h"

namespace xattn {

// Occupancy: one column group of up to 128 features fits 128 registers (four waves a SIMD), the others twice that.
template <int D, int NC, int WAVES>
__global__ void __launch_bounds__(64 * WAVES, D == 256 || NC == 2 ? 2 : 4) paged_decode_kernel(const PagedArgs a) {
  __shared__ __attribute__((aligned(1024))) char smem[kPagedDecodeLds<D, WAVES>];
  PagedItem it;
  int index = blockIdx.x;
  if (paged_item(a, paged_lane_row(a, 0), index, it)) paged_decode_item<D, NC, WAVES>(a, it, smem);
}

template <int D>
__device__ __forceinline__ void paged_prefill_item(const PagedArgs &a, const PagedItem &it, char *smem) {
  if constexpr (D == 256) paged_chunk_item_wide<D>(a, it, smem);
  else paged_chunk_item<D>(a, it, smem);
}

// Prefill items first, the much shorter decode items behind them, where they fill what the last prefill items leave idle,
// then the blocks without an item.  (A batch of 5 chunks and 3 single tokens, 256 features: 432 us, with the decode
// items first 447; 368 now.)
template <int D>
__global__ void __launch_bounds__(64 * kPagedChunkWaves, 2) paged_both_kernel(const PagedArgs few, const PagedArgs many) {
  constexpr int WAVES = kPagedChunkWaves, CHUNK = kPagedChunkLds<D>, DECODE = kPagedDecodeLds<D, WAVES>;
  __shared__ __attribute__((aligned(1024))) char smem[CHUNK > DECODE ? CHUNK : DECODE];
  PagedItem it;
  int index = blockIdx.x;
  const PagedRow lane_row = paged_lane_row(many, 0);
  if (paged_item(many, lane_row, index, it)) {
    paged_prefill_item<D>(many, it, smem);
  } else if (paged_item(few, lane_row, index, it)) {
    paged_decode_item<D, paged_decode_columns(D) / 16, WAVES>(few, it, smem);
  }
}

// Prefill items alone.
template <int D>
__global__ void __launch_bounds__(64 * kPagedChunkWaves, 2) paged_prefill_kernel(const PagedArgs a) {
  __shared__ __attribute__((aligned(1024))) char smem[kPagedChunkLds<D>];
  PagedItem it;
  int index = blockIdx.x;
  if (paged_item(a, paged_lane_row(a, 0), index, it)) paged_prefill_item<D>(a, it, smem);
}

// The running maximum, sum and output (N times four features) of a vector's runs so far.
template <int N>
struct MergedRuns {
  float best, total;
  f32x4 out[N];
  __device__ __forceinline__ MergedRuns() : best(kLowest), total(0.0f) {
#pragma unroll
    for (int n = 0; n < N; ++n) out[n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  __device__ __forceinline__ void add(float m, float l, const f32x4 (&part)[N]) {
    const float now = fmaxf(best, m), old = fast_exp2(best - now), keep = fast_exp2(m - now);
    best = now;
    total = total * old + l * keep;
#pragma unroll
    for (int n = 0; n < N; ++n) out[n] = out[n] * old + part[n] * keep;
  }
  // Runs begin, begin + stride, ...: the first run's record at ml and o, the runs ml_step and o_step apart, quad n of a
  // record at quad * n.  Four runs are read together.
  __device__ __forceinline__ void read(const float *ml, const float *o, int64_t ml_step, int64_t o_step, int64_t quad,
                                       int begin, int stride, int nsplit) {
    for (int s0 = begin; s0 < nsplit; s0 += 4 * stride) {
      f32x2 x[4];
      f32x4 part[4][N];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t s = min(s0 + e * stride, nsplit - 1);
        x[e] = *as_global(reinterpret_cast<const f32x2 *>(ml + s * ml_step));
#pragma unroll
        for (int n = 0; n < N; ++n) part[e][n] = *as_global(reinterpret_cast<const f32x4 *>(o + s * o_step + quad * n));
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (s0 + e * stride < nsplit) add(x[e].x, x[e].y, part[e]);
    }
  }
};

// Joins the runs of rows that were cut, of either launch.  Decode rows (blocks below few_blocks, the row counting slowest)
// have few vectors and many runs: a block takes one vector, D/4 threads side by side four features each, its 256 / (D/4)
// teams every TEAMS-th run, and joins them in LDS.  Prefill rows have many vectors of few runs: threads side by side take
// vectors side by side, kMergeQuads quads of features each, N at a time, so records are read in runs of 256 bytes and more.
// N = 2 leaves eight blocks a CU, for launches with many blocks without work (64 single tokens: 4.9 us, with three blocks a
// CU 6.2; 92 MB of records of 5 chunks 18.8 us); N = 4 waits for memory once, for prefill rows alone (512 tokens of one
// row, 17 MB of records: 5.6 us, a vector a team 7.6).
template <int D, int N>
__global__ void __launch_bounds__(kMergeThreads) paged_merge_kernel(const PagedArgs few, const PagedArgs many, int few_blocks,
                                                                    int few_per_row, int many_per_row) {
  constexpr int TEAMS = kMergeThreads / (D / 4), VECTORS = 4 * kMergeThreads * kMergeQuads / D;
  __shared__ f32x4 outs[TEAMS][D / 4];
  __shared__ f32x2 sums[TEAMS];
  const bool together = (int)blockIdx.x < few_blocks;
  const PagedArgs &a = together ? few : many;
  const uint32_t at = together ? blockIdx.x : blockIdx.x - few_blocks, per_row = together ? few_per_row : many_per_row;
  const uint32_t row = at / per_row, in_row = at - row * per_row;
  const uint32_t per = together ? min(a.tile, a.T * a.G) : (a.tile + VECTORS - 1) / VECTORS;
  const uint32_t unit = in_row / per, first = in_row - unit * per;
  const int tile = unit / a.cache.Hkv, h = unit - tile * a.cache.Hkv;
  PagedItem it;
  paged_row_items(a, row, it);
  if (it.nsplit <= 1 || tile >= it.tiles) return;
  const int vectors = min(it.count * a.G - tile * a.tile, a.tile);
  const int64_t item = (int64_t)it.record + (int64_t)tile * it.nsplit * a.cache.Hkv + h;
  const int64_t ml_step = 2 * (int64_t)a.cache.Hkv * a.tile, o_step = (int64_t)a.cache.Hkv * a.tile * D;
  // Output of four features from 4 f on.
  auto finish = [&](int column, int f, const f32x4 &sum, float total) {
    const int j = tile * a.tile + column, t = j / a.G;
    const f32x4 out = sum * (total == 0.0f ? 0.0f : 1.0f / total);
    *as_global(reinterpret_cast<u32x2 *>(
        a.out + (((int64_t)row * a.T + t) * a.Hq + h * a.G + (j - t * a.G)) * D + 4 * f)) =
        u32x2{pack_bf16x2(out[0], out[1]), pack_bf16x2(out[2], out[3])};
  };
  if (together) {
    if ((int)first >= vectors) return;
    const int team = threadIdx.x / (D / 4), f = threadIdx.x % (D / 4);
    const int64_t record = item * a.tile + first;
    MergedRuns<1> r;
    r.read(a.part_ml + 2 * record, a.part_o + record * D + 4 * f, ml_step, o_step, 0, team, TEAMS, it.nsplit);
    outs[team][f] = r.out[0];
    if (f == 0) sums[team] = f32x2{r.best, r.total};
    __syncthreads();
    if (team != 0) return;
#pragma unroll
    for (int e = 1; e < TEAMS; ++e) r.add(sums[e].x, sums[e].y, {outs[e][f]});
    finish(first, f, r.out[0], r.total);
  } else {
    const int column = first * VECTORS + threadIdx.x % VECTORS, f = kMergeQuads * (threadIdx.x / VECTORS);
    if (column >= vectors) return;
    const float *const o = a.part_o + 4 * ((item * (D / 4) + f) * a.tile + column);
    for (int n0 = 0; n0 < kMergeQuads; n0 += N) {
      MergedRuns<N> r;
      r.read(a.part_ml + 2 * (item * a.tile + column), o + (int64_t)4 * n0 * a.tile, ml_step, o_step, 4 * a.tile, 0, 1, it.nsplit);
#pragma unroll
      for (int n = 0; n < N; ++n) finish(column, f + n0 + n, r.out[n], r.total);
    }
  }
}

template <int D, int NC, int WAVES>
static void launch_decode(const PagedLaunch &l, hipStream_t stream) {
  hipLaunchKernelGGL((paged_decode_kernel<D, NC, WAVES>), dim3(l.items), dim3(64 * WAVES), 0, stream, l.a);
}

template <int D>
static hipError_t launch_d(const PagedLaunches &l, hipStream_t stream) {
  const dim3 block(64 * kPagedChunkWaves);
  const PagedArgs &few = l.few.a, &many = l.many.a;
  if (l.few.items > 0 && l.many.items > 0) {
    hipLaunchKernelGGL((paged_both_kernel<D>), dim3(l.few.items + l.many.items), block, 0, stream, few, many);
  } else if (l.many.items > 0) {
    hipLaunchKernelGGL((paged_prefill_kernel<D>), dim3(l.many.items), block, 0, stream, many);
  } else if (few.tile == 32) {
    if constexpr (paged_decode_columns(D) == 32) launch_decode<D, 2, 8>(l.few, stream);
  } else if (l.few.waves == kPagedRowWaves) {
    if constexpr (D < 256) launch_decode<D, 1, kPagedRowWaves>(l.few, stream);
  } else {
    launch_decode<D, 1, 4>(l.few, stream);
  }
  if (l.bytes() > 0) {
    const int rows = few.B, few_per_row = (int)l.few_merges(), many_per_row = (int)l.many_merges();
    auto merge = l.few.items == 0 ? paged_merge_kernel<D, kMergeQuads> : paged_merge_kernel<D, 2>;
    hipLaunchKernelGGL(merge, dim3((unsigned)rows * (few_per_row + many_per_row)), dim3(kMergeThreads), 0, stream, few, many,
                       rows * few_per_row, few_per_row, many_per_row);
  }
  return hipGetLastError();
}

hipError_t launch_paged_attention(const PagedLaunches &l, hipStream_t stream) {
  switch (l.few.a.cache.D) {
    case 64: return launch_d<64>(l, stream);
    case 128: return launch_d<128>(l, stream);
    default: return launch_d<256>(l, stream);
  }
}

}  // namespace xattn
