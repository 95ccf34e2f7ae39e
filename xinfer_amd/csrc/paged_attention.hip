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
  if (paged_item(a, paged_lane_row(a, 0), blockIdx.x, it)) paged_decode_item<D, NC, WAVES>(a, blockIdx.x, it, smem);
}

template <int D>
__device__ __forceinline__ void paged_prefill_item(const PagedArgs &a, int index, const PagedItem &it, char *smem) {
  if constexpr (D == 256) paged_chunk_item_wide<D>(a, index, it, smem);
  else paged_chunk_item<D>(a, index, it, smem);
}

// Prefill items first, the much shorter decode items behind them, where they fill what the last prefill items leave idle,
// then the blocks without an item.  (A batch of 5 chunks and 3 single tokens, 256 features: 432 us, with the decode
// items first 447; 395 now.)
template <int D>
__global__ void __launch_bounds__(64 * kPagedChunkWaves, 2) paged_both_kernel(const PagedArgs few, const PagedArgs many) {
  constexpr int WAVES = kPagedChunkWaves, CHUNK = kPagedChunkLds<D>, DECODE = kPagedDecodeLds<D, WAVES>;
  __shared__ __attribute__((aligned(1024))) char smem[CHUNK > DECODE ? CHUNK : DECODE];
  PagedItem it;
  int index = blockIdx.x;
  const PagedRow lane_row = paged_lane_row(many, 0);
  if (paged_item(many, lane_row, index, it)) {
    paged_prefill_item<D>(many, index, it, smem);
  } else {
    index -= it.begin;
    if (paged_item(few, lane_row, index, it)) paged_decode_item<D, paged_decode_columns(D) / 16, WAVES>(few, index, it, smem);
  }
}

// Prefill items alone.
template <int D>
__global__ void __launch_bounds__(64 * kPagedChunkWaves, 2) paged_prefill_kernel(const PagedArgs a) {
  __shared__ __attribute__((aligned(1024))) char smem[kPagedChunkLds<D>];
  PagedItem it;
  if (paged_item(a, paged_lane_row(a, 0), blockIdx.x, it)) paged_prefill_item<D>(a, blockIdx.x, it, smem);
}

// The running maximum, sum and output (four features) of records read so far.
struct MergedRuns {
  float best, total;
  f32x4 out;
  __device__ __forceinline__ void add(float m, float l, const f32x4 &part) {
    const float now = fmaxf(best, m), old = fast_exp2(best - now), keep = fast_exp2(m - now);
    best = now;
    total = total * old + l * keep;
    out = out * old + part * keep;
  }
};

// Runs begin, begin + stride, ... of N vectors, the first at record `at`, the others TEAMS apart (or at `spare`, if nearer).
// The records of four runs are read together.
template <int D, int N>
__device__ __forceinline__ void merge_runs(const PagedArgs &a, int64_t at, int spare, int64_t step, int begin, int stride,
                                           int nsplit, int f, MergedRuns (&r)[N]) {
  constexpr int TEAMS = kMergeThreads / (D / 4);
#pragma unroll
  for (int n = 0; n < N; ++n) r[n] = MergedRuns{kLowest, 0.0f, f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
  for (int s0 = begin; s0 < nsplit; s0 += 4 * stride) {
    f32x2 ml[N][4];
    f32x4 part[N][4];
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t record = at + min(n * TEAMS, spare) + min(s0 + e * stride, nsplit - 1) * step;
        ml[n][e] = *as_global(reinterpret_cast<const f32x2 *>(a.part_ml + 2 * record));
        part[n][e] = *as_global(reinterpret_cast<const f32x4 *>(a.part_o + record * D + 4 * f));
      }
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (s0 + e * stride < nsplit) r[n].add(ml[n][e].x, ml[n][e].y, part[n][e]);
  }
}

// Joins the runs of rows that were cut, of either launch.  D/4 threads side by side take a query vector, 4 features
// each; a block has 256 / (D/4) such teams.  Decode rows (blocks below few_blocks, the row counting slowest) have few
// vectors and many runs: a block takes one vector, its teams every TEAMS-th run, and joins them in LDS.  Prefill rows
// have many vectors of few runs: a team takes kMergeVectors of them, N at a time.  N = 4 waits for memory once but leaves
// three blocks a CU, which pays in a launch of prefill rows alone (512 vectors a head of one row, 4 runs: 6.3 us, with
// N = 1 7.6) and costs in the others, whose blocks without work are many (64 single tokens: 6.2 us, with N = 1 4.8).
template <int D, int N>
__global__ void __launch_bounds__(kMergeThreads) paged_merge_kernel(const PagedArgs few, const PagedArgs many, int few_blocks,
                                                          int few_per_row, int many_per_row) {
  constexpr int TEAMS = kMergeThreads / (D / 4);
  __shared__ f32x4 outs[TEAMS][D / 4];
  __shared__ f32x2 sums[TEAMS];
  const bool together = (int)blockIdx.x < few_blocks;
  const PagedArgs &a = together ? few : many;
  const uint32_t at = together ? blockIdx.x : blockIdx.x - few_blocks, per_row = together ? few_per_row : many_per_row;
  const uint32_t row = at / per_row, in_row = at - row * per_row;
  const uint32_t per = together ? min(a.tile, a.T * a.G) : (a.tile + TEAMS * kMergeVectors - 1) / (TEAMS * kMergeVectors);
  const uint32_t unit = in_row / per, first = in_row - unit * per;
  const int tile = unit / a.cache.Hkv, h = unit - tile * a.cache.Hkv;
  PagedItem it;
  paged_row_items(a, row, it);
  if (it.nsplit <= 1 || tile >= it.tiles) return;
  const int team = threadIdx.x / (D / 4), f = threadIdx.x % (D / 4);
  const int vectors = min(it.count * a.G - tile * a.tile, a.tile);
  if (together && (int)first >= vectors) return;
  const int64_t step = (int64_t)a.cache.Hkv * a.tile;
  const int64_t record0 = ((int64_t)it.begin + (int64_t)tile * it.nsplit * a.cache.Hkv + h) * a.tile;
  auto finish = [&](const MergedRuns &r, int column) {
    const int j = tile * a.tile + column, t = j / a.G;
    const f32x4 out = r.out * (r.total == 0.0f ? 0.0f : 1.0f / r.total);
    *as_global(reinterpret_cast<u32x2 *>(
        a.out + (((int64_t)row * a.T + t) * a.Hq + h * a.G + (j - t * a.G)) * D + 4 * f)) =
        u32x2{pack_bf16x2(out[0], out[1]), pack_bf16x2(out[2], out[3])};
  };
  if (together) {
    MergedRuns r[1];
    merge_runs<D, 1>(a, record0 + first, 0, step, team, TEAMS, it.nsplit, f, r);
    outs[team][f] = r[0].out;
    if (f == 0) sums[team] = f32x2{r[0].best, r[0].total};
    __syncthreads();
    if (team != 0) return;
#pragma unroll
    for (int e = 1; e < TEAMS; ++e) r[0].add(sums[e].x, sums[e].y, outs[e][f]);
    finish(r[0], first);
  } else {
    for (int n0 = 0; n0 < kMergeVectors; n0 += N) {
      // Vectors past the row's last are read as the last of the team.
      const int column = (first * kMergeVectors + n0) * TEAMS + team, spare = vectors - 1 - column;
      if (spare < 0) return;
      MergedRuns r[N];
      merge_runs<D, N>(a, record0 + column, spare, step, 0, 1, it.nsplit, f, r);
#pragma unroll
      for (int n = 0; n < N; ++n)
        if (n * TEAMS <= spare) finish(r[n], column + n * TEAMS);
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
    auto merge = l.few.items == 0 ? paged_merge_kernel<D, kMergeVectors> : paged_merge_kernel<D, 1>;
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
