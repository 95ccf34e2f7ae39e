// Attention over the paged 4-bit cache for rows of many query vectors a KV head: prompt chunks.
//
// A block takes an item (paged_plan.h): 128 query vectors of a (row, KV head) over a run of keys in 64-key groups.  Up to
// 128 features each half of its 8 waves takes all of them, 32 a wave, over every other group (paged_chunk_item).  A wave
// reads the group's keys as they lie in the cache, as the A operand of the scaled 32x32x64 product against its queries'
// two e4m3 terms (paged_mfma.h): row m of tile t (of two) is key 2 m + t, so a lane's two keys have their scales in
// neighbouring bytes.  A lane (column q, half h) then holds 32 scores of its query, and for each 16 keys 8 neighbouring
// ones, which is the B operand of the bf16 PV product: nothing of the softmax crosses lanes but the maximum and, at the
// end, the sum of the two halves.
//
// The waves of a group turn its values into bf16 (exact) in LDS together, a group ahead, and each reads them transposed
// as the A operand.  One barrier a round.
//
// 256 features of 32 vectors would take 128 registers for the output and 64 for the queries, which leaves no two
// waves a SIMD.  There 8 waves take 16 vectors each (paged_chunk_item_wide), with the products and layouts of the
// decode kernel (paged_decode.h) but values staged by the whole block.
//
// Weights are rounded to bf16 (2^-8 of a weight at most, on average lost in the sum).  Their sum is taken before it, with
// 256 features after it, a group's by half as many instructions (5 chunks and 3 single tokens: 411 us, 428 with the
// sum before; with 128 features it makes no difference).
//
// What bounds it: matrix and vector unit share a SIMD's issue, and two waves hide little more.  512 tokens in each of 8 rows
// of 8192 keys, page size 64: 16 / 8 heads of 128 features 0.28 to 0.29 ms (920 to 960 TFLOP/s; the matrix units work 47 %
// of the time, the vector units 57 %, a quarter of that exponentials), 32 / 8 heads 0.51 to 0.54 (990 to 1040), 16 / 4 heads
// of 256 features 0.50 to 0.52 (1020 to 1060; 46 and 43 %, LDS 36 %, and waits for it and the block's barrier).  One row
// of 512 tokens and 2048 keys, 16 / 8 heads: 29 to 30 us with the merge, of which the rounds are 10, the way to the first
// (plan, queries, first keys) 5, the records 3 to write and 5 to merge; 64 tiles fill a quarter of the CUs, so it has to be
// cut.
#pragma once

#include "paged_decode.h"

namespace xattn {

constexpr int kPagedChunkWaves = 8;  // of a prefill block
constexpr int kChunkWaves = kPagedChunkWaves / 2, kChunkThreads = 64 * kChunkWaves;  // of half a block

template <int D>
struct ChunkShape {
  static constexpr int KS = D / 64;                                  // 64-feature steps of the scores
  static constexpr int DT = D / 32;                                  // 32-feature tiles of the output
  static constexpr int ROW = 2 * D, STAGE = 64 * ROW;                // staged values of a group
  static constexpr int UNITS = 64 * (D / 32);                        // (key, block) units of a group
};

// Slot of 16-byte chunk c of staged row r: c ^ S(r), with 128 features c ^ S(r) ^ 2 (c / 8).  LDS serves 128 bytes a clock.
// What one takes of a transposing read are two neighbouring chunks of four rows, of a store chunks 4 b + const. of two rows'
// four blocks (64 features: four rows' two blocks); either lies in eight different slots modulo eight.
template <int D>
__device__ __forceinline__ int chunk_swizzle(int r) {
  return D == 64 ? 5 * (r & 1) ^ (r & 2) : 5 * (r & 3);
}

template <bool B>
struct Flag {
  static constexpr bool value = B;
};

// The block's barrier for what its waves have stored in LDS.  Loads from memory stay under way (__syncthreads would wait
// for them, and with that for a memory round trip every group).
__device__ __forceinline__ void staged_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory"); }

// LDS of a prefill block: staged groups, two for each half of the waves, and the queries' terms and scales, later the
// second half's maxima and sums (256 features: three groups for all waves).
template <int D>
constexpr int kPagedChunkLds = D == 256 ? 3 * (64 * 2 * D + 65 * (D / 2)) : 4 * 64 * 2 * D + kPagedPrefillTile * (2 * D + D / 32);

// Item `it` of the plan, by the whole block; smem: kPagedChunkLds bytes, 1024-byte aligned.
template <int D>
__device__ __forceinline__ void paged_chunk_item(const PagedArgs &a, const PagedItem &it, char *smem) {
  using S = ChunkShape<D>;
  constexpr int COLS = 32 * kChunkWaves;
  const int tid = threadIdx.x & (kChunkThreads - 1), lane = tid & 63, m = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int side = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kChunkThreads);  // which groups: every other one
  paged_zero_padded<D, 2 * kChunkThreads>(a, it);

  // This wave's queries.
  const int vectors = it.count * a.G, j = it.tile * COLS + 32 * wave + m;
  const int t = j / a.G, head = it.h * a.G + (j - t * a.G);
  const bool there = j < vectors;
  const int last_key = there ? it.length - it.count + t : -1;
  const int wave_first = it.tile * COLS + 32 * wave;
  const int all_see = it.length - it.count + wave_first / a.G;  // all of the wave's queries see keys up to this one,
  const int none_see = wave_first < vectors                     // and none of them this one or a later
                           ? it.length - it.count + (min(wave_first + 32, vectors) - 1) / a.G + 1 : 0;
  const int tile_end = it.length - it.count + (min(it.tile * COLS + COLS, vectors) - 1) / a.G + 1;
  const int group_end = min(it.group_end, (tile_end + kGroupKeys - 1) / kGroupKeys);

  // The block's queries are read row by row, 8 features a lane, turned into their terms once for both halves and
  // passed through LDS; each wave reading its own would touch a line for every 16 or 32 bytes, and twice.
  // 16-byte chunk c of vector v's terms lies at c ^ v.
  constexpr int LANES = D / 8, LOADS = COLS * LANES / (2 * kChunkThreads), SPREAD = D / 16 - 1;
  char *const terms = smem + 4 * S::STAGE;
  uint8_t *const scales = reinterpret_cast<uint8_t *>(terms + 2 * COLS * D);
  const int load_first = threadIdx.x / LANES, load_chunk = threadIdx.x % LANES;
  u32x4 first[S::KS][2], second[S::KS][2], qx[LOADS];
  int qscale[S::KS];
#pragma unroll
  for (int n = 0; n < LOADS; ++n) {
    const int i = it.tile * COLS + load_first + n * (COLS / LOADS), token = i / a.G;
    const uint16_t *const q = a.q.p + it.row * a.q.sb + (it.h * a.G + (i - token * a.G)) * a.q.sh + token * a.q.st;
    qx[n] = i < vectors ? load16(q + 8 * load_chunk) : u32x4{0, 0, 0, 0};
  }
  auto convert_queries = [&]() {
#pragma unroll
    for (int n = 0; n < LOADS; ++n) {
      const int i = load_first + n * (COLS / LOADS), scale = query_scale(quad_max(largest(qx[n], 0u)));
      u32x2 x, rest;
      split_query(qx[n], scale, x, rest);
      char *const to = terms + i * D + ((load_chunk >> 1) ^ (i & SPREAD)) * 16 + 8 * (load_chunk & 1);
      *reinterpret_cast<u32x2 *>(to) = x;
      *reinterpret_cast<u32x2 *>(to + COLS * D) = rest;
      if (load_chunk % 4 == 0) scales[i * (D / 32) + load_chunk / 4] = (uint8_t)scale;
    }
    staged_barrier();
    const int i = 32 * wave + m;
#pragma unroll
    for (int s = 0; s < S::KS; ++s) {
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const char *const from = terms + i * D + ((4 * s + 2 * p + h) ^ (i & SPREAD)) * 16;
        first[s][p] = *reinterpret_cast<const u32x4 *>(from);
        second[s][p] = *reinterpret_cast<const u32x4 *>(from + COLS * D);
      }
      const int mine = scales[i * (D / 32) + 2 * s + h];
      qscale[s] = mine | (mine == 255 ? 255 : mine - 4) << 8;
    }
  };

  f32x16 o[S::DT];
#pragma unroll
  for (int d = 0; d < S::DT; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = 0.0f;
  float top = kLowest, sum = 0.0f;

  const int shift = a.cache.page_shift - 6, size = 1 << a.cache.page_shift;
  typedef const __attribute__((address_space(4))) int32_t *table_ptr;
  const table_ptr table = (table_ptr)(a.table + (int64_t)it.row * a.width);
  auto page_of = [&](int group) {
    const int page = group < group_end ? table[group >> shift] : -1;
    return page >= 0 && page < a.cache.pages ? page : -1;
  };
  auto place = [&](int group) { return (group & ((1 << shift) - 1)) * kGroupKeys; };

  // Keys of a group: lane (m, h) holds keys 2 m + t, blocks 2 s + h.
  u32x4 k[2][S::KS];
  uint32_t ks[S::KS];
  uint32_t key_at = 2 * m * (D / 2) + 16 * h, key_scale_at = h * size + 2 * m;
  auto load_keys = [&](int group, int page) {
    const int64_t hd = (int64_t)max(page, 0) * a.cache.Hkv + it.h;
    const uint8_t *const codes = a.cache.key + (hd * size + place(group)) * (D / 2);
    const uint8_t *const scales = a.cache.key_scale + hd * (D / 32) * size + place(group);
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int s = 0; s < S::KS; ++s)
        k[x][s] = *as_global(reinterpret_cast<const u32x4 *>(codes + x * (D / 2) + 32 * s + key_at));
#pragma unroll
    for (int s = 0; s < S::KS; ++s) ks[s] = *as_global(reinterpret_cast<const uint16_t *>(scales + 2 * s * size + key_scale_at));
  };
  // Values of a group: a thread of the half stages one (key, block), the block counting fastest.
  static_assert(S::UNITS <= kChunkThreads, "one unit a thread");
  u32x4 v;
  uint32_t vs;
  const int block = tid % (D / 32), row = tid / (D / 32);
  const uint32_t value_at = 16 * tid, value_scale_at = block * size + row;
  const uint32_t stage = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)smem + side * 2 * S::STAGE;
  const bool stages = S::UNITS == kChunkThreads || tid < S::UNITS;
  const uint32_t put_at = stage + row * S::ROW + ((4 * block) ^ chunk_swizzle<D>(row) ^ (block & 2)) * 16;
  auto load_values = [&](int group, int page) {
    const int64_t hd = (int64_t)max(page, 0) * a.cache.Hkv + it.h;
    const uint8_t *const codes = a.cache.value + (hd * size + place(group)) * (D / 2);
    const uint8_t *const scales = a.cache.value_scale + hd * (D / 32) * size + place(group);
    if (stages) {
      v = *as_global(reinterpret_cast<const u32x4 *>(codes + value_at));
      vs = *as_global(scales + value_scale_at);
    }
  };
  auto put_values = [&](int buffer) {
    if (stages) {
      const float scale = kv4_scale_value(min((int)vs, kKv4MaxScale));
#pragma unroll
      for (int c = 0; c < 4; ++c)
        *(__attribute__((address_space(3))) u32x4 *)((put_at ^ (16 * c)) + buffer * S::STAGE) = kv4_values(v[c], scale);
    }
  };
  // Transposing reads: lane (m, h) gets feature 32 d + m of keys 16 b + 8 h + 0..7.
  const int x = 8 * h + ((lane & 15) >> 2);
  uint32_t get_at = stage + x * S::ROW + ((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ chunk_swizzle<D>(x)) * 16 + 8 * (lane & 1);

  f32x16 s[2];
  uint32_t pw[4][4];
  // A group's scores, then the loads of the half's next keys.
  auto scores = [&](int next, int next_page) {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[0][r] = s[1][r] = 0.0f;
#pragma unroll
    for (int i = 0; i < S::KS; ++i) {
      s[0] = mfma32_fp4<0, 0>(k[0][i], first[i], s[0], (int)ks[i], qscale[i]);
      s[1] = mfma32_fp4<1, 0>(k[1][i], first[i], s[1], (int)ks[i], qscale[i]);
      s[0] = mfma32_fp4<0, 1>(k[0][i], second[i], s[0], (int)ks[i], qscale[i]);
      s[1] = mfma32_fp4<1, 1>(k[1][i], second[i], s[1], (int)ks[i], qscale[i]);
    }
    asm volatile("" : "+v"(s[0]), "+v"(s[1]) : : "memory");
    load_keys(next, next_page);
  };
  // Weights of a group: s[x][r] is key 16 (r / 4) + 8 h + 2 (r % 4) + x.
  auto weights = [&](int group, int page) {
    if (group * kGroupKeys + kGroupKeys - 1 > all_see || page < 0) {
      const int key = group * kGroupKeys + 8 * h, last = page < 0 ? -1 : last_key;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int at = key + 16 * (r / 4) + 2 * (r % 4);
        s[0][r] = at <= last ? s[0][r] : -INFINITY;
        s[1][r] = at + 1 <= last ? s[1][r] : -INFINITY;
      }
    }
    float best = max3(s[0][0], s[1][0], s[0][1]);
#pragma unroll
    for (int r = 1; r < 16; ++r) best = max3(best, s[1][r], s[0][(r + 1) & 15]);
    best = fmaxf(top, pair_max32(best) * a.scale_log2);
    if (__any(best > top)) {
      const float keep = fast_exp2(top - best);
      sum *= keep;
#pragma unroll
      for (int d = 0; d < S::DT; ++d) o[d] *= keep;
      top = best;
    }
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float p0 = fast_exp2(fmaf(s[0][4 * b + w], a.scale_log2, -top)), p1 = fast_exp2(fmaf(s[1][4 * b + w], a.scale_log2, -top));
        sum += p0 + p1;
        pw[b][w] = pack_weights(p0, p1);
      }
  };
  auto output = [&](int buffer) {
    const uint32_t get = get_at + buffer * S::STAGE;
    pipelined<4 * S::DT, 4>(
        [&](int n) {
          const int b = n / S::DT, d = n % S::DT;
          const uint32_t at = (get ^ (64 * d) ^ (16 * (d & 2))) + 16 * b * S::ROW;
          const u32x2 lo = read_transposed(at), hi = read_transposed(at + 4 * S::ROW);
          return as_bf16x8(u32x4{lo.x, lo.y, hi.x, hi.y});
        },
        [&](int n, const bf16x8 &w) {
          const int b = n / S::DT, d = n % S::DT;
          o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w, as_bf16x8(u32x4{pw[b][0], pw[b][1], pw[b][2], pw[b][3]}), o[d], 0, 0, 0);
        });
  };
  // The two halves of the waves take alternate groups.  Waves w and w + 4 share a SIMD, and between two barriers the
  // first half computes weights, then the matrix products (this group's output, its next one's scores), the second
  // half the products first (its last group's output, this one's scores), then weights: one's matrix work runs
  // beside the other's vector work.  Each half has a loop of its own: in a common one the compiler's waits for
  // loads would be those of either order.
  const int begin = it.group_begin, rounds = (group_end - begin + 1) / 2;
  auto sweep = [&](auto order) {
    constexpr bool AHEAD = decltype(order)::value;
    const int start = begin + (AHEAD ? 0 : 1);
    int page = page_of(start), next_page = page_of(start + 2);
    load_values(start, page);
    load_keys(start, page);
    convert_queries();
    if constexpr (AHEAD) {
      put_values(0);
      load_values(start + 2, next_page);
      scores(start + 2, next_page);
    }
    int group = start;
    for (int round = 0; round < rounds; ++round, group += 2) {
      asm volatile("" : "+v"(key_at), "+v"(key_scale_at), "+v"(get_at));
      const int after_page = page_of(group + 4);
      const bool active = group * kGroupKeys < none_see && group < group_end;  // uniform in the wave
      staged_barrier();  // the values that this round's outputs read are in LDS
      if constexpr (AHEAD) {
        put_values((round & 1) ^ 1);
        load_values(group + 4, after_page);
        if (active) {
          weights(group, page);
          output(round & 1);
        }
        scores(group + 4, after_page);
      } else {
        if (round > 0 && (group - 2) * kGroupKeys < none_see) output((round & 1) ^ 1);
        scores(group + 2, next_page);
        put_values(round & 1);
        load_values(group + 2, next_page);
        if (active) weights(group, page);
      }
      page = next_page, next_page = after_page;
    }
    if constexpr (!AHEAD) {
      staged_barrier();
      if (group - 2 < group_end && (group - 2) * kGroupKeys < none_see) output((rounds & 1) ^ 1);
    } else {
      staged_barrier();
    }
  };
  if (rounds > 0) {
    if (side == 0) sweep(Flag<true>{});
    else sweep(Flag<false>{});
  }

  // The second half hands its output over in LDS, a word of all lanes side by side.
  sum = pair_sum32(sum);
  float *const over = reinterpret_cast<float *>(smem) + wave * (32 * D) + lane;
  f32x2 *const over_ml = reinterpret_cast<f32x2 *>(smem + 4 * S::STAGE) + 64 * wave + lane;
  __syncthreads();
  if (side == 1) {
    *over_ml = f32x2{top, sum};
#pragma unroll
    for (int d = 0; d < S::DT; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) over[(16 * d + r) * 64] = o[d][r];
  }
  __syncthreads();
  if (side == 1 || !there) return;
  const f32x2 other = *over_ml;
  const float best = fmaxf(top, other.x), mine = fast_exp2(top - best), theirs = fast_exp2(other.x - best);
  sum = sum * mine + other.y * theirs;
#pragma unroll
  for (int d = 0; d < S::DT; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = o[d][r] * mine + over[(16 * d + r) * 64] * theirs;
  // o[d][r] is feature 32 d + 8 (r / 4) + 4 h + r % 4.  Records hold four features of the tile's vectors side by side: whole
  // lines a store.
  if (it.nsplit > 1) {
    const int64_t record = (int64_t)it.record * COLS + 32 * wave + m;
    float *const part = a.part_o + 4 * (((int64_t)it.record * (D / 4) + h) * COLS + 32 * wave + m);
#pragma unroll
    for (int d = 0; d < S::DT; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        *as_global(reinterpret_cast<f32x4 *>(part + 4 * (8 * d + 2 * r) * COLS)) =
            f32x4{o[d][4 * r], o[d][4 * r + 1], o[d][4 * r + 2], o[d][4 * r + 3]};
    if (h == 0) *as_global(reinterpret_cast<f32x2 *>(a.part_ml + 2 * record)) = f32x2{best, sum};
  } else {
    const float by = sum == 0.0f ? 0.0f : 1.0f / sum;
    uint16_t *const out = a.out + (((int64_t)it.row * a.T + t) * a.Hq + head) * D + 4 * h;
#pragma unroll
    for (int d = 0; d < S::DT; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        *as_global(reinterpret_cast<u32x2 *>(out + 32 * d + 8 * r)) =
            u32x2{pack_bf16x2(o[d][4 * r] * by, o[d][4 * r + 1] * by), pack_bf16x2(o[d][4 * r + 2] * by, o[d][4 * r + 3] * by)};
  }
}

// The same for 256 features: 8 waves of 16 query vectors.
template <int D>
__device__ __forceinline__ void paged_chunk_item_wide(const PagedArgs &a, const PagedItem &it, char *smem) {
  using S = PagedShape<D>;
  constexpr int WAVES = kPagedChunkWaves, THREADS = 64 * WAVES, COLS = 16 * WAVES, BLOCKS = D / 32, STAGE = 64 * S::ROW, KEYS = 65 * (D / 2);
  static_assert(64 * BLOCKS == THREADS, "a thread stages one block of one key");
  const int tid = threadIdx.x, lane = tid & 63, m = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  paged_zero_padded<D, THREADS>(a, it);

  const int vectors = it.count * a.G, wave_first = it.tile * COLS + 16 * wave, j = wave_first + m;
  const int t = j / a.G, head = it.h * a.G + (j - t * a.G);
  const bool there = j < vectors;
  const int last_key = there ? it.length - it.count + t : -1;
  const int all_see = it.length - it.count + wave_first / a.G;  // all of the wave's queries see keys up to this one,
  const int none_see = wave_first < vectors                     // and none of them this one or a later
                           ? it.length - it.count + (min(wave_first + 16, vectors) - 1) / a.G + 1 : 0;
  const int tile_end = it.length - it.count + (min(it.tile * COLS + COLS, vectors) - 1) / a.G + 1;
  const int group_end = min(it.group_end, (tile_end + kGroupKeys - 1) / kGroupKeys);
  QueryOperand<D> q;
  u32x4 qx[S::KC][QueryOperand<D>::PIECES][2];
  q.fetch(a.q.p + it.row * a.q.sb + head * a.q.sh + t * a.q.st, there, g, qx);

  f32x4 o[S::DT];
#pragma unroll
  for (int d = 0; d < S::DT; ++d) o[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float top = kLowest, sum = 0.0f;

  const int shift = a.cache.page_shift - 6, size = 1 << a.cache.page_shift;
  typedef const __attribute__((address_space(4))) int32_t *table_ptr;
  const table_ptr table = (table_ptr)(a.table + (int64_t)it.row * a.width);
  auto entry_of = [&](int group) { return group < group_end ? table[group >> shift] : -1; };
  auto checked = [&](int page) { return page >= 0 && page < a.cache.pages ? page : -1; };
  auto page_of = [&](int group) { return checked(entry_of(group)); };
  auto place = [&](int group) { return (group & ((1 << shift) - 1)) * kGroupKeys; };

  // Staged values: 16-byte chunk c of key r lies at slot c ^ S(r) ^ (c / 8), which puts the eight blocks of a key that eight
  // lanes store, and the chunk pairs of four rows that 16 lanes read, in different slots modulo eight.
  auto swizzle = [](int r) { return 2 * ((r & 3) + 4 * ((r >> 4) & 1)); };
  const int key = tid / BLOCKS, block = tid % BLOCKS;
  const uint32_t stage = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)smem;
  const uint32_t put_at = stage + key * S::ROW + ((4 * block) ^ swizzle(key) ^ (block >> 1)) * 16;
  const int x = 16 * g + (m >> 2);
  uint32_t get_at = stage + x * S::ROW + (((m & 3) >> 1) ^ swizzle(x)) * 16 + 8 * (m & 1);
  u32x4 v;
  uint32_t vs;
  auto load_values = [&](int group, int page) {
    const int64_t hd = (int64_t)max(page, 0) * a.cache.Hkv + it.h;
    v = *as_global(reinterpret_cast<const u32x4 *>(a.cache.value + (hd * size + place(group)) * (D / 2) + 16 * tid));
    vs = *as_global(a.cache.value_scale + hd * BLOCKS * size + place(group) + (uint32_t)(block * size + key));
  };
  auto put_values = [&](int buffer) {
    const float scale = kv4_scale_value(min((int)vs, kKv4MaxScale));
#pragma unroll
    for (int c = 0; c < 4; ++c)
      *(__attribute__((address_space(3))) u32x4 *)((put_at ^ (16 * c)) + buffer * STAGE) = kv4_values(v[c], scale);
  };

  // Keys are staged too, as they are: from the lanes' own rows a load would take one clock for 16 bytes of each lane, and
  // every wave would read all of them (5 chunks, 3 single tokens: 370 us, 390 so; with 128 features, where half as many
  // loads a product do it, staging cost 4 %).  Chunk c of key r lies at c ^ (r / 4)
  // of row r + r / 32: a lane reads keys 4 m + t, and 16 lanes' reads fill even and odd rows.
  const uint32_t keys = stage + 3 * STAGE;
  const uint32_t put_key_at = keys + (key + (key >> 5)) * (D / 2) + (block ^ ((key >> 2) & 7)) * 16;
  uint32_t get_key_at = keys + (4 * m + (m >> 3)) * (D / 2) + (g ^ (m & 7)) * 16;
  auto load_codes = [&](int group, int page) {
    const int64_t hd = (int64_t)max(page, 0) * a.cache.Hkv + it.h;
    return *as_global(reinterpret_cast<const u32x4 *>(a.cache.key + (hd * size + place(group)) * (D / 2) + 16 * tid));
  };
  auto put_codes = [&](int buffer, const u32x4 &codes) {
    *(__attribute__((address_space(3))) u32x4 *)(put_key_at + buffer * KEYS) = codes;
  };
  GroupLoads<D> in;
  in.init(size, stage, m, g);
  f32x4 s[4];
  uint32_t pw[2][4];
  // A group's scores, then the loads of the next one's scales.
  auto scores = [&](int buffer, int next, int next_page) {
    const uint32_t get = get_key_at + buffer * KEYS;
#pragma unroll
    for (int i = 0; i < S::KL; ++i)
      in.k[i] = *(const __attribute__((address_space(3))) u32x4 *)((get ^ (64 * (i % S::KC))) + (i / S::KC) * (D / 2));
    paged_scores<D>(in, q, g, s);
    asm volatile("" : "+v"(s[0]), "+v"(s[1]), "+v"(s[2]), "+v"(s[3]) : : "memory");
    in.key_scales(a, max(next_page, 0), it.h, place(next));
  };
  // Weights of a group: s[t][i] is key 16 g + 4 i + t.
  auto weights = [&](int group, int page) {
    if (group * kGroupKeys + kGroupKeys - 1 > all_see || page < 0) {
      const int at = group * kGroupKeys + 16 * g, last = page < 0 ? -1 : last_key;
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[u][i] = at + 4 * i + u <= last ? s[u][i] : -INFINITY;
    }
    float best = max3(s[0][0], s[1][0], s[2][0]);
    best = max3(best, s[3][0], s[0][1]);
#pragma unroll
    for (int i = 1; i < 4; ++i) best = max3(max3(best, s[1][i], s[2][i]), s[3][i], s[0][(i + 1) & 3]);
    best = fmaxf(top, pair_max32(pair_max16(best)) * a.scale_log2);
    if (__any(best > top)) {
      const float keep = fast_exp2(top - best);
      sum *= keep;
#pragma unroll
      for (int d = 0; d < S::DT; ++d) o[d] *= keep;
      top = best;
    }
    float part = 0.0f;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int i = 2 * u + w / 2, z = 2 * (w & 1);
        const float p0 = fast_exp2(fmaf(s[z][i], a.scale_log2, -top)), p1 = fast_exp2(fmaf(s[z + 1][i], a.scale_log2, -top));
        pw[u][w] = pack_weights(p0, p1);
        part = add_weights(pw[u][w], part);
      }
    sum += part;
  };
  auto output = [&](int buffer) {
    const uint32_t get = get_at + buffer * STAGE;
    __builtin_amdgcn_s_setprio(1);  // before the other wave's vector work (5 chunks, 3 single tokens: 395 us, 407 without)
    pipelined<2 * S::DT, 8>(
        [&](int k) {
          const int u = k / S::DT, d = k % S::DT;
          const uint32_t at = (get ^ (32 * d) ^ (16 * (d >> 2))) + 8 * u * S::ROW;
          const u32x2 lo = read_transposed(at), hi = read_transposed(at + 4 * S::ROW);
          return as_bf16x8(u32x4{lo.x, lo.y, hi.x, hi.y});
        },
        [&](int k, const bf16x8 &x) {
          const int u = k / S::DT, d = k % S::DT;
          o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, as_bf16x8(u32x4{pw[u][0], pw[u][1], pw[u][2], pw[u][3]}), o[d], 0, 0, 0);
        });
    __builtin_amdgcn_s_setprio(0);
  };
  // Waves w and w + 4 share a SIMD.  Between two barriers the first half of the waves computes weights, then the
  // matrix products (this group's output, the next one's scores); the second half the products first (the last
  // group's output, this one's scores), then weights: one's matrix work runs beside the other's vector work.  So three
  // groups' values are staged: the last, this and the next one, and the keys of this and the two next.
  // Each half has a loop of its own: in a common one the compiler's waits for loads would be those of either order.
  const int begin = it.group_begin;
  auto sweep = [&](auto order) {
    constexpr bool AHEAD = decltype(order)::value;
    int page = page_of(begin), next_page = page_of(begin + 1), after_page = page_of(begin + 2), far_page = page_of(begin + 3);
    load_values(begin, page);
    u32x4 codes = load_codes(begin, page), next_codes = load_codes(begin + 1, next_page);
    in.key_scales(a, max(page, 0), it.h, place(begin));
    q.convert(qx, m, g);
    put_values(0);
    put_codes(0, codes);
    put_codes(1, next_codes);
    load_values(begin + 1, next_page);
    codes = load_codes(begin + 2, after_page);
    staged_barrier();
    if constexpr (AHEAD) scores(0, begin + 1, next_page);
    int last = 2, now = 0, next = 1;  // staged groups' buffers
    for (int group = begin; group < group_end; ++group) {
      asm volatile("" : "+v"(in.key_scale_at), "+v"(get_at), "+v"(get_key_at));
      const int far_entry = entry_of(group + 4);  // looked at when it has arrived, at the end
      const bool active = group * kGroupKeys < none_see;  // uniform in the wave
      staged_barrier();  // every wave has stored its part of this group's values and of the next one's keys
      if constexpr (!AHEAD) {
        if (group > begin && (group - 1) * kGroupKeys < none_see) output(last);
        scores(now, group + 1, next_page);
      }
      put_values(next);
      put_codes(last, codes);
      load_values(group + 2, after_page);
      codes = load_codes(group + 3, far_page);
      if (active) weights(group, page);
      if constexpr (AHEAD) {
        if (active) output(now);
        scores(next, group + 2, after_page);
      }
      page = next_page, next_page = after_page, after_page = far_page, far_page = checked(far_entry);
      const int free = last;
      last = now, now = next, next = free;
    }
    if constexpr (!AHEAD) {
      if ((group_end - 1) * kGroupKeys < none_see) output(last);
    }
  };
  if (begin < group_end) {
    if (wave < WAVES / 2) sweep(Flag<true>{});
    else sweep(Flag<false>{});
  }

  sum = pair_sum32(pair_sum16(sum));
  if (!there) return;
  // o[d][i] is feature 16 d + 4 g + i.  Records hold four features of the tile's vectors side by side: whole lines a store.
  if (it.nsplit > 1) {
    const int64_t record = (int64_t)it.record * COLS + 16 * wave + m;
    float *const part = a.part_o + 4 * (((int64_t)it.record * (D / 4) + g) * COLS + 16 * wave + m);
#pragma unroll
    for (int d = 0; d < S::DT; ++d) *as_global(reinterpret_cast<f32x4 *>(part + 4 * 4 * d * COLS)) = o[d];
    if (g == 0) *as_global(reinterpret_cast<f32x2 *>(a.part_ml + 2 * record)) = f32x2{top, sum};
  } else {
    const float by = sum == 0.0f ? 0.0f : 1.0f / sum;
    uint16_t *const out = a.out + (((int64_t)it.row * a.T + t) * a.Hq + head) * D + 4 * g;
#pragma unroll
    for (int d = 0; d < S::DT; ++d)
      *as_global(reinterpret_cast<u32x2 *>(out + 16 * d)) =
          u32x2{pack_bf16x2(o[d][0] * by, o[d][1] * by), pack_bf16x2(o[d][2] * by, o[d][3] * by)};
  }
}

}  // namespace xattn
