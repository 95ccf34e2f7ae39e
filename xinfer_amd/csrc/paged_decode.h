// Attention over the paged 4-bit cache for rows of few query vectors a KV head: single tokens and short runs of them.
//
// A block takes an item (paged_plan.h): up to 16 * NC query vectors of a (row, KV head) over a run of
// keys, one 64-key group at a time per wave.  A wave keeps the running maximum and sum of the softmax and its
// output in registers; the waves meet in LDS at the end, runs in the merge kernel.
//
// Scores are S^T = K Q^T on the scaled matrix cores straight from the cache's codes (paged_mfma.h): row m of tile t
// (of four) is key 4 m + t of the group, so a lane's four keys have their scales in one word and the instruction picks
// the byte.  Lane (column q, g = lane / 16) then holds the scores of keys 16 g .. 16 g + 15 of its query: the softmax
// needs two exchanges for the maximum, and the weights are the PV product's B operand where they are.  That
// product's A operand is V^T: a value's codes become bf16 (exact, one conversion a pair) and pass through LDS,
// half a group at a time, to be read transposed.
//
// Weights are rounded to bf16.  With up to 8 vectors the other 8 columns hold what that rounding loses
// (w - bf16(w)), at no further matrix work, which leaves 2^-16 of a weight; with more the rounding is up to 2^-8.
//
// What bounds it: memory where there is much to read (64 rows of 1605 to 16384 keys, 16 / 8 heads of 128 features: 637 MB
// in 139 us, 4.6 TB/s, the vector units at work 40 % of the time; 8 rows of 55 to 13312 keys, 34 MB: 17.0 us, 4 of them
// the merge), and latency where there is little (one row of 1 to 64 keys 6.1 us, 1024 keys 10.5 with the merge).  A wave's
// group takes some 200 vector instructions, 64 conversions and 16 exponentials: 16 waves on one CU 0.35 us a group.
#pragma once

#include "paged_mfma.h"
#include "paged_plan.h"

namespace xattn {

constexpr float kLowest = -3.0e38f;  // running maximum before any key

template <int D>
struct PagedShape {
  static constexpr int KC = D == 256 ? 2 : 1;      // 128-feature chunks of a key (D = 64: half a chunk)
  static constexpr int KL = D == 64 ? 2 : 4 * KC;  // 16-byte loads a lane makes of a group's keys
  static constexpr int VL = D / 64;                // and of half a group's values
  static constexpr int DT = D / 16;                // 16-feature tiles of the output
  static constexpr int ROW = 2 * D, STAGE = 32 * ROW;
};

// Slot of 16-byte chunk c of staged row r.  The XOR spreads what one LDS pass serves over all banks: the stores of 8
// consecutive rows (one chunk each) and the transposing reads of rows 8 g + 4 s + 0..3, g = 0..3 (a pair of chunks
// each).
template <int D>
__device__ __forceinline__ int stage_swizzle(int r) {
  return D == 64 ? 2 * (((r >> 1) & 1) + 2 * ((r >> 3) & 1)) ^ ((r >> 2) & 1)
                 : 2 * ((r & 3) + 4 * ((r >> 3) & 1)) ^ ((r >> 2) & 1);
}

typedef short i16x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ u32x2 read_transposed(uint32_t lds) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4 *)(lds)));
}

// A lane's loads of a 64-key group and KV head, and its places in the staged half group.  A lane's offsets are few
// words kept for the whole item, from which every address of an iteration follows by a constant.
template <int D>
struct GroupLoads {
  using S = PagedShape<D>;
  u32x4 k[S::KL];
  uint32_t ks[S::KC];
  u32x4 v[2][S::VL];
  uint32_t vs[2][S::VL];
  uint32_t key_at, key_scale_at, value_at, value_scale_at;  // in a group's codes and scales
  uint32_t put_at, get_at;                                  // LDS bytes

  __device__ __forceinline__ void init(int size, uint32_t stage, int m, int g) {
    // Keys: load i of D = 64 takes key 4 m + 2 (g / 2) + i, block g % 2; else key 4 m + i / KC, block 4 (i % KC) + g.
    key_at = D == 64 ? (4 * m + 2 * (g >> 1)) * 32 + 16 * (g & 1) : 4 * m * (D / 2) + 16 * g;
    key_scale_at = (D == 64 ? (g & 1) : g) * size + 4 * m;
    // Values: load w of half u takes row r of the half, key 16 (r / 8) + 8 u + r % 8.
    const int r = D == 64 ? 16 * (g >> 1) + m : m, block = D == 64 ? (g & 1) : g, key = 16 * (r >> 3) + (r & 7);
    value_at = key * (D / 2) + 16 * block;
    value_scale_at = block * size + key;
    put_at = stage + r * S::ROW + ((4 * block) ^ stage_swizzle<D>(r)) * 16;
    const int x = 8 * g + (m >> 2);
    get_at = stage + x * S::ROW + (((m & 3) >> 1) ^ stage_swizzle<D>(x)) * 16 + 8 * (m & 1);
  }
  // Keeps the compiler from carrying every address of the loop in a register of its own.
  __device__ __forceinline__ void renew() {
    asm volatile("" : "+v"(key_at), "+v"(key_scale_at), "+v"(value_at), "+v"(value_scale_at), "+v"(put_at), "+v"(get_at));
  }

  __device__ __forceinline__ void keys(const PagedArgs &a, int page, int h, int at) {
    const int size = 1 << a.cache.page_shift;
    const int64_t head = (int64_t)page * a.cache.Hkv + h;
    const uint8_t *const codes = a.cache.key + (head * size + at) * (D / 2);
#pragma unroll
    for (int i = 0; i < S::KL; ++i)
      k[i] = *as_global(reinterpret_cast<const u32x4 *>(codes + (i / S::KC) * (D / 2) + (i % S::KC) * 64 + key_at));
    key_scales(a, page, h, at);
  }
  __device__ __forceinline__ void key_scales(const PagedArgs &a, int page, int h, int at) {
    const int size = 1 << a.cache.page_shift;
    const uint8_t *const scales = a.cache.key_scale + ((int64_t)page * a.cache.Hkv + h) * (D / 32) * size + at;
#pragma unroll
    for (int c = 0; c < S::KC; ++c)
      ks[c] = *as_global(reinterpret_cast<const uint32_t *>(scales + 4 * c * size + key_scale_at));
  }
  __device__ __forceinline__ void values(const PagedArgs &a, int page, int h, int at) {
    const int size = 1 << a.cache.page_shift;
    const int64_t head = (int64_t)page * a.cache.Hkv + h;
    const uint8_t *const codes = a.cache.value + (head * size + at) * (D / 2);
    const uint8_t *const scales = a.cache.value_scale + head * (D / 32) * size + at;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int w = 0; w < S::VL; ++w) {
        const int key = 32 * (w / S::KC) + 8 * u, c = w % S::KC;
        v[u][w] = *as_global(reinterpret_cast<const u32x4 *>(codes + key * (D / 2) + 64 * c + value_at));
        vs[u][w] = *as_global(scales + 4 * c * size + key + value_scale_at);
      }
  }
  // Half u's values into LDS as bf16.
  __device__ __forceinline__ void put(int u) const {
#pragma unroll
    for (int w = 0; w < S::VL; ++w) {
      const float scale = kv4_scale_value(min((int)vs[u][w], kKv4MaxScale));
#pragma unroll
      for (int c = 0; c < 4; ++c)
        *(__attribute__((address_space(3))) u32x4 *)((put_at ^ (16 * c)) + 16 * (w / S::KC) * S::ROW + 256 * (w % S::KC)) =
            kv4_values(v[u][w][c], scale);
    }
  }
  // Features 16 d .. of the staged half: this lane's feature of keys 16 g + 8 u + 0..7.
  __device__ __forceinline__ bf16x8 get(int d) const {
    const u32x2 x = read_transposed(get_at ^ (32 * d)), y = read_transposed((get_at ^ (32 * d + 16)) + 4 * S::ROW);
    return as_bf16x8(u32x4{x.x, x.y, y.x, y.y});
  }
};

// The largest of three; a NaN counts for nothing.
__device__ __forceinline__ float max3(float x, float y, float z) { return fmaxf(fmaxf(x, y), z); }

// STEPS products whose A operands come from LDS, DEPTH reads ahead of their use.  The order is kept: left alone, the
// compiler reads one operand at a time and every product waits for LDS.
template <int STEPS, int DEPTH, typename Get, typename Use>
__device__ __forceinline__ void pipelined(Get get, Use use) {
  bf16x8 x[DEPTH];
#pragma unroll
  for (int k = 0; k < DEPTH && k < STEPS; ++k) x[k] = get(k);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int k = 0; k < STEPS; ++k) {
    use(k, x[k % DEPTH]);
    if (k + DEPTH < STEPS) x[k % DEPTH] = get(k + DEPTH);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// A query column's operands: the two e4m3 terms of each chunk, their scale bytes (terms' in bytes 0 and 1).
template <int D>
struct QueryOperand {
  using S = PagedShape<D>;
  static constexpr int PIECES = D == 64 ? 1 : 2;
  u32x4 first[S::KC][2], second[S::KC][2];
  int scale[S::KC];
  // The column's features of this lane, zero where there is no such column.
  __device__ __forceinline__ void fetch(const uint16_t *q, bool there, int g, u32x4 (&x)[S::KC][PIECES][2]) const {
#pragma unroll
    for (int c = 0; c < S::KC; ++c)
#pragma unroll
      for (int p = 0; p < PIECES; ++p)
#pragma unroll
        for (int e = 0; e < 2; ++e) x[c][p][e] = there ? load16(q + 128 * c + 64 * p + 16 * g + 8 * e) : u32x4{0, 0, 0, 0};
  }
  __device__ __forceinline__ void convert(const u32x4 (&x)[S::KC][PIECES][2], int m, int g) {
#pragma unroll
    for (int c = 0; c < S::KC; ++c) {
      int s[2] = {127, 127};
#pragma unroll
      for (int p = 0; p < PIECES; ++p) {
        // The block's other 16 features are in lane group g ^ 1.
        const uint32_t top = largest(x[c][p][1], largest(x[c][p][0], 0u));
        const auto r = __builtin_amdgcn_permlane16_swap(top, top, false, false);
        s[p] = query_scale(max(r[0], r[1]));
        split_query(x[c][p][0], x[c][p][1], s[p], first[c][p], second[c][p]);
      }
      if constexpr (D == 64) first[c][1] = second[c][1] = u32x4{0, 0, 0, 0};
      // Block g's scale is with lane group 2 (g % 2), of its first piece for g < 2.
      const int from = m + 32 * (g & 1), b0 = __shfl(s[0], from), b1 = __shfl(s[1], from);
      const int mine = D == 64 || g < 2 ? b0 : b1;
      scale[c] = mine | (mine == 255 ? 255 : mine - 4) << 8;
    }
  }
};

// Scores of a group's keys against 16 queries: s[t][i] of lane (m, g) is query m's of key 16 g + 4 i + t.
template <int D>
__device__ __forceinline__ void paged_scores(const GroupLoads<D> &in, const QueryOperand<D> &q, int g, f32x4 (&s)[4]) {
  using S = PagedShape<D>;
  const f32x4 zero{0.0f, 0.0f, 0.0f, 0.0f};
  if constexpr (D == 64) {
    // Lane groups 0 and 1 hold tiles 0 and 1, lane groups 2 and 3 tiles 2 and 3, each half against zeros while the
    // other counts; a scale beside a zero has to be finite.
    const int low = g < 2 ? (int)in.ks[0] : 0x7f7f7f7f, high = g < 2 ? 0x7f7f7f7f : (int)in.ks[0];
    const int ql = g < 2 ? q.scale[0] : 0x7f7f, qh = g < 2 ? 0x7f7f : q.scale[0];
    const u32x4 none{0, 0, 0, 0};
    const u32x4 f1[2] = {none, q.first[0][0]}, r1[2] = {none, q.second[0][0]};
    s[0] = mfma16_fp4<0, 1>(in.k[0], q.second[0], mfma16_fp4<0, 0>(in.k[0], q.first[0], zero, low, ql), low, ql);
    s[1] = mfma16_fp4<1, 1>(in.k[1], q.second[0], mfma16_fp4<1, 0>(in.k[1], q.first[0], zero, low, ql), low, ql);
    s[2] = mfma16_fp4<2, 1>(in.k[0], r1, mfma16_fp4<2, 0>(in.k[0], f1, zero, high, qh), high, qh);
    s[3] = mfma16_fp4<3, 1>(in.k[1], r1, mfma16_fp4<3, 0>(in.k[1], f1, zero, high, qh), high, qh);
  } else {
#pragma unroll
    for (int t = 0; t < 4; ++t) s[t] = zero;
#pragma unroll
    for (int c = 0; c < S::KC; ++c) {
      const int qs = q.scale[c], ks = (int)in.ks[c];
      s[0] = mfma16_fp4<0, 1>(in.k[c], q.second[c], mfma16_fp4<0, 0>(in.k[c], q.first[c], s[0], ks, qs), ks, qs);
      s[1] = mfma16_fp4<1, 1>(in.k[S::KC + c], q.second[c], mfma16_fp4<1, 0>(in.k[S::KC + c], q.first[c], s[1], ks, qs), ks, qs);
      s[2] = mfma16_fp4<2, 1>(in.k[2 * S::KC + c], q.second[c], mfma16_fp4<2, 0>(in.k[2 * S::KC + c], q.first[c], s[2], ks, qs), ks, qs);
      s[3] = mfma16_fp4<3, 1>(in.k[3 * S::KC + c], q.second[c], mfma16_fp4<3, 0>(in.k[3 * S::KC + c], q.first[c], s[3], ks, qs), ks, qs);
    }
  }
}

// LDS of a decode block: the waves' staged values (then outputs), their maxima and sums.
template <int D, int WAVES>
constexpr int kPagedDecodeLds = WAVES * (PagedShape<D>::STAGE + 16 * 8);

// Item `it` of the plan, by the whole block; smem: kPagedDecodeLds bytes, 1024-byte aligned.
template <int D, int NC, int WAVES>
__device__ __forceinline__ void paged_decode_item(const PagedArgs &a, const PagedItem &it, char *smem) {
  using S = PagedShape<D>;
  constexpr int COLS = 16 * NC, THREADS = 64 * WAVES;
  f32x2 *const wave_ml = reinterpret_cast<f32x2 *>(smem + WAVES * S::STAGE);
  const int tid = threadIdx.x, lane = tid & 63, m = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (it.count < a.T) paged_zero_padded<D, THREADS>(a, it);
  if (it.count == 0) return;
  const int vectors = min(it.count * a.G - it.tile * COLS, COLS);
  const bool twice = NC == 1 && vectors <= 8;  // columns 8..15 repeat the queries and take the weights' rests

  const uint32_t rests = twice && m >= 8 ? ~0u : 0u;

  QueryOperand<D> q[NC];
  u32x4 qx[NC][S::KC][QueryOperand<D>::PIECES][2];
  int last_key[NC];  // the last key that this lane's query sees
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    const int column = twice ? m & 7 : m + 16 * n, j = it.tile * COLS + column, t = j / a.G;
    const bool there = column < vectors;
    q[n].fetch(a.q.p + it.row * a.q.sb + (it.h * a.G + (j - t * a.G)) * a.q.sh + t * a.q.st, there, g, qx[n]);
    last_key[n] = there ? it.length - it.count + t : -1;
  }
  const int all_see = it.length - it.count + it.tile * COLS / a.G;  // every query sees keys up to this one

  f32x4 o[NC][S::DT];
  float top[NC], sum[NC];
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    top[n] = kLowest;
    sum[n] = 0.0f;
#pragma unroll
    for (int d = 0; d < S::DT; ++d) o[n][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  char *const stage = smem + wave * S::STAGE;

  const int shift = a.cache.page_shift - 6;  // pages by groups
  typedef const __attribute__((address_space(4))) int32_t *table_ptr;
  const table_ptr table = (table_ptr)(a.table + (int64_t)it.row * a.width);
  auto page_of = [&](int group) {
    const int page = group < it.group_end ? table[group >> shift] : -1;
    return page >= 0 && page < a.cache.pages ? page : -1;
  };
  auto place = [&](int group) { return (group & ((1 << shift) - 1)) * kGroupKeys; };

  // A group's loads are under way while the one before it is worked on, its page number while the one before that is.
  // Absent pages, and groups past the run, read page 0 and hide every key: no branch parts a group's work, which
  // would have the compiler keep two groups in registers.
  GroupLoads<D> in;
  in.init(1 << a.cache.page_shift, (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)stage, m, g);
  int group = it.group_begin + wave, page = page_of(group), next_page = page_of(group + WAVES);
  if (group < it.group_end) {
    in.keys(a, max(page, 0), it.h, place(group));
    in.values(a, max(page, 0), it.h, place(group));
  }
#pragma unroll
  for (int n = 0; n < NC; ++n) q[n].convert(qx[n], m, g);
  for (; group < it.group_end; group += WAVES) {
    in.renew();
    const int next = group + WAVES, after_page = page_of(next + WAVES), load_page = max(next_page, 0);
    f32x4 s[NC][4];
#pragma unroll
    for (int n = 0; n < NC; ++n) paged_scores<D>(in, q[n], g, s[n]);
    // The scores are taken here, before the registers of their keys are loaded anew.
#pragma unroll
    for (int n = 0; n < NC; ++n) asm volatile("" : "+v"(s[n][0]), "+v"(s[n][1]), "+v"(s[n][2]), "+v"(s[n][3]) : : "memory");
    in.keys(a, load_page, it.h, place(next));
    __builtin_amdgcn_sched_barrier(0);

    // Weights: s[n][t][i] is key 16 g + 4 i + t of the group.
    uint32_t pw[NC][2][4];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      if (group * kGroupKeys + kGroupKeys - 1 > all_see || page < 0) {
        const int key = group * kGroupKeys + 16 * g, last = page < 0 ? -1 : last_key[n];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[n][t][i] = key + 4 * i + t <= last ? s[n][t][i] : -INFINITY;
      }
      float x = fmaxf(fmaxf(s[n][0][0], s[n][1][0]), fmaxf(s[n][2][0], s[n][3][0]));
#pragma unroll
      for (int i = 1; i < 4; ++i) x = fmaxf(x, fmaxf(fmaxf(s[n][0][i], s[n][1][i]), fmaxf(s[n][2][i], s[n][3][i])));
      x = pair_max32(pair_max16(x));
      const float now = fmaxf(top[n], x * a.scale_log2);
      if (__any(now > top[n])) {
        const float keep = fast_exp2(top[n] - now);
        sum[n] *= keep;
#pragma unroll
        for (int d = 0; d < S::DT; ++d) o[n][d] *= keep;
        top[n] = now;
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int i = 2 * u + w / 2, t = 2 * (w & 1);
          const float p0 = fast_exp2(fmaf(s[n][t][i], a.scale_log2, -now)), p1 = fast_exp2(fmaf(s[n][t + 1][i], a.scale_log2, -now));
          sum[n] += p0 + p1;
          if constexpr (NC == 1) {
            const uint32_t word = pack_weights(p0, p1) & rests;
            pw[n][u][w] = pack_weights(p0 - bf16_lo(word), p1 - bf16_hi(word));
          } else {
            pw[n][u][w] = pack_weights(p0, p1);
          }
        }
    }

    __builtin_amdgcn_sched_barrier(0);
    // Output: half the group's values in LDS at a time, read transposed.
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      in.put(u);
      if (u == 1) in.values(a, load_page, it.h, place(next));
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      auto use = [&](int d, const bf16x8 &v) {
#pragma unroll
        for (int n = 0; n < NC; ++n)
          o[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              v, as_bf16x8(u32x4{pw[n][u][0], pw[n][u][1], pw[n][u][2], pw[n][u][3]}), o[n][d], 0, 0, 0);
      };
      if constexpr (D == 256 || NC == 2) {
        pipelined<S::DT, 4>([&](int d) { return in.get(d); }, use);
      } else {
        // Four waves a SIMD fill each other's waits, and there are no registers to read ahead.
#pragma unroll
        for (int d = 0; d < S::DT; ++d) {
          if (d % 4 == 0) __builtin_amdgcn_sched_barrier(0);
          use(d, in.get(d));
        }
      }
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
    }
    page = next_page, next_page = after_page;
  }

  // The waves' outputs, and the weights' rests (columns 8..15), meet in LDS.
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    const float l = pair_sum32(pair_sum16(sum[n]));
    if (twice) {
#pragma unroll
      for (int d = 0; d < S::DT; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][d][i] += dpp_move<kDppRowRor8>(o[n][d][i]);
    }
    __syncthreads();
    const int columns = min(vectors - 16 * n, 16);
    if (g == 0) wave_ml[16 * wave + m] = f32x2{top[n], l};
    if (m < columns) {
#pragma unroll
      for (int d = 0; d < S::DT; ++d)
        *reinterpret_cast<f32x4 *>(stage + m * (4 * D) + ((4 * d + g) ^ (m & 7)) * 16) = o[n][d];
    }
    __syncthreads();
    for (int i = tid; i < columns * (D / 4); i += THREADS) {
      const int column = i / (D / 4), f = i - column * (D / 4);
      float best = kLowest, total = 0.0f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) best = fmaxf(best, wave_ml[16 * w + column].x);
      f32x4 out{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        const f32x2 ml = wave_ml[16 * w + column];
        const float keep = fast_exp2(ml.x - best);
        total += ml.y * keep;
        out += *reinterpret_cast<const f32x4 *>(smem + w * S::STAGE + column * (4 * D) + (f ^ (column & 7)) * 16) * keep;
      }
      if (it.nsplit > 1) {
        const int64_t record = (int64_t)it.record * COLS + 16 * n + column;
        *as_global(reinterpret_cast<f32x4 *>(a.part_o + record * D + 4 * f)) = out;
        if (f == 0) *as_global(reinterpret_cast<f32x2 *>(a.part_ml + 2 * record)) = f32x2{best, total};
      } else {
        const int j = it.tile * COLS + 16 * n + column, t = j / a.G;
        const float by = total == 0.0f ? 0.0f : 1.0f / total;
        out *= by;
        *as_global(reinterpret_cast<u32x2 *>(
            a.out + (((int64_t)it.row * a.T + t) * a.Hq + it.h * a.G + (j - t * a.G)) * D + 4 * f)) =
            u32x2{pack_bf16x2(out[0], out[1]), pack_bf16x2(out[2], out[3])};
      }
    }
  }
}

}  // namespace xattn
