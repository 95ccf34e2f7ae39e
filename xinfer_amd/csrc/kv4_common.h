// The 4-bit KV cache's format and arguments (kv4_cache.hip, paged_reserve.hip, paged_attention.hip).
//
// A key or value vector is held as blocks of 32 features: codes e2m1 (a sign and a magnitude of 0, 0.5, 1, 1.5, 2,
// 3, 4 or 6, the even feature in a byte's low half) and an e8m0 scale byte s for 2^(s - 127), the operand format of
// gfx950's scaled matrix instructions.  For a block whose largest magnitude is a,
//   s - 127 = e = floor(log2 a) - 2, one more where a > 7 * 2^e, kept in [-125, 125],
// and a feature's code is the value nearest to x / 2^e, ties to the even code.  7 is half way between the grid's 6
// and the next power's 8, so a block's largest feature is off by no more than half the grid's last step.  The range
// of e keeps every held value a normal bf16 number or zero, so reading it in bf16 is exact.
// A token whose key or value has an infinity or a NaN holds zeros, and 255 (NaN) in all of its key's scales: the
// scores of every query that sees it are NaN, and its value never poisons a query that does not.
//
// Pages of P tokens (P in {64, 128, 256}); per page and KV head the codes are [P][D/2] bytes and the scales
// [D/32][P], so a lane of the attention kernels finds the scales of consecutive keys in one word.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include "kernel_args.h"

namespace xattn {

constexpr int kKv4Block = 32;
constexpr int kKv4MinScale = 2, kKv4MaxScale = 252, kKv4NanScale = 255;

struct Kv4Cache {
  uint8_t *key, *key_scale, *value, *value_scale;
  int64_t pages;
  int32_t Hkv, D, page_shift;  // page size = 1 << page_shift
};

struct Kv4AppendArgs {
  View key, value;  // [B, Hkv, T, D]
  const int64_t *slots;
  int64_t slot_sb, slot_st;
  Kv4Cache cache;
  int32_t B, T;
};

struct Kv4ReadArgs {
  Kv4Cache cache;
  const int64_t *slots;
  int64_t slot_sb, slot_st;
  uint16_t *key, *value;  // contiguous [B, Hkv, T, D]
  int32_t B, T;
};

struct Kv4NormRopeArgs {
  View q, k, v;  // [B, H, T, D]
  const uint16_t *q_weight, *k_weight;
  View cos, sin;  // [B, T, R] (sb, st; sh unused)
  const int64_t *slots;
  int64_t slot_sb, slot_st;
  uint16_t *q_out;  // contiguous [B, Hq, T, D]
  Kv4Cache cache;
  float eps, offset;
  int32_t B, T, Hq, R;  // R: rotated features
};

struct ReserveArgs {
  const int32_t *before, *after, *counts;  // [B]
  const int64_t *counters;                 // head, tail
  int32_t *table;                          // [B, width]
  int32_t *ring;                           // [ring_size]
  int32_t *lengths;                        // [2, B]
  int64_t *positions, *slots;              // [B, T]
  int64_t *new_counters;
  int64_t ring_size;
  int32_t B, T, width, page_shift;
};

struct PagedArgs {
  View q;  // [B, Hq, T, D]
  Kv4Cache cache;
  const int32_t *table;  // [B, width]
  const int32_t *lengths;  // [2, B]
  uint16_t *out;           // contiguous [B, T, Hq, D]
  float scale_log2;
  int32_t B, Hq, G, T, width;
  int32_t max_length;  // at most width << page_shift
  // Work items (paged_plan.h).  A launch takes the rows with vectors_min to vectors_max query vectors a KV head;
  // from 0 on, the rows without any too.
  int32_t vectors_min, vectors_max;
  int32_t tile, min_groups, target;
  float record_groups;  // cost of a record in groups' time; 0: the target as it is (paged_run)
  float *part_o;  // unnormalised outputs of rows cut into runs: decode [item][tile][D], prefill [item][D / 4][tile][4]
  float *part_ml;  // [item][tile][2] running maximum (log2 units) and sum
};

// A paged attention call: rows of few query vectors a KV head go to the decode kernel, the others, where the shapes
// allow any, to the prefill kernel.
struct PagedLaunch {
  PagedArgs a;
  int64_t items;    // of the plan, at most; 0: no launch
  int64_t records;  // of cut rows' items, at most; 0: no row can be cut
  int tiles;        // of a row and KV head, at most
  size_t bytes;     // of the records
  int waves;        // of a decode block
};
constexpr int kMergeThreads = 256, kMergeQuads = 4;  // of a merge block; quads of features a thread takes of a prefill row
struct PagedLaunches {
  PagedLaunch few, many;
  size_t bytes() const { return few.bytes + many.bytes; }
  // Merge blocks of a row.
  int64_t few_merges() const {
    return few.bytes == 0 ? 0 : (int64_t)few.a.cache.Hkv * few.tiles * (few.a.tile < few.a.T * few.a.G ? few.a.tile : few.a.T * few.a.G);
  }
  int64_t many_merges() const {
    const int vectors = 4 * kMergeThreads * kMergeQuads / many.a.cache.D;
    return many.bytes == 0 ? 0 : (int64_t)many.a.cache.Hkv * many.tiles * ((many.a.tile + vectors - 1) / vectors);
  }
};

// Query vectors a KV head that one decode item takes at most (256 features leave registers for one group of 16).
constexpr int paged_decode_columns(int dim) { return dim == 256 ? 16 : 32; }
constexpr int kPagedRowWaves = 16;      // of a decode block that takes a whole row: all that a CU holds (up to 128 features)
constexpr int kPagedPrefillTile = 128;  // query vectors of a prefill item

}  // namespace xattn
