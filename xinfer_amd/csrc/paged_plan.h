// Work items of attention over the paged cache, laid out on the device from the rows' lengths.
//
// A launch is sized by the shapes alone.  Its waves each compute the same plan from the lengths: a row's keys are cut into
// `nsplit` runs of 64-key groups, its query vectors (query heads of a KV head times tokens) into tiles, and an item is a
// (tile, run, KV head).  Runs take at least `min_groups` groups, and as many more as leave at most about `target` items
// (paged_run), so a few long rows fill the chip and many rows are not cut at all.  Items past the plan's last end at once.
// The KV head counts fastest: consecutive blocks go to the 8 XCDs in turn, so with 8 KV heads the tiles of one head meet
// in one XCD's L2.
//
// What bounds it: latency.  A block knows its item some 1.3 us after its start (arguments, lengths, a dozen exchanges
// among lanes); a block without one holds its place on a CU for about 3 us.
#pragma once

#include "kv4_device.h"

namespace xattn {

constexpr int kGroupKeys = 64;

struct PagedRow {
  int count, length;
};
__device__ __forceinline__ PagedRow paged_row(const PagedArgs &a, int r) {
  PagedRow p;
  p.count = min(max(a.lengths[r], 0), min(a.T, a.max_length));
  p.length = min(max(a.lengths[a.B + r], p.count), a.max_length);
  return p;
}

// The lane's row of 64 from `base` on.
__device__ __forceinline__ PagedRow paged_lane_row(const PagedArgs &a, int base) {
  const int r = base + (int)(threadIdx.x & 63);
  return r < a.B ? paged_row(a, r) : PagedRow{0, 0};
}

struct PagedItem {
  int row, count, length;
  int h, tile, split, nsplit, tiles;
  int group_begin, group_end;  // 64-key groups of the run
  int record;                  // of cut rows' items, which are counted apart: this one's
};

// What a launch takes of row r: 64-key groups and tiles; no tiles: the row is another launch's.
struct PagedShare {
  int groups, tiles;
};
__device__ __forceinline__ PagedShare paged_share(const PagedArgs &a, const PagedRow &p) {
  const int vectors = p.count * a.G;
  PagedShare s{0, 0};
  if (vectors == 0) {
    s.tiles = a.vectors_min == 0 ? 1 : 0;  // only zeros to write
  } else if (vectors >= a.vectors_min && vectors <= a.vectors_max) {
    s.groups = (p.length + kGroupKeys - 1) / kGroupKeys;
    s.tiles = (vectors + a.tile - 1) / a.tile;
  }
  return s;
}

// Rows 64 at a time, one a lane: what the plan looks at.  The first 64 stay in registers.
struct PagedRows {
  PagedRow p;
  PagedShare s;
  __device__ __forceinline__ void load(const PagedArgs &a, int base) { take(a, base, paged_lane_row(a, base)); }
  __device__ __forceinline__ void take(const PagedArgs &a, int base, const PagedRow &row) {
    p = row;
    s = base + (int)(threadIdx.x & 63) < a.B ? paged_share(a, p) : PagedShare{0, 0};
  }
};

__device__ __forceinline__ int paged_splits(const PagedShare &s, int run) { return max(1, (s.groups + run - 1) / run); }

// Groups of a run at most.
//
// Prefill items of ragged batches are long and of different lengths, so what a target of items gives is estimated for
// eight: n items of at most m groups on kPagedSlots blocks at a time take no longer than ceil(n / slots) m, nor than
// their mean load and m; an item costs kPagedItemGroups more (queries in, output out) and a record what it is written
// and read for (a.record_groups).  On a batch of 5 rows of 33 to 223 groups, 256 features: 432 us with targets up to
// 768, 499 with 512 or 256 (368 now); uniform batches choose 256 (4 rows of 64 groups, 128 features: 94 us, with 256 alone 92, the rest
// being blocks without an item).
constexpr int kPagedSlots = 256;
constexpr float kPagedItemGroups = 4.0f;

__device__ __forceinline__ int paged_run(const PagedArgs &a, const PagedRows &first) {
  float total = (float)first.s.groups * (float)first.s.tiles;
  for (int base = 64; base < a.B; base += 64) {
    PagedRows rows;
    rows.load(a, base);
    total += (float)rows.s.groups * (float)rows.s.tiles;
  }
  total = group_sum<64>(total) * (float)a.cache.Hkv;
  if (a.record_groups <= 0.0f) return max(a.min_groups, (int)(total / (float)a.target) + 1);
  // Eight targets at a time, each by eight lanes, which take every eighth row.
  const int lane = threadIdx.x & 63, target = min(kPagedSlots + kPagedSlots / 4 * (lane >> 3), a.target);
  const int run = max(a.min_groups, (int)(total / (float)target) + 1);
  float n = 0.0f, records = 0.0f, longest = 0.0f;
  for (int base = 0; base < a.B; base += 8) {
    const int from = base + (lane & 7), groups = __shfl(first.s.groups, from), tiles = __shfl(first.s.tiles, from);
    const int nsplit = max(1, (groups + run - 1) / run);
    const float items = (float)(tiles * nsplit);
    n += items;
    records += nsplit > 1 ? items : 0.0f;
    longest = fmaxf(longest, (float)((groups + nsplit - 1) / nsplit));
  }
  n = group_sum<8>(n) * (float)a.cache.Hkv;
  records = group_sum<8>(records) * (float)a.cache.Hkv;
  for (int mask = 1; mask < 8; mask *= 2) longest = fmaxf(longest, __shfl_xor(longest, mask));
  const float m = longest + kPagedItemGroups, rounds = ceilf(n / (float)kPagedSlots) * m;
  const float cost = fminf(rounds, (total + n * kPagedItemGroups) / (float)kPagedSlots + m) + records * a.record_groups;
  float best = cost;
  for (int mask = 8; mask < 64; mask *= 2) best = fminf(best, __shfl_xor(best, mask));
  return __builtin_amdgcn_readlane(run, __builtin_ctzll(__ballot(cost == best)));
}

// What lane `at` holds of its row.
__device__ __forceinline__ void paged_take(PagedItem &it, const PagedRows &rows, int nsplit, int at) {
  it.count = __builtin_amdgcn_readlane(rows.p.count, at);
  it.length = __builtin_amdgcn_readlane(rows.p.length, at);
  it.nsplit = __builtin_amdgcn_readlane(nsplit, at);
  it.tiles = __builtin_amdgcn_readlane(rows.s.tiles, at);
  it.group_end = __builtin_amdgcn_readlane(rows.s.groups, at);
}

// Item `index` of the plan, false past its last, index then goes down by how many there are.  Every lane of a wave calls it, with the same index and its row of the first 64.
__device__ __forceinline__ bool paged_item(const PagedArgs &a, const PagedRow &lane_row, int &index, PagedItem &it) {
  const int Hkv = a.cache.Hkv;
  PagedRows rows;
  rows.take(a, 0, lane_row);
  const int run = paged_run(a, rows);
  for (int base = 0, records = 0;;) {
    const int nsplit = paged_splits(rows.s, run), items = rows.s.tiles * nsplit * Hkv, cut = nsplit > 1 ? items : 0;
    const int upto = wave_scan(items), cut_upto = wave_scan(cut);
    const uint64_t past = __ballot(upto > index);
    if (past != 0) {
      const int at = __builtin_ctzll(past);
      it.row = base + at;
      paged_take(it, rows, nsplit, at);
      const uint32_t i = index - __builtin_amdgcn_readlane(upto - items, at), rest = i / (uint32_t)Hkv;
      it.record = records + __builtin_amdgcn_readlane(cut_upto - cut, at) + (int)i;
      it.h = i - rest * Hkv;
      it.tile = rest / (uint32_t)it.nsplit;
      it.split = rest - it.tile * it.nsplit;
      // The first `more` runs take one group more than the others.
      const int groups = it.group_end, each = (uint32_t)groups / (uint32_t)it.nsplit, more = groups - each * it.nsplit;
      it.group_begin = it.split * each + min(it.split, more);
      it.group_end = it.group_begin + each + (it.split < more ? 1 : 0);
      return true;
    }
    index -= __builtin_amdgcn_readlane(upto, 63);
    records += __builtin_amdgcn_readlane(cut_upto, 63);
    base += 64;
    if (base >= a.B) return false;
    rows.load(a, base);
  }
}

// Row `row`'s part of the plan: its first record, splits and tiles.
__device__ __forceinline__ void paged_row_items(const PagedArgs &a, int row, PagedItem &it) {
  PagedRows rows;
  rows.load(a, 0);
  const int run = paged_run(a, rows);
  for (int base = 0, records = 0;; rows.load(a, base)) {
    const int nsplit = paged_splits(rows.s, run), cut = nsplit > 1 ? rows.s.tiles * nsplit * a.cache.Hkv : 0, upto = wave_scan(cut);
    if (row < base + 64) {
      it.row = row;
      paged_take(it, rows, nsplit, row - base);
      it.record = records + __builtin_amdgcn_readlane(upto - cut, row - base);
      return;
    }
    base += 64;
    records += __builtin_amdgcn_readlane(upto, 63);
  }
}

// Zeros for the row's padded queries of the item's head, by the item of its first tile and run.
template <int D, int THREADS>
__device__ __forceinline__ void paged_zero_padded(const PagedArgs &a, const PagedItem &it) {
  if (it.tile != 0 || it.split != 0) return;
  constexpr int CHUNKS = D / 8;
  uint16_t *const out = a.out + ((int64_t)it.row * a.T * a.Hq + (int64_t)it.h * a.G) * D;
  for (int i = threadIdx.x / CHUNKS; i < (a.T - it.count) * a.G; i += THREADS / CHUNKS) {
    const int t = i / a.G;
    store16(out + ((int64_t)(it.count + t) * a.Hq + (i - t * a.G)) * D + 8 * (threadIdx.x % CHUNKS), u32x4{0, 0, 0, 0});
  }
}

}  // namespace xattn
