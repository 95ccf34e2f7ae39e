// C ABI of the paged 4-bit KV cache (include/xinfer_attention.h): validation and launches.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <limits>

#include "xinfer_attention.h"
#include "kv4_common.h"
#include "launch.h"

namespace xattn {
namespace {

constexpr int64_t kIntMax = std::numeric_limits<int32_t>::max();
constexpr int64_t kMostTokens = int64_t(1) << 30;  // of a page table's row: positions stay in 32 bits
constexpr int64_t kMostRows = 65535;               // of a batch
// A launch's threads are counted in 32 bits.
bool launchable(int64_t threads) { return threads < (int64_t(1) << 32) - 1024; }

bool aligned16(const void *p) { return p != nullptr && (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int page_shift(int64_t page_size) { return page_size == 64 ? 6 : page_size == 128 ? 7 : page_size == 256 ? 8 : -1; }

bool cache_of(const xinfer_kv4_cache &c, Kv4Cache &out) {
  if (page_shift(c.page_size) < 0 || (c.dim != 64 && c.dim != 128 && c.dim != 256)) return false;
  // Pages are counted in 32 bits (a table's entries); places inside the cache are 64-bit.
  if (c.pages < 1 || c.pages > kIntMax || c.kv_heads < 1 || c.kv_heads > 65535) return false;
  for (const void *p : {c.key, c.key_scale, c.value, c.value_scale})
    if (!aligned16(p)) return false;
  out = Kv4Cache{static_cast<uint8_t *>(c.key), static_cast<uint8_t *>(c.key_scale), static_cast<uint8_t *>(c.value),
                 static_cast<uint8_t *>(c.value_scale), c.pages, (int32_t)c.kv_heads, (int32_t)c.dim,
                 page_shift(c.page_size)};
  return true;
}

// 16-byte rows: unit feature stride, other strides divisible by 8, aligned data.
bool rows_ok(const xinfer_view4 &t) {
  if (!aligned16(t.data) || (t.size[3] > 1 && t.stride[3] != 1)) return false;
  for (int i = 0; i < 3; ++i)
    if (t.size[i] > 1 && t.stride[i] % 8 != 0) return false;
  return true;
}

// key/value [B, Hkv, T, D] of the cache; D / 8 threads take each of B * T * heads rows.
bool new_tokens_ok(const xinfer_view4 &key, const xinfer_view4 &value, const Kv4Cache &cache, int64_t heads) {
  for (int i = 0; i < 4; ++i)
    if (key.size[i] < 0 || value.size[i] != key.size[i]) return false;
  return key.size[1] == cache.Hkv && key.size[3] == cache.D && key.size[0] <= kIntMax && key.size[2] <= kIntMax &&
         (key.size[0] == 0 || key.size[2] <= kIntMax / key.size[0]) &&
         key.size[0] * key.size[2] <= kIntMax / heads && launchable(key.size[0] * key.size[2] * heads * (cache.D / 8));
}

View view_of(const xinfer_view4 &t) {
  return View{static_cast<const uint16_t *>(t.data), t.stride[0], t.stride[1], t.stride[2]};
}

// Launches and workspace of a paged attention call come from the shapes and the bound on the lengths alone.
constexpr int kPagedCus = 256;
constexpr int kRowGroups = 1;  // 64-key groups a wave of a decode block that takes a whole row

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Rows may be cut into runs of at least min_groups groups, for about `target` items; whole_groups: rows of no more are not
// cut, as the merge's launch costs more than it saves.
PagedLaunch paged_launch(const PagedArgs &shapes, int vectors_min, int vectors_max, int tile, int min_groups, int target,
                         int whole_groups) {
  PagedLaunch l{shapes, 0, 0, 0, 0, 8};
  l.a.vectors_min = vectors_min;
  l.a.vectors_max = vectors_max;
  l.a.tile = tile;
  l.a.target = target;
  l.tiles = (int)ceil_div(std::min<int64_t>((int64_t)shapes.T * shapes.G, vectors_max), tile);
  // A row and tile has at most one run more than its share of the target.
  const int64_t whole = (int64_t)shapes.B * shapes.cache.Hkv * l.tiles, groups = ceil_div(shapes.max_length, 64);
  const int64_t runs = groups <= whole_groups ? 1 : ceil_div(groups, min_groups);
  l.a.min_groups = runs <= 1 ? (int)std::max<int64_t>(groups, 1) : min_groups;
  l.items = runs <= 1 ? whole : std::min(whole * runs, whole + target);
  // A row is cut where it has more groups than a run, so its items are fewer than twice its share of the target.
  l.records = runs <= 1 ? 0 : std::min(l.items, 2 * (int64_t)target);
  l.bytes = (size_t)l.records * tile * (shapes.cache.D + 2) * sizeof(float);
  return l;
}

// Decode blocks and items.  One column group: blocks of 4 waves and items enough to fill the chip (16 waves a CU up to
// 128 features, 8 of 256), since single waves wait for memory and LDS most of the time; runs of two groups a wave, or of
// one where all those items have a CU of their own.  (8 ragged rows, 128 features: 17.9 us, with 8 waves 19.2, now 17.0; one row
// of 1024 keys: runs of one group 10.8 us, of two 12.1.)  Two column groups: blocks of 8 waves, one a CU, all at once
// (six tokens in 8 rows, 32 / 8 heads: 25.4 us, with 4 waves and two blocks a CU 27.5).  In a prefill launch: its
// blocks' 8 waves.
//
// Rows of 9 to some 16 groups, in no more blocks than CUs, are not cut: a block of all 16 waves a CU holds spares the merge's
// launch, but the CU needs 0.35 us a group (64 features: 0.2), so the limit is higher where the cut rows' groups would
// share CUs too.  (128 features, 8 KV heads, 12 groups: 1 row 10.4 us, cut 10.3; 16 rows 11.0, cut 11.9; 32 rows 11.8, cut
// 14.6.  16 groups: 16 rows 12.4, cut 12.1; 24 rows 12.8, cut 14.8.  64 features, 16 groups: 1 row 8.4, cut 9.1; 32 rows
// 9.3, cut 12.1.  256 features hold 8 waves only, 16 groups: 15.7, cut 12.3.)
PagedLaunch paged_decode_launch(const PagedArgs &shapes, int vectors_max, int tile, bool alone) {
  const int64_t whole = (int64_t)shapes.B * shapes.cache.Hkv * ceil_div(std::min(shapes.T * shapes.G, vectors_max), tile);
  const int64_t groups = ceil_div(shapes.max_length, 64);
  const int row_groups = (shapes.cache.D == 64 ? 16 : 12) * (whole > kPagedCus / 2 ? 4 : 3) / 3;
  const bool rows = alone && tile == 16 && shapes.cache.D < 256 && whole <= kPagedCus && groups > 8 && groups <= row_groups;
  const int waves = rows ? kPagedRowWaves : alone && tile == 16 ? 4 : 8;
  const int64_t resident = kPagedCus * (waves == 8 ? 1 : shapes.cache.D == 256 ? 2 : 4);
  const int64_t target = waves == 4 ? resident : std::max(resident - whole, resident / 2);
  const bool spread = waves == 4 && whole * ceil_div(shapes.max_length, 64 * waves) <= kPagedCus;
  PagedLaunch l = paged_launch(shapes, 0, vectors_max, tile, spread ? waves : 8, (int)target, rows ? (int)groups : 8);
  l.waves = waves;
  return l;
}

int paged_launchable(const PagedLaunches &call) {
  return launchable((call.few.items + call.many.items) * 1024) &&
                 launchable(call.few.a.B * (call.few_merges() + call.many_merges()) * kMergeThreads)
             ? XINFER_OK
             : XINFER_ERR_KV4_SHAPE;
}

int paged_call(const xinfer_view4 &q, const xinfer_kv4_cache &cache, int64_t table_width, int64_t max_length,
               PagedLaunches &call) {
  PagedArgs a{};
  if (!cache_of(cache, a.cache)) return XINFER_ERR_KV4_CACHE;
  const int64_t B = q.size[0], Hq = q.size[1], T = q.size[2];
  if (B < 0 || B > kMostRows || T < 0 || q.size[3] != a.cache.D) return XINFER_ERR_KV4_SHAPE;
  if (Hq < 1 || Hq > 65535 || Hq % a.cache.Hkv != 0) return XINFER_ERR_HEADS;
  if (table_width < 1 || table_width > kMostTokens >> a.cache.page_shift || max_length < 0) return XINFER_ERR_PAGES;
  // Query vectors and items are counted in 32 bits.
  if (T > (kIntMax >> 8) / Hq || B * Hq * T > kIntMax >> 4) return XINFER_ERR_KV4_SHAPE;
  const int64_t capacity = table_width << a.cache.page_shift;
  a.B = (int32_t)B;
  a.Hq = (int32_t)Hq;
  a.G = (int32_t)(Hq / a.cache.Hkv);
  a.T = (int32_t)T;
  a.width = (int32_t)table_width;
  a.max_length = (int32_t)(max_length == 0 ? capacity : std::min(max_length, capacity));
  const int columns = paged_decode_columns(a.cache.D), vectors = a.T * a.G;
  call.many = PagedLaunch{a, 0, 0, 0, 0, 8};
  if (vectors <= 32) {
    call.few = paged_decode_launch(a, 32, vectors <= 16 ? 16 : columns, true);
    return paged_launchable(call);
  }
  // Rows of more vectors than a decode item has go to the prefill kernel; one row alone does whatever its count.
  const bool alone = B == 1;
  call.few = alone ? PagedLaunch{a, 0, 0, 0, 0, 8} : paged_decode_launch(a, columns, columns, false);
  call.many = paged_launch(a, alone ? 0 : columns + 1, kIntMax, kPagedPrefillTile, 8, alone || B > 64 ? kPagedCus : 3 * kPagedCus, 8);
  if (!alone) {
    // A record of 128 vectors is written and read at some 5 TB/s; a group of an item takes about 2 us.
    if (B <= 64) call.many.a.record_groups = kPagedPrefillTile * 8.0f * (float)a.cache.D / 5e6f / 2.0f;
  }
  return paged_launchable(call);
}

int done(hipError_t e) { return e == hipSuccess ? XINFER_OK : XINFER_ERR_LAUNCH; }

}  // namespace
}  // namespace xattn

using namespace xattn;

extern "C" {

int xinfer_paged_kv_reserve(const int32_t *kv_before, const int32_t *kv_lengths, const int32_t *query_lengths,
                            int64_t rows, int64_t tokens, int64_t page_size, const int64_t *counters,
                            int32_t *block_table, int64_t table_width, int32_t *free_pages, int64_t ring_size,
                            int32_t *lengths, int64_t *positions, int64_t *slots, int64_t *new_counters,
                            void *stream) {
  const int shift = page_shift(page_size);
  if (shift < 0 || table_width < 1 || table_width > kMostTokens >> shift || ring_size < 1 || ring_size > kIntMax)
    return XINFER_ERR_PAGES;
  if (rows < 0 || tokens < 0 || tokens > kIntMax) return XINFER_ERR_ARGUMENT;
  if (rows > kIntMax / table_width) return XINFER_ERR_PAGES;
  if (rows > kMostRows) return XINFER_ERR_ARGUMENT;
  if (!counters || !new_counters || counters == new_counters) return XINFER_ERR_ARGUMENT;
  if (rows > 0 && (!kv_before || !kv_lengths || !query_lengths || !block_table || !free_pages || !lengths))
    return XINFER_ERR_ARGUMENT;
  if (rows > 0 && tokens > 0 && (!positions || !slots)) return XINFER_ERR_ARGUMENT;
  const ReserveArgs a{kv_before, kv_lengths, query_lengths, counters, block_table, free_pages, lengths, positions, slots,
                      new_counters, ring_size, (int32_t)rows, (int32_t)tokens, (int32_t)table_width, shift};
  return done(launch_reserve(a, static_cast<hipStream_t>(stream)));
}

int xinfer_append_kv4(const xinfer_view4 *key, const xinfer_view4 *value, const int64_t *slots,
                      int64_t slot_stride_b, int64_t slot_stride_t, const xinfer_kv4_cache *cache, void *stream) {
  if (!key || !value || !cache) return XINFER_ERR_ARGUMENT;
  Kv4AppendArgs a{};
  if (!cache_of(*cache, a.cache)) return XINFER_ERR_KV4_CACHE;
  if (!new_tokens_ok(*key, *value, a.cache, a.cache.Hkv)) return XINFER_ERR_KV4_SHAPE;
  if (key->size[0] == 0 || key->size[2] == 0) return XINFER_OK;
  if (!slots) return XINFER_ERR_ARGUMENT;
  if (!rows_ok(*key) || !rows_ok(*value)) return XINFER_ERR_LAYOUT;
  a.key = view_of(*key);
  a.value = view_of(*value);
  a.slots = slots;
  a.slot_sb = slot_stride_b;
  a.slot_st = slot_stride_t;
  a.B = (int32_t)key->size[0];
  a.T = (int32_t)key->size[2];
  return done(launch_append_kv4(a, static_cast<hipStream_t>(stream)));
}

int xinfer_read_kv4(const xinfer_kv4_cache *cache, const int64_t *slots, int64_t slot_stride_b,
                    int64_t slot_stride_t, int64_t batch, int64_t tokens, void *key, void *value, void *stream) {
  if (!cache) return XINFER_ERR_ARGUMENT;
  Kv4ReadArgs a{};
  if (!cache_of(*cache, a.cache)) return XINFER_ERR_KV4_CACHE;
  const xinfer_view4 out{key, {batch, cache->kv_heads, tokens, cache->dim}, {0, 0, 0, 1}};
  if (!new_tokens_ok(out, out, a.cache, a.cache.Hkv)) return XINFER_ERR_KV4_SHAPE;
  if (batch == 0 || tokens == 0) return XINFER_OK;
  if (!slots) return XINFER_ERR_ARGUMENT;
  if (!aligned16(key) || !aligned16(value)) return XINFER_ERR_LAYOUT;
  a.slots = slots;
  a.slot_sb = slot_stride_b;
  a.slot_st = slot_stride_t;
  a.key = static_cast<uint16_t *>(key);
  a.value = static_cast<uint16_t *>(value);
  a.B = (int32_t)batch;
  a.T = (int32_t)tokens;
  return done(launch_read_kv4(a, static_cast<hipStream_t>(stream)));
}

int xinfer_qk_norm_rope_append_kv4(const xinfer_view4 *q, const xinfer_view4 *key, const xinfer_view4 *value,
                                   const void *q_weight, const void *k_weight, double eps, double weight_offset,
                                   const xinfer_view4 *cos, const xinfer_view4 *sin, const int64_t *slots,
                                   int64_t slot_stride_b, int64_t slot_stride_t, void *q_out,
                                   const xinfer_kv4_cache *cache, void *stream) {
  if (!q || !key || !value || !cos || !sin || !cache) return XINFER_ERR_ARGUMENT;
  Kv4NormRopeArgs a{};
  if (!cache_of(*cache, a.cache)) return XINFER_ERR_KV4_CACHE;
  const int64_t B = key->size[0], T = key->size[2], Hq = q->size[1], R = cos->size[3];
  if (q->size[0] != B || q->size[2] != T || q->size[3] != a.cache.D || Hq < 1 || Hq > 65535 ||
      !new_tokens_ok(*key, *value, a.cache, Hq + a.cache.Hkv + 128 / (a.cache.D / 8)) || R < 16 || R > a.cache.D || R % 16 != 0)
    return XINFER_ERR_KV4_SHAPE;
  for (const xinfer_view4 *r : {cos, sin})
    if (r->size[0] != B || r->size[1] != 1 || r->size[2] != T || r->size[3] != R) return XINFER_ERR_KV4_SHAPE;
  if (!(std::isfinite(eps) && eps >= 0)) return XINFER_ERR_EPS;
  if (!std::isfinite(weight_offset)) return XINFER_ERR_ARGUMENT;
  if (B == 0 || T == 0) return XINFER_OK;
  if (!q_weight || !k_weight || !slots || !q_out) return XINFER_ERR_ARGUMENT;
  for (const xinfer_view4 *t : {q, key, value, cos, sin})
    if (!rows_ok(*t)) return XINFER_ERR_LAYOUT;
  for (const void *p : {q_weight, k_weight, static_cast<const void *>(q_out)})
    if (!aligned16(p)) return XINFER_ERR_LAYOUT;
  a.q = view_of(*q);
  a.k = view_of(*key);
  a.v = view_of(*value);
  a.q_weight = static_cast<const uint16_t *>(q_weight);
  a.k_weight = static_cast<const uint16_t *>(k_weight);
  a.cos = view_of(*cos);
  a.sin = view_of(*sin);
  a.slots = slots;
  a.slot_sb = slot_stride_b;
  a.slot_st = slot_stride_t;
  a.q_out = static_cast<uint16_t *>(q_out);
  a.eps = (float)eps;
  a.offset = (float)weight_offset;
  a.B = (int32_t)B;
  a.T = (int32_t)T;
  a.Hq = (int32_t)Hq;
  a.R = (int32_t)R;
  return done(launch_norm_rope_kv4(a, static_cast<hipStream_t>(stream)));
}

size_t xinfer_paged_attention_kv4_workspace_size(const xinfer_view4 *q, const xinfer_kv4_cache *cache,
                                                 int64_t table_width, int64_t max_length) {
  PagedLaunches call{};
  if (!q || !cache || paged_call(*q, *cache, table_width, max_length, call) != XINFER_OK) return 0;
  return call.bytes();
}

int xinfer_paged_attention_kv4(const xinfer_view4 *q, const xinfer_kv4_cache *cache, const int32_t *block_table,
                               int64_t table_width, const int32_t *lengths, int64_t max_length, double scale,
                               void *out, void *workspace, size_t workspace_bytes, void *stream) {
  if (!q || !cache) return XINFER_ERR_ARGUMENT;
  PagedLaunches call{};
  const int status = paged_call(*q, *cache, table_width, max_length, call);
  if (status != XINFER_OK) return status;
  if (!(std::isfinite(scale) && scale > 0)) return XINFER_ERR_SCALE;
  if (q->size[0] == 0 || q->size[2] == 0) return XINFER_OK;
  if (!block_table || !lengths || !out) return XINFER_ERR_ARGUMENT;
  if (!rows_ok(*q) || !aligned16(out)) return XINFER_ERR_LAYOUT;
  if (call.bytes() > 0 && (!aligned16(workspace) || workspace_bytes < call.bytes())) return XINFER_ERR_WORKSPACE;
  uint8_t *records = static_cast<uint8_t *>(workspace);
  for (PagedLaunch *l : {&call.few, &call.many}) {
    l->a.q = view_of(*q);
    l->a.table = block_table;
    l->a.lengths = lengths;
    l->a.out = static_cast<uint16_t *>(out);
    l->a.scale_log2 = (float)(scale * 1.4426950408889634);
    l->a.part_o = reinterpret_cast<float *>(records);
    l->a.part_ml = l->a.part_o + l->records * l->a.tile * l->a.cache.D;
    records += l->bytes;
  }
  return done(launch_paged_attention(call, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
