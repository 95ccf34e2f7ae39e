/*
 * C ABI of libxinfer_attention_ops.so: attention over each request's populated
 * KV prefix and the in-place KV-cache append, for AMD MI355X (gfx950).
 *
 * Every entry point takes plain device pointers, element strides and host-side
 * lengths; none allocates device memory and none synchronises the host with the
 * device.  Work is enqueued on `stream` (a hipStream_t; NULL is the null stream).
 * Tensors are bf16 (stored as raw uint16 bits).  Return value: 0 on success, or
 * a status code whose message `xinfer_status_string` returns.  The messages
 * reproduce the reference operator's TORCH_CHECK texts where one exists.
 *
 * The torch.library operators and the AOTInductor C shims that the reference
 * exports are defined in the same library; they validate torch-specific
 * properties and call the entry points below.
 */
#ifndef XINFER_ATTENTION_H
#define XINFER_ATTENTION_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Status codes.  Messages (xinfer_status_string) follow the reference:
 * compiler/common/kernels/attention.cpp:17-35 and :84-104. */
enum {
  XINFER_OK = 0,
  XINFER_ERR_QKV_SHAPES = 1,      /* "Invalid Q/K/V shapes"                        attention.cpp:17-19 */
  XINFER_ERR_Q_SHAPE = 2,         /* "Unsupported Q shape"                         attention.cpp:90-91 */
  XINFER_ERR_KV_SHAPE = 3,        /* "Expected matching full-capacity K/V ..."     attention.cpp:92-94 */
  XINFER_ERR_HEADS = 4,           /* "Query heads must be a positive multiple ..." attention.cpp:95-96 */
  XINFER_ERR_HEAD_DIM = 5,        /* "Flash head dimension must be ..."            attention.cpp:97-98 */
  XINFER_ERR_PREFIX = 6,          /* "Invalid valid-prefix length"                 attention.cpp:102 */
  XINFER_ERR_SCALE = 7,           /* "Attention scale must be finite and positive" attention.cpp:103 */
  XINFER_ERR_OFFSETS_START = 8,   /* "Cumulative lengths must start at zero"       attention.cpp:35 */
  XINFER_ERR_LENGTHS = 9,         /* "Invalid query/KV lengths"                    attention.cpp:43-45 */
  XINFER_ERR_WORKSPACE = 10,      /* workspace smaller than its *_workspace_size, or not 16-byte aligned */
  XINFER_ERR_LAYOUT = 11,         /* feature stride != 1 or rows not 16-byte aligned */
  XINFER_ERR_CACHE = 12,          /* cache tensors not contiguous [B,H,C,D] / shape mismatch */
  XINFER_ERR_LAUNCH = 13,         /* a HIP kernel launch failed */
  XINFER_ERR_ARGUMENT = 14,       /* null pointer, negative size or stride, misaligned page table */
  XINFER_ERR_ROPE_SHAPE = 15,     /* xinfer_qk_norm_rope_append shapes (no reference message) */
  XINFER_ERR_EPS = 16,            /* RMSNorm epsilon not finite and >= 0 (no reference message) */
  XINFER_ERR_SCRATCH = 17,        /* the call needs more than XINFER_NOALLOC_SCRATCH_BYTES of scratch */
  XINFER_ERR_CAPTURE_ROWS = 18,   /* graph-capture mode: more than 64 rows */
  XINFER_ERR_KV4_CACHE = 19,      /* 4-bit cache: head dim, page size, alignment or size */
  XINFER_ERR_KV4_SHAPE = 20,      /* 4-bit cache: tensors that do not match it or each other */
  XINFER_ERR_PAGES = 21           /* page tables: page size, table width or ring size */
};

/* A strided rank-4 view of bf16 device memory, [batch, heads, sequence, dim].
 * Strides are in elements.  The attention kernels need stride[3] == 1, the
 * other strides multiples of 8 and `data` 16-byte aligned (XINFER_ERR_LAYOUT
 * otherwise); the append kernel accepts any strides for key/value. */
typedef struct xinfer_view4 {
  const void *data;
  int64_t size[4];
  int64_t stride[4];
} xinfer_view4;

/* Message for a status code (static storage, never NULL). */
const char *xinfer_status_string(int status);

/* ---------------------------------------------------------------------------
 * xinfer::flash_attention -- replaces compiler/common/kernels/attention.cpp:82-124
 * (schema :133-134, fake compiler/common/attention.py:63-83).
 *
 * q [B,Hq,T,D], k/v [B,Hkv,C,D]; every row attends with all T queries over the
 * first `valid_length` cache positions, lower-right causal: query i sees keys
 * j <= valid_length - T + i.  out: contiguous [B,Hq,T,D] bf16, written fully.
 * ------------------------------------------------------------------------- */
size_t xinfer_flash_attention_workspace_size(const xinfer_view4 *q, const xinfer_view4 *k,
                                             int64_t valid_length);
int xinfer_flash_attention(const xinfer_view4 *q, const xinfer_view4 *k, const xinfer_view4 *v,
                           int64_t valid_length, double scale, void *out, void *workspace,
                           size_t workspace_bytes, void *stream);

/* ---------------------------------------------------------------------------
 * xinfer::batched_flash_attention -- replaces attention.cpp:14-79
 * (schema :129-131, fake compiler/common/attention.py:86-94).
 *
 * host_offsets: host int32 [2][B+1]; row 0 = cumulative real-query counts,
 * row 1 = cumulative populated KV lengths (both start at 0), exactly the CPU
 * `offsets` tensor of batched_attention_metadata (attention.py:27-40).  Row r
 * attends with its first count_r queries over k/v[r, :, :L_r], lower-right
 * causal; out[r, :, count_r:] is written as zeros.
 *
 * blocks: NULL, or the DEVICE int32 page table of attention.cpp:39-40, 56-58,
 * 68-70, one entry per row at blocks[r * blocks_stride] (blocks_stride >= 0,
 * the table's row stride; 4-byte aligned): row r then reads its keys and
 * values from k/v[blocks[r]] instead of k/v[r], each entry clamped into
 * [0, B).  The reference applies its table only when the cache capacity C is
 * a multiple of 256; xinfer::batched_flash_attention passes it under that
 * condition and NULL otherwise.  The kernels read it on the device: the
 * identity table costs one scalar read per work item.
 * ------------------------------------------------------------------------- */
size_t xinfer_batched_flash_attention_workspace_size(const xinfer_view4 *q, const xinfer_view4 *k,
                                                     const int32_t *host_offsets);
int xinfer_batched_flash_attention(const xinfer_view4 *q, const xinfer_view4 *k,
                                   const xinfer_view4 *v, const int32_t *host_offsets,
                                   const int32_t *blocks, int64_t blocks_stride, double scale,
                                   void *out, void *workspace, size_t workspace_bytes, void *stream);

/* Same operation with the output written through a caller-supplied view of
 * q's sizes [B,Hq,T,D] (unit feature stride, other strides multiples of 8,
 * 16-byte aligned data), e.g. [B,T,Hq,D] storage viewed as [B,Hq,T,D].  The
 * view's elements must be distinct and must not overlap q, k, v or the
 * workspace.  The workspace is the one *_workspace_size reports.  No reference counterpart:
 * it serves xinfer::batched_flash_attention_bthd, the optional variant that
 * spares compiler/qwen3/adapters/attention.py:61 its transpose copy. */
int xinfer_batched_flash_attention_out(const xinfer_view4 *q, const xinfer_view4 *k,
                                       const xinfer_view4 *v, const int32_t *host_offsets,
                                       const int32_t *blocks, int64_t blocks_stride,
                                       double scale, const xinfer_view4 *out, void *workspace,
                                       size_t workspace_bytes, void *stream);

/* Graph-capture ("capture once, replay every step") variant of
 * xinfer_batched_flash_attention.  No counterpart in the reference, which
 * leaves graph capture to future runtime work (PLAN.md:35-37): it is for
 * serving loops that capture one step in a HIP graph and replay it while the
 * lengths change.  device_offsets is the DEVICE copy of
 * the cumulative offsets (int32 [2][B+1], batched_attention_metadata's
 * cuda_offsets); the kernels read every row's count and length from it when
 * they run, so nothing about the launch depends on host lengths and a
 * captured call stays valid after the caller rewrites device_offsets in place
 * (and the page table, read the same way).
 * The workspace size depends on the shapes only (all rows at capacity C).
 * Shapes with T * (Hq/Hkv) <= 8 take the decode kernels; larger ones take the
 * prefill kernels, whose key split size, work list and XCD runs a plan kernel
 * chooses from device_offsets at run time and writes into the workspace (at
 * most 8 splits a row; the workspace holds records for the most items such a
 * plan can make).  B <= 64 (XINFER_ERR_CAPTURE_ROWS otherwise).  Device lengths are not validated on
 * the host: counts are clamped to [0, min(T, C)] and lengths to [max(count, 1), C], so
 * bad values give wrong rows but never an access outside the tensors.
 * Results agree with xinfer_batched_flash_attention within rounding; the
 * kernels are the same, but every launch covers the capacity. */
size_t xinfer_batched_flash_attention_graph_workspace_size(const xinfer_view4 *q, const xinfer_view4 *k);
int xinfer_batched_flash_attention_graph(const xinfer_view4 *q, const xinfer_view4 *k, const xinfer_view4 *v,
                                         const int32_t *device_offsets, const int32_t *blocks,
                                         int64_t blocks_stride, double scale, void *out, void *workspace,
                                         size_t workspace_bytes, void *stream);

/* Allocation-free variant of xinfer_batched_flash_attention.  No counterpart in
 * the reference: it is for callers that cannot allocate device memory or pass
 * a workspace -- code under HIP graph capture, tight serving loops, harnesses
 * that forbid hipMalloc.  Same arguments, checks, kernels and results as
 * xinfer_batched_flash_attention, bit for bit; the split records go to a
 * static device array of the library (one per GPU, held until the process
 * ends) instead of a caller's workspace, and the call allocates nothing.
 * A call whose records (the size xinfer_batched_flash_attention_workspace_size
 * reports) exceed XINFER_NOALLOC_SCRATCH_BYTES splits its rows of up to 32 query
 * vectors per KV head less, which is slower and rounds differently; if the
 * other rows' records alone exceed it, the call returns XINFER_ERR_SCRATCH and
 * launches nothing.  The current device must be the
 * stream's.  Calls that overlap in time on one GPU share its array and race:
 * order them on one stream. */
#define XINFER_NOALLOC_SCRATCH_BYTES (32u << 20)
int xinfer_batched_flash_attention_noalloc(const xinfer_view4 *q, const xinfer_view4 *k,
                                           const xinfer_view4 *v, const int32_t *host_offsets,
                                           const int32_t *blocks, int64_t blocks_stride,
                                           double scale, void *out, void *stream);

/* ---------------------------------------------------------------------------
 * xinfer::append_kv_batched -- replaces the Triton op
 * compiler/common/kernels/kv_cache.py:8-72.
 *
 * cache_key[r,h,positions[r,t],:] = key[r,h,t,:] (same for value) for
 * t < count_r = cu_query[r+1] - cu_query[r]; positions of padded tokens are
 * not used (they are loaded with the rest, so every one of the B*T entries
 * must be readable).  positions: device int64 [B,T] with strides
 * (pos_stride_b, pos_stride_t); cu_query: device int32 [B+1].  Caches are contiguous
 * [B,Hkv,C,D] bf16 and are the only memory written.  A position outside
 * [0, C) is skipped instead of being written out of bounds.
 * ------------------------------------------------------------------------- */
int xinfer_append_kv_batched(const xinfer_view4 *key, const xinfer_view4 *value,
                             const int64_t *positions, int64_t pos_stride_b, int64_t pos_stride_t,
                             const int32_t *cu_query, const xinfer_view4 *cache_key,
                             const xinfer_view4 *cache_value, void *stream);

/* ---------------------------------------------------------------------------
 * xinfer::qk_norm_rope_append -- replaces the eager step before the attention
 * operator, compiler/qwen3/adapters/attention.py:44-51 (q_norm/k_norm, i.e.
 * transformers Qwen3RMSNorm, then apply_rotary_pos_emb, then
 * KVCache.update = append_kv_batched, compiler/qwen3/model.py:49-52).
 *
 * q [B,Hq,T,D], key/value [B,Hkv,T,D]: projections viewed per head (any
 * strides with unit feature stride, others divisible by 8, 16-byte aligned);
 * q_weight/k_weight: the [D] RMSNorm weights; cos/sin [B,1,T,D] (stride[1]
 * unused): the rotary tables of the tokens; D in {64, 128, 256}.
 *   xn = bf16(w * bf16(x * rsqrt(mean(x^2) + eps)))   per (token, head) row
 *   x' = bf16(bf16(xn * cos) + bf16(rotate_half(xn) * sin))
 * q_out: contiguous [B,Hq,T,D] receives q' for every token.  cache_key
 * receives k' and cache_value v at [r, h, positions[r,t]] for t < count_r
 * (count_r, positions and the skipping of positions outside [0, C) as in
 * xinfer_append_kv_batched).  No reference counterpart in the C ABI: the
 * reference runs this step as separate eager or compiled PyTorch ops.
 * ------------------------------------------------------------------------- */
int xinfer_qk_norm_rope_append(const xinfer_view4 *q, const xinfer_view4 *key, const xinfer_view4 *value,
                               const void *q_weight, const void *k_weight, double eps,
                               const xinfer_view4 *cos, const xinfer_view4 *sin, const int64_t *positions,
                               int64_t pos_stride_b, int64_t pos_stride_t, const int32_t *cu_query,
                               void *q_out, const xinfer_view4 *cache_key, const xinfer_view4 *cache_value,
                               void *stream);

/* ---------------------------------------------------------------------------
 * xinfer::projection_gemv -- replaces the Triton op
 * compiler/common/kernels/projection_gemv.py:10-62 (the decoder's singleton
 * projections, selected by compiler/common/passes/projection_gemv.py).
 *
 * out[i] = sum_j weight[i, j] * x[j] for i < n, j < k: x [k] contiguous,
 * weight [n, k] contiguous row-major, out [n]; all XINFER_BF16 or all
 * XINFER_FP32 (dtype), accumulated in fp32.  out must not overlap x or weight.
 * ------------------------------------------------------------------------- */
enum { XINFER_BF16 = 0, XINFER_FP32 = 1 };
int xinfer_projection_gemv(const void *x, const void *weight, void *out, int64_t n, int64_t k, int dtype,
                           void *stream);

/* ---------------------------------------------------------------------------
 * Paged 4-bit KV cache.  No reference counterpart: the reference holds bf16
 * caches of one page per row.
 *
 * A key or value vector is held as blocks of 32 features.  A feature takes
 * four bits, e2m1: a sign and a magnitude of 0, 0.5, 1, 1.5, 2, 3, 4 or 6, the
 * even feature in a byte's low half; a block has one scale byte s, for
 * 2^(s - 127).  A block whose largest magnitude is a has
 * s - 127 = e = floor(log2 a) - 2, one more where a > 7 * 2^e, kept in
 * [-125, 125]; a feature takes the value nearest to it, ties to the even code.
 * A token whose key or value has an infinity or a NaN holds zeros, and 255 in
 * all of its key's scales: queries that see it get NaN.  Value scales above
 * 252 (which no call writes) are read as 252.
 *
 * Pages of `page_size` tokens (64, 128 or 256): codes uint8
 * [pages][kv_heads][page_size][dim / 2], scales uint8
 * [pages][kv_heads][dim / 32][page_size], key and value apart, 16-byte
 * aligned; dim in {64, 128, 256}.  A slot is page * page_size + place.
 * ------------------------------------------------------------------------- */
typedef struct xinfer_kv4_cache {
  void *key, *key_scale, *value, *value_scale;
  int64_t pages, kv_heads, page_size, dim;
} xinfer_kv4_cache;

/* Pages, slots and positions of a step from the rows' lengths, on the device.
 * Row r held ceil(kv_before[r] / P) pages and is to hold ceil(kv_lengths[r] / P),
 * with its last query_lengths[r] tokens new.  free_pages is a ring with a place
 * for every page: entries counters[0] <= i < counters[1] (modulo ring_size) are
 * free.  Growing rows take pages from its head in row order into block_table
 * [rows][table_width]; shrinking rows (an ended request has length 0) put theirs
 * at its tail, for later calls.  A row whose pages, with those of the rows before
 * it, exceed the free ones, or that does not fit its table row, keeps its pages and
 * takes no part:
 * lengths[0][r] (new tokens) is 0 and lengths[1][r] is kv_before[r]; otherwise
 * they are query_lengths[r] and kv_lengths[r].  positions and slots [rows][tokens]
 * are written whole: of token t < lengths[0][r] the position kv_lengths[r] -
 * query_lengths[r] + t and its slot, else 0 and -1.  new_counters receives the
 * ring's head and tail; it must not be counters.  The same inputs give the same
 * results again.  Out-of-range lengths are clamped ([0, tokens] new tokens,
 * lengths of at least that), so no input reaches outside the arrays.
 * table_width * page_size is at most 2^30, rows at most 65535, rows * table_width
 * below 2^31. */
int xinfer_paged_kv_reserve(const int32_t *kv_before, const int32_t *kv_lengths, const int32_t *query_lengths,
                            int64_t rows, int64_t tokens, int64_t page_size, const int64_t *counters,
                            int32_t *block_table, int64_t table_width, int32_t *free_pages, int64_t ring_size,
                            int32_t *lengths, int64_t *positions, int64_t *slots, int64_t *new_counters,
                            void *stream);

/* Quantises key/value [B,Hkv,T,D] (bf16, layout as for attention tensors) into
 * slots [B,T] (device int64, strides in elements).  Slots outside the cache,
 * negative ones among them, are skipped.  The slots of one call are distinct; one
 * given twice holds a mixture of its tokens. */
int xinfer_append_kv4(const xinfer_view4 *key, const xinfer_view4 *value, const int64_t *slots,
                      int64_t slot_stride_b, int64_t slot_stride_t, const xinfer_kv4_cache *cache, void *stream);

/* What the cache holds at slots [B,T], as bf16 (exact): key and value contiguous
 * [B,Hkv,T,D], 16-byte aligned, zero for slots outside the cache, NaN for keys of
 * tokens that were not finite. */
int xinfer_read_kv4(const xinfer_kv4_cache *cache, const int64_t *slots, int64_t slot_stride_b,
                    int64_t slot_stride_t, int64_t batch, int64_t tokens, void *key, void *value, void *stream);

/* q/k RMSNorm, rotary embedding and append in one launch.  Per (token, head)
 * row: y = x * rsqrt(mean(x^2) + eps) * (weight + weight_offset), then the first
 * R features turn by cos/sin [B,1,T,R] (R = cos->size[3], a multiple of 16 up to D):
 * y_i cos_i - y_{i+R/2} sin_i for i < R/2, y_i cos_i + y_{i-R/2} sin_i for the
 * second half.  The query is computed in fp32 and rounded once into q_out, contiguous
 * [B,Hq,T,D], for every token; the key is quantised without a rounding in front
 * (where fp32 could decide a code, in 64 bits) and appended with the value as in
 * xinfer_append_kv4.  weight_offset: 0, or 1 for weights stored minus
 * one. */
int xinfer_qk_norm_rope_append_kv4(const xinfer_view4 *q, const xinfer_view4 *key, const xinfer_view4 *value,
                                   const void *q_weight, const void *k_weight, double eps, double weight_offset,
                                   const xinfer_view4 *cos, const xinfer_view4 *sin, const int64_t *slots,
                                   int64_t slot_stride_b, int64_t slot_stride_t, void *q_out,
                                   const xinfer_kv4_cache *cache, void *stream);

/* Attention over the cache: q [B,Hq,T,D]; row r's first lengths[0][r] queries see
 * its lengths[1][r] keys, lower-right causal (query i sees keys up to length -
 * count + i), key p in page block_table[r][p / P].  lengths is DEVICE int32 [2][B],
 * as xinfer_paged_kv_reserve writes it; the launch depends on the shapes and on
 * max_length alone, so a captured call serves every set of lengths up to it.
 * max_length: the host's bound on the rows' lengths (0: the table's
 * capacity); longer rows are read as max_length keys.  With M the smaller of
 * the two, counts are clamped to [0, min(T, M)] and lengths to [count, M].  Keys of table
 * entries outside the cache count as absent.  out: contiguous bf16 [B,T,Hq,D], zero
 * for padded queries and for queries that see no key.  The workspace is 16-byte
 * aligned and serves one call at a time. */
size_t xinfer_paged_attention_kv4_workspace_size(const xinfer_view4 *q, const xinfer_kv4_cache *cache,
                                                 int64_t table_width, int64_t max_length);
int xinfer_paged_attention_kv4(const xinfer_view4 *q, const xinfer_kv4_cache *cache, const int32_t *block_table,
                               int64_t table_width, const int32_t *lengths, int64_t max_length, double scale,
                               void *out, void *workspace, size_t workspace_bytes, void *stream);

/* The AOTInductor C shims of the same library are declared in
 * xinfer_attention_aoti.h. */

#ifdef __cplusplus
}
#endif

#endif /* XINFER_ATTENTION_H */
