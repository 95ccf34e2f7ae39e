// torch.library registration and AOTInductor C shims of the paged 4-bit KV cache: a thin layer over the C ABI
// (include/xinfer_attention.h), as torch_ops.cpp is over the other operators.  Outputs and workspaces come from the
// caching allocator, launches go to the current stream of the inputs' device.
#include <ATen/ATen.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/inductor/aoti_torch/utils.h>
#include <torch/library.h>

#include <cmath>
#include <initializer_list>
#include <tuple>

#include "xinfer_attention.h"
#include "xinfer_attention_aoti.h"

namespace xinfer {
namespace {

using Tensors = std::initializer_list<const at::Tensor *>;

// A view of `t` [B, H, T, D] or, with `token_major`, of `t` [B, T, H, D] as [B, H, T, D]: no tensor is made for it.
xinfer_view4 view4(const at::Tensor &t, bool token_major = false) {
  xinfer_view4 v{};
  v.data = t.data_ptr();
  const int order[4] = {0, token_major ? 2 : 1, token_major ? 1 : 2, 3};
  for (int i = 0; i < 4; ++i) {
    v.size[i] = t.size(order[i]);
    v.stride[i] = t.stride(order[i]);
  }
  return v;
}
// `t` [B, T, R] as [B, 1, T, R].
xinfer_view4 view3(const at::Tensor &t) {
  return xinfer_view4{t.data_ptr(), {t.size(0), 1, t.size(1), t.size(2)}, {t.stride(0), 0, t.stride(1), t.stride(2)}};
}

// Rows the kernels read in place: unit feature stride, other strides divisible by 8, 16-byte aligned data; others
// are copied.
at::Tensor in_rows(const at::Tensor &t) {
  const int64_t last = t.dim() - 1;
  bool fine = (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0 && (t.size(last) <= 1 || t.stride(last) == 1);
  for (int64_t i = 0; i < last; ++i) fine = fine && (t.size(i) <= 1 || t.stride(i) % 8 == 0);
  return fine ? t : t.clone(at::MemoryFormat::Contiguous);
}

// A tensor on `like`'s device straight from the allocator (a call through the dispatcher takes twice the time).
at::Tensor new_tensor(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor &like) {
  return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}

void *stream_of(const at::Tensor &t) {
  return static_cast<void *>(c10::hip::getCurrentHIPStream(t.device().index()).stream());
}

void check_status(int status) { TORCH_CHECK(status == XINFER_OK, xinfer_status_string(status)); }

void check_colocated(const at::Tensor &first, Tensors others) {
  bool fine = first.is_cuda();
  for (const at::Tensor *t : others) fine = fine && t->device() == first.device();
  TORCH_CHECK(fine, "xinfer paged KV cache requires colocated CUDA tensors");
}

void check_bf16(Tensors tensors) {
  for (const at::Tensor *t : tensors)
    TORCH_CHECK(t->scalar_type() == at::kBFloat16, "xinfer paged KV cache requires BF16 activations and weights");
}

// Weights may ask for gradients, as a model's do outside of training.
void check_inference(Tensors activations) {
  for (const at::Tensor *t : activations)
    TORCH_CHECK(!t->requires_grad(), "xinfer paged KV cache supports inference only");
}

xinfer_kv4_cache cache_of(const at::Tensor &key, const at::Tensor &key_scale, const at::Tensor &value,
                          const at::Tensor &value_scale) {
  bool fine = true;
  for (const at::Tensor *t : {&key, &key_scale, &value, &value_scale})
    fine = fine && t->scalar_type() == at::kByte && t->dim() == 4 && t->is_contiguous() && t->device() == key.device();
  TORCH_CHECK(fine, "Expected contiguous uint8 cache tensors of four dimensions on one device");
  TORCH_CHECK(value.sizes() == key.sizes() && value_scale.sizes() == key_scale.sizes() &&
                  key_scale.size(0) == key.size(0) && key_scale.size(1) == key.size(1) &&
                  key_scale.size(3) == key.size(2) && key_scale.size(2) * 16 == key.size(3),
              "Expected cache codes [N,Hkv,P,D/2] and scales [N,Hkv,D/32,P]");
  return xinfer_kv4_cache{key.data_ptr(),  key_scale.data_ptr(), value.data_ptr(), value_scale.data_ptr(),
                          key.size(0),     key.size(1),          key.size(2),      2 * key.size(3)};
}

void check_slots(const at::Tensor &slots, int64_t batch, int64_t tokens) {
  TORCH_CHECK(slots.scalar_type() == at::kLong && slots.dim() == 2 && slots.size(0) == batch && slots.size(1) == tokens,
              "Expected int64 slots [B,T]");
}

}  // namespace

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> paged_kv_reserve(
    const at::Tensor &kv_before, const at::Tensor &kv_lengths, const at::Tensor &query_lengths, int64_t tokens,
    int64_t page_size, const at::Tensor &counters, const at::Tensor &block_table, const at::Tensor &free_pages) {
  check_colocated(kv_before, {&kv_lengths, &query_lengths, &counters, &block_table, &free_pages});
  TORCH_CHECK(kv_before.dim() == 1, "Expected int32 row lengths [B]");
  const int64_t rows = kv_before.size(0);
  for (const at::Tensor *t : {&kv_before, &kv_lengths, &query_lengths})
    TORCH_CHECK(t->scalar_type() == at::kInt && t->dim() == 1 && t->size(0) == rows, "Expected int32 row lengths [B]");
  TORCH_CHECK(counters.scalar_type() == at::kLong && counters.dim() == 1 && counters.size(0) == 2 &&
                  counters.is_contiguous(),
              "Expected int64 counters [2]");
  TORCH_CHECK(block_table.scalar_type() == at::kInt && block_table.dim() == 2 && block_table.size(0) == rows &&
                  block_table.is_contiguous(),
              "Expected a contiguous int32 block table [B,M]");
  TORCH_CHECK(free_pages.scalar_type() == at::kInt && free_pages.dim() == 1 && free_pages.is_contiguous(),
              "Expected a contiguous int32 ring of free pages");
  TORCH_CHECK(tokens >= 0, "Expected a number of new tokens");
  c10::DeviceGuard guard(kv_before.device());
  auto before = kv_before.contiguous(), after = kv_lengths.contiguous(), counts = query_lengths.contiguous();
  auto lengths = new_tensor({2, rows}, at::kInt, counters);
  auto positions = new_tensor({rows, tokens}, at::kLong, counters), slots = new_tensor({rows, tokens}, at::kLong, counters);
  auto next = new_tensor({2}, at::kLong, counters);
  auto ints = [](const at::Tensor &t) { return static_cast<int32_t *>(t.data_ptr()); };
  auto longs = [](const at::Tensor &t) { return static_cast<int64_t *>(t.data_ptr()); };
  check_status(xinfer_paged_kv_reserve(ints(before), ints(after), ints(counts), rows, tokens, page_size, longs(counters),
                                       ints(block_table), block_table.size(1), ints(free_pages), free_pages.size(0),
                                       ints(lengths), longs(positions), longs(slots), longs(next),
                                       stream_of(kv_before)));
  return {lengths, positions, slots, next};
}

void append_kv4(const at::Tensor &key, const at::Tensor &value, const at::Tensor &slots, const at::Tensor &key_codes,
                const at::Tensor &key_scales, const at::Tensor &value_codes, const at::Tensor &value_scales) {
  check_colocated(key, {&value, &slots, &key_codes, &key_scales, &value_codes, &value_scales});
  TORCH_CHECK(key.dim() == 4 && value.sizes() == key.sizes(), "Expected key/value [B,Hkv,T,D]");
  check_bf16({&key, &value});
  check_inference({&key, &value});
  check_slots(slots, key.size(0), key.size(2));
  const auto cache = cache_of(key_codes, key_scales, value_codes, value_scales);
  c10::DeviceGuard guard(key.device());
  auto k = in_rows(key), v = in_rows(value);
  auto kv = view4(k), vv = view4(v);
  check_status(xinfer_append_kv4(&kv, &vv, static_cast<const int64_t *>(slots.data_ptr()), slots.stride(0),
                                 slots.stride(1), &cache, stream_of(key)));
}

std::tuple<at::Tensor, at::Tensor> read_kv4(const at::Tensor &key_codes, const at::Tensor &key_scales,
                                            const at::Tensor &value_codes, const at::Tensor &value_scales,
                                            const at::Tensor &slots) {
  check_colocated(key_codes, {&key_scales, &value_codes, &value_scales, &slots});
  TORCH_CHECK(slots.scalar_type() == at::kLong && slots.dim() == 2, "Expected int64 slots [B,T]");
  const auto cache = cache_of(key_codes, key_scales, value_codes, value_scales);
  c10::DeviceGuard guard(slots.device());
  auto key = new_tensor({slots.size(0), cache.kv_heads, slots.size(1), cache.dim}, at::kBFloat16, slots);
  auto value = new_tensor(key.sizes(), at::kBFloat16, slots);
  check_status(xinfer_read_kv4(&cache, static_cast<const int64_t *>(slots.data_ptr()), slots.stride(0), slots.stride(1),
                               slots.size(0), slots.size(1), key.data_ptr(), value.data_ptr(), stream_of(slots)));
  return {key, value};
}

at::Tensor qk_norm_rope_append_kv4(const at::Tensor &q, const at::Tensor &key, const at::Tensor &value,
                                   const at::Tensor &q_weight, const at::Tensor &k_weight, double eps,
                                   double weight_offset, const at::Tensor &cos, const at::Tensor &sin,
                                   const at::Tensor &slots, const at::Tensor &key_codes, const at::Tensor &key_scales,
                                   const at::Tensor &value_codes, const at::Tensor &value_scales) {
  check_colocated(q, {&key, &value, &q_weight, &k_weight, &cos, &sin, &slots, &key_codes, &key_scales, &value_codes,
                      &value_scales});
  TORCH_CHECK(q.dim() == 4 && key.dim() == 4 && value.sizes() == key.sizes() && key.size(0) == q.size(0) &&
                  key.size(1) == q.size(1) && key.size(3) == q.size(3) && cos.dim() == 3 && cos.sizes() == sin.sizes() &&
                  cos.size(0) == q.size(0) && cos.size(1) == q.size(1) && q_weight.dim() == 1 &&
                  q_weight.size(0) == q.size(3) && k_weight.sizes() == q_weight.sizes(),
              "Expected q [B,T,Hq,D], key/value [B,T,Hkv,D], cos/sin [B,T,R] and [D] weights");
  check_bf16({&q, &key, &value, &q_weight, &k_weight, &cos, &sin});
  check_inference({&q, &key, &value});
  check_slots(slots, q.size(0), q.size(1));
  const auto cache = cache_of(key_codes, key_scales, value_codes, value_scales);
  c10::DeviceGuard guard(q.device());
  auto output = new_tensor({q.size(0), q.size(2), q.size(1), q.size(3)}, at::kBFloat16, q);
  const auto qr = in_rows(q), kr = in_rows(key), vr = in_rows(value), cr = in_rows(cos), sr = in_rows(sin);
  const auto qw = in_rows(q_weight), kw = in_rows(k_weight);
  // Per-head views [B,H,T,D] and [B,1,T,R].
  const auto qv = view4(qr, true), kv = view4(kr, true), vv = view4(vr, true), cv = view3(cr), sv = view3(sr);
  check_status(xinfer_qk_norm_rope_append_kv4(&qv, &kv, &vv, qw.data_ptr(), kw.data_ptr(), eps, weight_offset, &cv, &sv,
                                              static_cast<const int64_t *>(slots.data_ptr()), slots.stride(0),
                                              slots.stride(1), output.data_ptr(), &cache, stream_of(q)));
  return output;
}

at::Tensor paged_attention_kv4(const at::Tensor &q, const at::Tensor &key_codes, const at::Tensor &key_scales,
                               const at::Tensor &value_codes, const at::Tensor &value_scales,
                               const at::Tensor &block_table, const at::Tensor &lengths, int64_t max_length,
                               double scale) {
  check_colocated(q, {&key_codes, &key_scales, &value_codes, &value_scales, &block_table, &lengths});
  TORCH_CHECK(q.dim() == 4, "Expected q [B,Hq,T,D]");
  check_bf16({&q});
  TORCH_CHECK(block_table.scalar_type() == at::kInt && block_table.dim() == 2 && block_table.size(0) == q.size(0) &&
                  block_table.is_contiguous(),
              "Expected a contiguous int32 block table [B,M]");
  TORCH_CHECK(lengths.scalar_type() == at::kInt && lengths.dim() == 2 && lengths.size(0) == 2 &&
                  lengths.size(1) == q.size(0) && lengths.is_contiguous(),
              "Expected contiguous int32 lengths [2,B]");
  TORCH_CHECK(!q.requires_grad(), "xinfer attention supports inference only");
  const auto cache = cache_of(key_codes, key_scales, value_codes, value_scales);
  c10::DeviceGuard guard(q.device());
  auto output = new_tensor({q.size(0), q.size(2), q.size(1), q.size(3)}, at::kBFloat16, q);
  auto query = in_rows(q);
  auto qv = view4(query);
  const size_t bytes = xinfer_paged_attention_kv4_workspace_size(&qv, &cache, block_table.size(1), max_length);
  at::Tensor workspace;
  if (bytes > 0) workspace = new_tensor({static_cast<int64_t>(bytes)}, at::kByte, q);
  check_status(xinfer_paged_attention_kv4(&qv, &cache, static_cast<const int32_t *>(block_table.data_ptr()),
                                          block_table.size(1), static_cast<const int32_t *>(lengths.data_ptr()),
                                          max_length, scale, output.data_ptr(), bytes > 0 ? workspace.data_ptr() : nullptr, bytes,
                                          stream_of(q)));
  return output;
}

}  // namespace xinfer

TORCH_LIBRARY_FRAGMENT(xinfer, m) {
  m.def("paged_kv_reserve(Tensor kv_before, Tensor kv_lengths, Tensor query_lengths, SymInt tokens, SymInt page_size, "
        "Tensor counters, Tensor(a6!) block_table, Tensor(a7!) free_pages) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("append_kv4(Tensor key, Tensor value, Tensor slots, Tensor(a3!) key_codes, Tensor(a4!) key_scales, "
        "Tensor(a5!) value_codes, Tensor(a6!) value_scales) -> ()");
  m.def("read_kv4(Tensor key_codes, Tensor key_scales, Tensor value_codes, Tensor value_scales, Tensor slots) "
        "-> (Tensor, Tensor)");
  m.def("qk_norm_rope_append_kv4(Tensor q, Tensor key, Tensor value, Tensor q_weight, Tensor k_weight, float eps, "
        "float weight_offset, Tensor cos, Tensor sin, Tensor slots, Tensor(a10!) key_codes, Tensor(a11!) key_scales, "
        "Tensor(a12!) value_codes, Tensor(a13!) value_scales) -> Tensor");
  m.def("paged_attention_kv4(Tensor q, Tensor key_codes, Tensor key_scales, Tensor value_codes, Tensor value_scales, "
        "Tensor block_table, Tensor lengths, SymInt max_length, float scale) -> Tensor",
        {at::Tag::flexible_layout});
}

TORCH_LIBRARY_IMPL(xinfer, CUDA, m) {
  m.impl("paged_kv_reserve", TORCH_FN(xinfer::paged_kv_reserve));
  m.impl("append_kv4", TORCH_FN(xinfer::append_kv4));
  m.impl("read_kv4", TORCH_FN(xinfer::read_kv4));
  m.impl("qk_norm_rope_append_kv4", TORCH_FN(xinfer::qk_norm_rope_append_kv4));
  m.impl("paged_attention_kv4", TORCH_FN(xinfer::paged_attention_kv4));
}

using torch::aot_inductor::new_tensor_handle;
using torch::aot_inductor::resolve_tensor_dispatch_flags;

extern "C" {

AOTI_TORCH_EXPORT AOTITorchError aoti_torch_cuda_paged_kv_reserve(
    AtenTensorHandle kv_before, AtenTensorHandle kv_lengths, AtenTensorHandle query_lengths, int64_t tokens,
    int64_t page_size, AtenTensorHandle counters, AtenTensorHandle block_table, AtenTensorHandle free_pages,
    AtenTensorHandle *lengths, AtenTensorHandle *positions, AtenTensorHandle *slots, AtenTensorHandle *new_counters) {
  AOTI_TORCH_CONVERT_EXCEPTION_TO_ERROR_CODE({
    auto [l, p, s, c] = xinfer::paged_kv_reserve(
        resolve_tensor_dispatch_flags(kv_before), resolve_tensor_dispatch_flags(kv_lengths),
        resolve_tensor_dispatch_flags(query_lengths), tokens, page_size, resolve_tensor_dispatch_flags(counters),
        resolve_tensor_dispatch_flags(block_table), resolve_tensor_dispatch_flags(free_pages));
    *lengths = new_tensor_handle(std::move(l));
    *positions = new_tensor_handle(std::move(p));
    *slots = new_tensor_handle(std::move(s));
    *new_counters = new_tensor_handle(std::move(c));
  });
}

AOTI_TORCH_EXPORT AOTITorchError aoti_torch_cuda_append_kv4(
    AtenTensorHandle key, AtenTensorHandle value, AtenTensorHandle slots, AtenTensorHandle key_codes,
    AtenTensorHandle key_scales, AtenTensorHandle value_codes, AtenTensorHandle value_scales,
    AtenTensorHandle * /*unused_output*/) {
  AOTI_TORCH_CONVERT_EXCEPTION_TO_ERROR_CODE({
    xinfer::append_kv4(resolve_tensor_dispatch_flags(key), resolve_tensor_dispatch_flags(value),
                       resolve_tensor_dispatch_flags(slots), resolve_tensor_dispatch_flags(key_codes),
                       resolve_tensor_dispatch_flags(key_scales), resolve_tensor_dispatch_flags(value_codes),
                       resolve_tensor_dispatch_flags(value_scales));
  });
}

AOTI_TORCH_EXPORT AOTITorchError aoti_torch_cuda_read_kv4(AtenTensorHandle key_codes, AtenTensorHandle key_scales,
                                                          AtenTensorHandle value_codes, AtenTensorHandle value_scales,
                                                          AtenTensorHandle slots, AtenTensorHandle *key,
                                                          AtenTensorHandle *value) {
  AOTI_TORCH_CONVERT_EXCEPTION_TO_ERROR_CODE({
    auto [k, v] = xinfer::read_kv4(resolve_tensor_dispatch_flags(key_codes), resolve_tensor_dispatch_flags(key_scales),
                                   resolve_tensor_dispatch_flags(value_codes),
                                   resolve_tensor_dispatch_flags(value_scales), resolve_tensor_dispatch_flags(slots));
    *key = new_tensor_handle(std::move(k));
    *value = new_tensor_handle(std::move(v));
  });
}

AOTI_TORCH_EXPORT AOTITorchError aoti_torch_cuda_qk_norm_rope_append_kv4(
    AtenTensorHandle q, AtenTensorHandle key, AtenTensorHandle value, AtenTensorHandle q_weight,
    AtenTensorHandle k_weight, double eps, double weight_offset, AtenTensorHandle cos, AtenTensorHandle sin,
    AtenTensorHandle slots, AtenTensorHandle key_codes, AtenTensorHandle key_scales, AtenTensorHandle value_codes,
    AtenTensorHandle value_scales, AtenTensorHandle *output) {
  AOTI_TORCH_CONVERT_EXCEPTION_TO_ERROR_CODE({
    *output = new_tensor_handle(xinfer::qk_norm_rope_append_kv4(
        resolve_tensor_dispatch_flags(q), resolve_tensor_dispatch_flags(key), resolve_tensor_dispatch_flags(value),
        resolve_tensor_dispatch_flags(q_weight), resolve_tensor_dispatch_flags(k_weight), eps, weight_offset,
        resolve_tensor_dispatch_flags(cos), resolve_tensor_dispatch_flags(sin), resolve_tensor_dispatch_flags(slots),
        resolve_tensor_dispatch_flags(key_codes), resolve_tensor_dispatch_flags(key_scales),
        resolve_tensor_dispatch_flags(value_codes), resolve_tensor_dispatch_flags(value_scales)));
  });
}

AOTI_TORCH_EXPORT AOTITorchError aoti_torch_cuda_paged_attention_kv4(
    AtenTensorHandle q, AtenTensorHandle key_codes, AtenTensorHandle key_scales, AtenTensorHandle value_codes,
    AtenTensorHandle value_scales, AtenTensorHandle block_table, AtenTensorHandle lengths, int64_t max_length, double scale,
    AtenTensorHandle *output) {
  AOTI_TORCH_CONVERT_EXCEPTION_TO_ERROR_CODE({
    *output = new_tensor_handle(xinfer::paged_attention_kv4(
        resolve_tensor_dispatch_flags(q), resolve_tensor_dispatch_flags(key_codes),
        resolve_tensor_dispatch_flags(key_scales), resolve_tensor_dispatch_flags(value_codes),
        resolve_tensor_dispatch_flags(value_scales), resolve_tensor_dispatch_flags(block_table),
        resolve_tensor_dispatch_flags(lengths), max_length, scale));
  });
}

}  // extern "C"
