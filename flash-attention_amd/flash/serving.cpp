// Tensor checks, output and scratch allocation, one call into the C ABI (include/flash_hip.h) for each serving operator.
#include "serving.hpp"

#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/AutogradState.h>
#include <hip/hip_runtime_api.h>

#include <cmath>
#include <map>
#include <mutex>
#include <sstream>
#include <stdexcept>

#include "../../include/flash_hip.h"

namespace flash {

namespace {

using torch::Tensor;
using Maybe = std::optional<Tensor>;

template <typename... Parts>
void refuse_if(bool condition, const Parts&... parts) {
  if (!condition) return;
  std::ostringstream text;
  (text << ... << parts);
  throw std::invalid_argument(text.str());
}

void raise(int rc) {
  if (rc == FLASH_HIP_OK) return;
  if (rc == FLASH_HIP_ERR_INVALID_ARGUMENT || rc == FLASH_HIP_ERR_UNSUPPORTED_DIM) throw std::invalid_argument(flash_hip_last_error());
  throw std::runtime_error(flash_hip_last_error());
}

int dtype_of(const Tensor& t, const char* what, bool cache = false) {
  if (t.scalar_type() == at::kHalf) return FLASH_F16;
  if (t.scalar_type() == at::kBFloat16) return FLASH_BF16;
  if (cache && t.scalar_type() == at::kFloat8_e4m3fn) return FLASH_E4M3;
  refuse_if(true, what, " must be float16 or bfloat16", cache ? " or float8_e4m3fn" : "", ", got ", t.scalar_type());
  return -1;
}

// [rows, heads, d] with adjacent elements
void check_rows(const Tensor& t, const char* what) {
  refuse_if(t.dim() != 3, what, " must be [tokens, heads, d], got ", t.dim(), " dims");
  refuse_if(t.size(2) > 1 && t.stride(2) != 1, what, ": the elements of a row must be adjacent");
}
void check_int32(const Tensor& t, const char* what, int64_t dims) {
  refuse_if(t.scalar_type() != at::kInt, what, " must be int32, got ", t.scalar_type());
  refuse_if(t.dim() != dims, what, " must have ", dims, " dimension(s), got ", t.dim());
  refuse_if(t.size(dims - 1) > 1 && t.stride(dims - 1) != 1, what, ": entries must be adjacent");
}
// No tensor of a call, an output among them, takes part in a derivative: neither backward nor forward.
void check_no_grad(std::initializer_list<const Tensor*> tensors) {
  const bool backward = at::GradMode::is_enabled(), forward = c10::AutogradState::get_tls_state().get_fw_grad_mode();
  for (const Tensor* t : tensors) {
    if (!t->defined()) continue;
    refuse_if(backward && t->requires_grad(), "there is no backward pass: detach the tensors or run under no_grad");
    refuse_if(forward && t->_fw_grad(/*level=*/0).defined(), "there is no forward-mode derivative: detach the tensors");
  }
}
// Tensors that the call writes are modified, for whoever saved them (those of inference mode keep no count)
void modified(std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors) {
    if (t->defined() && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
  }
}
void check_device(const Tensor& first, std::initializer_list<const Tensor*> tensors) {
  refuse_if(!first.is_cuda(), "tensors must be on a HIP device (there is no CPU path)");
  for (const Tensor* t : tensors) refuse_if(t->defined() && t->device() != first.device(), "tensors on different devices");
}
float scale_of(std::optional<double> given, int64_t d) {
  return given ? static_cast<float>(*given) : 1.0f / std::sqrt(static_cast<float>(d));
}
const Tensor kNone;
const Tensor& or_none(const Maybe& t) { return t ? *t : kNone; }

bool capturing(const c10::hip::HIPStreamMasqueradingAsCUDA& stream) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(stream.stream(), &status) != hipSuccess) throw std::runtime_error("hipStreamIsCapturing failed");
  return status != hipStreamCaptureStatusNone;
}
// The stream of a call.  Waiting for it would end a capture.
c10::hip::HIPStreamMasqueradingAsCUDA stream_of(c10::Device device, bool sync) {
  const auto stream = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(device.index());
  refuse_if(sync && capturing(stream), "the call is captured into a graph, which cannot wait for its result: pass sync=False");
  return stream;
}
void wait_for(const c10::hip::HIPStreamMasqueradingAsCUDA& stream) {
  const hipError_t e = hipStreamSynchronize(stream.stream());
  if (e != hipSuccess) throw std::runtime_error(hipGetErrorString(e));
}

// Scratch whose bytes [zeros.first, zeros.second) (-1: up to its end) are zero, and left zero by the calls that use it; one
// kind of scratch has one value of zeros.first.  Work on one stream runs in order, so its calls share a buffer that is filled
// once, on their first call (and again when a larger one is needed).  A graph under capture gets one of its own, filled by a
// node of the graph: it may be replayed on any stream, beside any other.  So does a call on a stream that torch did not
// make, whose handle may come to stand for another stream.  Buffers are kept until release_workspaces().
struct Kept {
  std::mutex mutex;
  std::map<std::tuple<int, c10::StreamId, int64_t>, Tensor> buffers;
};
Kept& kept() {
  static auto& all = *new Kept;  // (never destroyed: the allocator may be gone by then)
  return all;
}
Tensor stream_workspace(c10::Device device, const c10::hip::HIPStreamMasqueradingAsCUDA& stream, int64_t need, std::pair<int64_t, int64_t> zeros) {
  const auto options = at::TensorOptions().dtype(at::kByte).device(device);
  const c10::StreamId id = stream.unwrap().id();
  const bool own_stream = id == 0 || (id & 1) != 0;  // torch's numbering: the default stream, and the streams of its pools
  auto fresh = [&](int64_t bytes) {
    Tensor t = at::empty({bytes}, options);
    t.slice(0, zeros.first, zeros.second < 0 ? bytes : zeros.second).zero_();
    return t;
  };
  if (!own_stream || capturing(stream)) return fresh(need);
  const std::lock_guard<std::mutex> lock(kept().mutex);
  Tensor& t = kept().buffers[{device.index(), id, zeros.first}];
  if (!t.defined() || t.numel() < need) t = fresh(need + (1 << 16));
  return t;
}

flash_paged_cache describe(const Tensor& k, const Tensor& v, const Tensor& table, const Tensor* lens, const Tensor& k_scale, const Tensor& v_scale) {
  refuse_if(k.dim() != 4, "k_cache must be [pages, heads, page_size, d], got ", k.dim(), " dims");
  refuse_if(v.sizes() != k.sizes() || v.scalar_type() != k.scalar_type(), "v_cache must have the shape and type of k_cache");
  refuse_if(v.strides() != k.strides(), "v_cache must have the strides of k_cache");
  refuse_if(k.size(3) > 1 && k.stride(3) != 1, "cache: the elements of a row must be adjacent");
  check_int32(table, "page_table", 2);
  flash_paged_cache c{};
  c.dtype = dtype_of(k, "the cache", true);
  if (lens) {
    check_int32(*lens, "seq_lens", 1);
    refuse_if(lens->size(0) != table.size(0), "seq_lens must have one entry for each of the ", table.size(0), " rows of page_table, got ", lens->size(0));
    c.seq_lens = static_cast<const int32_t*>(lens->const_data_ptr());
  }
  for (const Tensor* s : {&k_scale, &v_scale}) {
    if (!s->defined()) continue;
    refuse_if(c.dtype != FLASH_E4M3, "k_scale and v_scale go with a float8_e4m3fn cache only");
    refuse_if(s->scalar_type() != at::kFloat || s->dim() != 1 || s->size(0) != k.size(1) || !s->is_contiguous(),
              "k_scale and v_scale must be contiguous float32 tensors of ", k.size(1), " entries");
  }
  c.k = const_cast<void*>(k.const_data_ptr());
  c.v = const_cast<void*>(v.const_data_ptr());
  c.num_pages = k.size(0);
  c.kv_heads = k.size(1);
  c.page_size = k.size(2);
  c.d = k.size(3);
  c.page_stride = k.stride(0);
  c.head_stride = k.stride(1);
  c.slot_stride = k.stride(2);
  c.k_scale = k_scale.defined() ? static_cast<const float*>(k_scale.const_data_ptr()) : nullptr;
  c.v_scale = v_scale.defined() ? static_cast<const float*>(v_scale.const_data_ptr()) : nullptr;
  c.page_table = static_cast<const int32_t*>(table.const_data_ptr());
  c.sequences = table.size(0);
  c.table_width = table.size(1);
  c.table_stride = table.size(0) > 1 ? table.stride(0) : table.size(1);
  return c;
}

flash_decode_args decode_args(const Tensor& q, const flash_paged_cache& c) {
  refuse_if(q.dim() != 3, "q must be [sequences, heads, d], got ", q.dim(), " dims");
  check_rows(q, "q");
  refuse_if(q.size(0) != c.sequences, "q must have one row for each of the ", c.sequences, " rows of page_table, got ", q.size(0));
  refuse_if(q.size(2) != c.d, "q and the cache must have the same head dim, got ", q.size(2), " and ", c.d);
  flash_decode_args a{};
  a.dtype = dtype_of(q, "q");
  a.q = q.const_data_ptr();
  a.q_heads = q.size(1);
  a.q_batch_stride = q.stride(0);
  a.q_head_stride = q.stride(1);
  a.softmax_scale = 1.0f;
  return a;
}

// a given output, or a new one; `given` is checked against q
Tensor output_for(const Tensor& q, const Maybe& given) {
  if (!given) return torch::empty(q.sizes(), q.options().memory_format(c10::nullopt).requires_grad(false));
  refuse_if(given->sizes() != q.sizes() || given->scalar_type() != q.scalar_type(), "out must have the shape and type of q");
  check_rows(*given, "out");
  return *given;
}

}  // namespace

Tensor forward_packed(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu_q, const Maybe& cu_k_given,
                      bool causal, std::optional<double> softmax_scale, const Maybe& out_given, bool sync) {
  check_rows(q, "q");
  check_rows(k, "k");
  check_rows(v, "v");
  flash_packed_args a{};
  a.dtype = dtype_of(q, "q");
  refuse_if(k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type(), "q, k, v must share one dtype");
  refuse_if(v.sizes() != k.sizes(), "v must have the shape of k");
  refuse_if(k.size(2) != q.size(2), "q and k must have the same head dim, got ", q.size(2), " and ", k.size(2));
  check_int32(cu_q, "cu_seqlens_q", 1);
  const Tensor& cu_k = cu_k_given ? *cu_k_given : cu_q;
  check_int32(cu_k, "cu_seqlens_k", 1);
  refuse_if(cu_q.size(0) < 1 || cu_k.size(0) != cu_q.size(0), "cu_seqlens_q and cu_seqlens_k must have one entry more than there are sequences, got ",
            cu_q.size(0), " and ", cu_k.size(0));
  refuse_if(!cu_k_given && k.size(0) != q.size(0), "without cu_seqlens_k there must be as many keys as queries, got ", k.size(0), " and ", q.size(0));
  check_no_grad({&q, &k, &v, &or_none(out_given)});
  a.sequences = cu_q.size(0) - 1;
  a.total_q = q.size(0);
  a.total_k = k.size(0);
  a.q_heads = q.size(1);
  a.kv_heads = k.size(1);
  a.d = q.size(2);
  a.causal = causal ? 1 : 0;
  a.softmax_scale = scale_of(softmax_scale, a.d);
  a.q_token_stride = q.stride(0);
  a.q_head_stride = q.stride(1);
  a.k_token_stride = k.stride(0);
  a.k_head_stride = k.stride(1);
  a.v_token_stride = v.stride(0);
  a.v_head_stride = v.stride(1);
  a.o_token_stride = a.q_heads * a.d;
  a.o_head_stride = a.d;
  if (out_given) {
    output_for(q, out_given);
    a.o_token_stride = out_given->stride(0);
    a.o_head_stride = out_given->stride(1);
  }
  // what needs no memory is refused before the device is looked at
  const int64_t need = flash_fwd_packed_workspace_bytes(&a);
  if (need < 0) throw std::invalid_argument(flash_hip_last_error());
  check_device(q, {&k, &v, &cu_q, &cu_k, &or_none(out_given)});
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  const auto stream = stream_of(q.device(), sync);
  Tensor o = output_for(q, out_given);
  a.q = q.const_data_ptr();
  a.k = k.const_data_ptr();
  a.v = v.const_data_ptr();
  a.o = o.data_ptr();
  a.cu_seqlens_q = static_cast<const int32_t*>(cu_q.const_data_ptr());
  a.cu_seqlens_k = static_cast<const int32_t*>(cu_k.const_data_ptr());
  Tensor scratch;
  if (need > 0) scratch = stream_workspace(q.device(), stream, need, {0, FLASH_PACKED_TICKET_BYTES});
  raise(flash_fwd_packed(&a, need > 0 ? scratch.data_ptr() : nullptr, need, stream.stream()));
  modified({&or_none(out_given)});
  if (sync) wait_for(stream);
  return o;
}

void release_workspaces() {
  decltype(Kept::buffers) all;  // (freed when the lock is given back)
  const std::lock_guard<std::mutex> lock(kept().mutex);
  all.swap(kept().buffers);
}

int64_t decode_workspace_bytes(const Tensor& q, const Tensor& k_cache, const Tensor& page_table) {
  const flash_paged_cache c = describe(k_cache, k_cache, page_table, nullptr, kNone, kNone);
  flash_decode_args a = decode_args(q, c);
  a.o_batch_stride = a.q_heads * c.d;
  a.o_head_stride = c.d;
  const int64_t bytes = flash_decode_paged_workspace_bytes(&a, &c);
  if (bytes < 0) throw std::invalid_argument(flash_hip_last_error());
  return bytes;
}

std::tuple<Tensor, Tensor> decode_paged(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& page_table,
                                        const Tensor& seq_lens, std::optional<double> softmax_scale, const Maybe& k_scale,
                                        const Maybe& v_scale, const Maybe& out_given, bool return_lse, const Maybe& workspace, bool sync) {
  const flash_paged_cache c = describe(k_cache, v_cache, page_table, &seq_lens, or_none(k_scale), or_none(v_scale));
  flash_decode_args a = decode_args(q, c);
  a.softmax_scale = scale_of(softmax_scale, c.d);
  check_no_grad({&q, &k_cache, &v_cache, &or_none(k_scale), &or_none(v_scale), &or_none(out_given), &or_none(workspace)});
  a.o_batch_stride = a.q_heads * c.d;
  a.o_head_stride = c.d;
  if (out_given) {
    output_for(q, out_given);
    a.o_batch_stride = out_given->stride(0);
    a.o_head_stride = out_given->stride(1);
  }
  const int64_t need = flash_decode_paged_workspace_bytes(&a, &c);
  if (need < 0) throw std::invalid_argument(flash_hip_last_error());
  if (workspace) {
    refuse_if(!workspace->is_contiguous() || static_cast<int64_t>(workspace->nbytes()) < need, "workspace must be contiguous and hold ", need, " bytes");
  }
  check_device(q, {&k_cache, &v_cache, &page_table, &seq_lens, &or_none(k_scale), &or_none(v_scale), &or_none(out_given), &or_none(workspace)});
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  const auto stream = stream_of(q.device(), sync);
  Tensor o = output_for(q, out_given), lse, scratch;
  a.o = o.data_ptr();
  if (return_lse) {
    lse = torch::empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat).requires_grad(false));
    a.lse = static_cast<float*>(lse.data_ptr());
  }
  if (need > 0) scratch = workspace ? *workspace : stream_workspace(q.device(), stream, need, {FLASH_DECODE_PARTS_BYTES, -1});
  raise(flash_decode_paged(&a, &c, need > 0 ? scratch.data_ptr() : nullptr, need, stream.stream()));
  modified({&or_none(out_given), &or_none(workspace)});
  if (sync) wait_for(stream);
  return {o, lse};
}

void cache_append(const Tensor& k, const Tensor& v, const Tensor& k_cache, const Tensor& v_cache, const Tensor& page_table,
                  const Tensor& seq_lens, const Maybe& cu_seqlens, const Maybe& k_scale, const Maybe& v_scale, bool sync) {
  const flash_paged_cache c = describe(k_cache, v_cache, page_table, &seq_lens, or_none(k_scale), or_none(v_scale));
  check_rows(k, "k");
  refuse_if(v.sizes() != k.sizes() || v.scalar_type() != k.scalar_type(), "v must have the shape and type of k");
  check_rows(v, "v");
  refuse_if(k.size(1) != c.kv_heads || k.size(2) != c.d, "k must be [tokens, ", c.kv_heads, ", ", c.d, "] like the cache's rows, got [", k.size(0),
            ", ", k.size(1), ", ", k.size(2), "]");
  flash_append_args a{};
  a.dtype = dtype_of(k, "k");
  a.tokens = k.size(0);
  if (cu_seqlens) {
    check_int32(*cu_seqlens, "cu_seqlens", 1);
    refuse_if(cu_seqlens->size(0) != c.sequences + 1, "cu_seqlens must have ", c.sequences + 1, " entries, got ", cu_seqlens->size(0));
    a.cu_seqlens = static_cast<const int32_t*>(cu_seqlens->const_data_ptr());
  }
  check_no_grad({&k, &v, &k_cache, &v_cache, &or_none(k_scale), &or_none(v_scale)});
  a.k = k.const_data_ptr();
  a.v = v.const_data_ptr();
  a.k_token_stride = k.stride(0);
  a.k_head_stride = k.stride(1);
  a.v_token_stride = v.stride(0);
  a.v_head_stride = v.stride(1);
  check_device(k, {&v, &k_cache, &v_cache, &page_table, &seq_lens, &or_none(cu_seqlens), &or_none(k_scale), &or_none(v_scale)});
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(k.device());
  const auto stream = stream_of(k.device(), sync);
  raise(flash_cache_append(&a, &c, stream.stream()));
  modified({&k_cache, &v_cache});
  if (sync) wait_for(stream);
}

}  // namespace flash
