// torch.ops.pyflash.* for PyTorch-ROCm: the reference's twelve operator names with the schema
// "(Tensor Q, Tensor K, Tensor V) -> Tensor" (reference pyflash/pyflash.cpp:10-35), each bound to
// flash::forward with the KernelType the reference binds it to, and the serving operators.  Loaded the same way:
//   torch.ops.load_library("build/pyflash/libpyflash.so")   (reference benchmarks/bench.py:12-14)
#include <torch/extension.h>

#include <optional>
#include <string>

#include "../flash/launch.hpp"
#include "../flash/serving.hpp"

namespace {

template <flash::KernelType KT>
torch::Tensor attention_op(torch::Tensor Q, torch::Tensor K, torch::Tensor V) {
  return flash::forward(std::move(Q), std::move(K), std::move(V), KT);
}

template <flash::KernelType KT>
void bind(torch::Library& m, const char* op_name) {
  const std::string schema = std::string(op_name) + "(Tensor Q, Tensor K, Tensor V) -> Tensor";
  // A plain function pointer: C++ exceptions travel through the dispatcher to torch's Python
  // binding, which translates them with the GIL held.  (The reference wraps the function with
  // torch::wrap_pybind_function, whose error path touches the interpreter without the GIL when
  // the op is invoked through torch.ops.)
  m.def(schema.c_str(), &attention_op<KT>);
}

using torch::Tensor;
using Maybe = std::optional<Tensor>;
// (None arrives as an undefined tensor)
Maybe given(const Tensor& out) { return out.defined() ? Maybe(out) : std::nullopt; }

}  // namespace

TORCH_LIBRARY(pyflash, m) {
  using KT = flash::KernelType;
  bind<KT::naive1D>(m, "naive");
  bind<KT::scalar2D>(m, "scalar2d");
  bind<KT::scalar2D_row_tile>(m, "scalar2d_row_tile");
  bind<KT::warp_wmma>(m, "warp_wmma");
  bind<KT::block_wmma>(m, "block_wmma");
  bind<KT::wmma_row_block>(m, "block_wmma_row_block");
  bind<KT::block_wmma_async>(m, "block_wmma_async");
  bind<KT::mma>(m, "mma");
  bind<KT::mma_swizzle>(m, "mma_swizzle");
  bind<KT::mma_qreg>(m, "mma_qreg");
  bind<KT::mma_qreg_f32x4load>(m, "mma_qreg_vld");
  bind<KT::mma_qreg_async>(m, "mma_qreg_async");

  // the serving operators (flash/serving.hpp); no counterpart in the reference
  // (an operator's result aliases the output it was given: a form of its own, so that the other one's is a new tensor)
  m.def("forward_packed(Tensor q, Tensor k, Tensor v, Tensor cu_seqlens_q, Tensor? cu_seqlens_k=None, *, bool causal=True, "
        "float? softmax_scale=None, bool sync=True) -> Tensor",
        [](const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu_q, const Maybe& cu_k, bool causal, std::optional<double> scale,
           bool sync) { return flash::forward_packed(q, k, v, cu_q, cu_k, causal, scale, std::nullopt, sync); });
  m.def("forward_packed.out(Tensor q, Tensor k, Tensor v, Tensor cu_seqlens_q, Tensor? cu_seqlens_k=None, *, bool causal=True, "
        "float? softmax_scale=None, Tensor(a!) out, bool sync=True) -> Tensor(a!)",
        [](const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu_q, const Maybe& cu_k, bool causal, std::optional<double> scale,
           const Tensor& out, bool sync) { return flash::forward_packed(q, k, v, cu_q, cu_k, causal, scale, given(out), sync); });
  m.def("decode_paged(Tensor q, Tensor k_cache, Tensor v_cache, Tensor page_table, Tensor seq_lens, *, "
        "float? softmax_scale=None, Tensor? k_scale=None, Tensor? v_scale=None, bool return_lse=False, "
        "Tensor(b!)? workspace=None, bool sync=True) -> (Tensor, Tensor)",
        [](const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& lens, std::optional<double> scale,
           const Maybe& k_scale, const Maybe& v_scale, bool lse, const Maybe& workspace, bool sync) {
          return flash::decode_paged(q, k, v, table, lens, scale, k_scale, v_scale, std::nullopt, lse, workspace, sync);
        });
  m.def("decode_paged.out(Tensor q, Tensor k_cache, Tensor v_cache, Tensor page_table, Tensor seq_lens, *, "
        "float? softmax_scale=None, Tensor? k_scale=None, Tensor? v_scale=None, Tensor(a!) out, bool return_lse=False, "
        "Tensor(b!)? workspace=None, bool sync=True) -> (Tensor(a!), Tensor)",
        [](const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& lens, std::optional<double> scale,
           const Maybe& k_scale, const Maybe& v_scale, const Tensor& out, bool lse, const Maybe& workspace, bool sync) {
          return flash::decode_paged(q, k, v, table, lens, scale, k_scale, v_scale, given(out), lse, workspace, sync);
        });
  m.def("release_workspaces() -> ()", &flash::release_workspaces);
  m.def("decode_workspace_bytes(Tensor q, Tensor k_cache, Tensor page_table) -> int", &flash::decode_workspace_bytes);
  m.def("cache_append(Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor page_table, Tensor seq_lens, "
        "Tensor? cu_seqlens=None, *, Tensor? k_scale=None, Tensor? v_scale=None, bool sync=True) -> ()",
        &flash::cache_append);
}
