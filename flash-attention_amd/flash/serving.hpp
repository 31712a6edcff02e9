// C++ entries of the serving operators on libtorch tensors: attention over packed prompts, writes into a paged
// key-value cache, and attention of one new token over it.  The reference has no counterpart (its flash::forward,
// flash/launch.hpp:23-24, takes equal lengths, one K/V head per query head and no mask).
//
// Like flash::forward they check their arguments (std::invalid_argument), run on the current HIP stream of the
// tensors' device and, with `sync`, wait for the result.  Shapes, types and strides are checked before the device, so
// that a refusal needs no GPU.  There is no derivative: tensors that require a gradient are refused while
// gradients are recorded, and so are tensors with a forward-mode tangent, scales and outputs among them.
#pragma once
#include <torch/torch.h>

#include <optional>
#include <tuple>

namespace flash {

// q [total_q, Hq, d], k and v [total_k, Hkv, d], any token and head strides; cu_seqlens_* int32 [sequences + 1].
// cu_seqlens_k absent: the keys are cut like the queries.  Returns `out`, or a new contiguous tensor like q (rows of
// no sequence are then undefined).  Calls with few rows over many keys use scratch (below 70 MB): one buffer for each of
// torch's streams, one of its own for every captured graph.
torch::Tensor forward_packed(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v,
                             const torch::Tensor& cu_seqlens_q, const std::optional<torch::Tensor>& cu_seqlens_k,
                             bool causal, std::optional<double> softmax_scale, const std::optional<torch::Tensor>& out,
                             bool sync);

// q [sequences, Hq, d]; caches [pages, Hkv, page_size, d]; page_table int32 [sequences, width]; seq_lens int32
// [sequences].  Returns the output and, when asked for, the logarithm of the weights' sum (float32 [sequences, Hq]; an
// undefined tensor otherwise).  `workspace`: at least decode_workspace_bytes bytes, zero-filled before its first use; absent,
// calls on one of torch's streams share one that is kept for it, and every captured graph has its own.
std::tuple<torch::Tensor, torch::Tensor> decode_paged(
    const torch::Tensor& q, const torch::Tensor& k_cache, const torch::Tensor& v_cache, const torch::Tensor& page_table,
    const torch::Tensor& seq_lens, std::optional<double> softmax_scale, const std::optional<torch::Tensor>& k_scale,
    const std::optional<torch::Tensor>& v_scale, const std::optional<torch::Tensor>& out, bool return_lse,
    const std::optional<torch::Tensor>& workspace, bool sync);
int64_t decode_workspace_bytes(const torch::Tensor& q, const torch::Tensor& k_cache, const torch::Tensor& page_table);

// Gives the scratch that is kept for streams back to torch's allocator, which hands it out again in the order of each
// stream: calls that are still running keep what they use.  Later calls allocate anew; captured graphs have their own.
void release_workspaces();

// k and v [tokens, Hkv, d] into the caches, in place.
void cache_append(const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& k_cache,
                  const torch::Tensor& v_cache, const torch::Tensor& page_table, const torch::Tensor& seq_lens,
                  const std::optional<torch::Tensor>& cu_seqlens, const std::optional<torch::Tensor>& k_scale,
                  const std::optional<torch::Tensor>& v_scale, bool sync);

}  // namespace flash
