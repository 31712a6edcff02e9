// C-ABI entry points of the serving operators (declared in include/flash_hip.h): argument checks, kernel choice,
// launch.  NaN and infinities mean something here (masked places may hold them), so this unit is compiled with them.
#include "../../include/flash_hip.h"

#include <hip/hip_runtime.h>

#include <cmath>

#include "attn_packed.hpp"
#include "attn_paged.hpp"
#include "cache_append.hpp"
#include "host.hpp"

namespace {

using flash_hip::set_error;

constexpr int64_t kMostIndex = (int64_t)1 << 30;  // tokens, positions, table entries: 32-bit with room to add
constexpr int64_t kMostStride = (int64_t)1 << 40;

#define REFUSE_IF(condition, ...) \
  do {                            \
    if (condition) return set_error(FLASH_HIP_ERR_INVALID_ARGUMENT, __VA_ARGS__); \
  } while (0)

int check_heads(int64_t q_heads, int64_t kv_heads, int64_t d) {
  REFUSE_IF(q_heads <= 0 || kv_heads <= 0 || q_heads > 65535, "head counts must be between 1 and 65535 (got %lld query, %lld K/V heads)",
            (long long)q_heads, (long long)kv_heads);
  REFUSE_IF(q_heads % kv_heads != 0, "the %lld query heads must be a multiple of the %lld K/V heads", (long long)q_heads,
            (long long)kv_heads);
  if (d <= 0 || d > 128 || d % 8 != 0)
    return set_error(FLASH_HIP_ERR_UNSUPPORTED_DIM, "Unsupported head dim %lld: a multiple of 8 up to 128 is needed", (long long)d);
  return FLASH_HIP_OK;
}
int check_scale(float scale) {
  REFUSE_IF(!(scale > 0.f) || !std::isfinite(scale * 1.44269504f), "softmax_scale must be positive and finite (got %g)", (double)scale);
  return FLASH_HIP_OK;
}
int check_16bit(int dtype) {
  REFUSE_IF(dtype != FLASH_F16 && dtype != FLASH_BF16, "tensors must be float16 or bfloat16 (got dtype %d)", dtype);
  return FLASH_HIP_OK;
}
// Rows that start at multiples of these strides, `rows` of them in the outer direction and `heads` in the inner one,
// on `align`-byte boundaries.  A stride of one row only is never used.
int check_rows(const char* what, const void* base, int64_t outer, int64_t rows, int64_t inner, int64_t heads, int64_t elem,
               int64_t align) {
  const int64_t unit = align / elem;
  REFUSE_IF(outer < 0 || inner < 0 || outer > kMostStride || inner > kMostStride, "%s: strides must not be negative", what);
  REFUSE_IF((uintptr_t)base % (uintptr_t)align != 0 || (rows > 1 && outer % unit != 0) || (heads > 1 && inner % unit != 0),
            "%s: rows must start on %lld-byte boundaries (strides %lld, %lld)", what, (long long)align, (long long)outer,
            (long long)inner);
  return FLASH_HIP_OK;
}

// Rows that a call writes: no element of them twice.
int check_written(const char* what, int64_t outer, int64_t rows, int64_t inner, int64_t heads, int64_t d) {
  REFUSE_IF(flash_hip::rows_meet({rows, outer}, {heads, inner}, {1, 0}, d), "%s: rows must not overlap in memory (strides %lld, %lld)", what,
            (long long)outer, (long long)inner);
  return FLASH_HIP_OK;
}

#define CHECK(call)                          \
  do {                                       \
    const int rc_ = (call);                  \
    if (rc_ != FLASH_HIP_OK) return rc_;     \
  } while (0)

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(FLASH_HIP_ERR_RUNTIME, "%s: kernel launch failed: %s", what, hipGetErrorString(e));
  return FLASH_HIP_OK;
}

// ---- the cache ------------------------------------------------------------------------------------------------
int check_cache(const flash_paged_cache* c, int dtype, bool memory) {
  REFUSE_IF(!c, "null flash_paged_cache");
  CHECK(check_16bit(dtype));
  REFUSE_IF(c->dtype != dtype && c->dtype != FLASH_E4M3, "a 16-bit cache must have the type of the other tensors (got dtype %d and %d)",
            c->dtype, dtype);
  REFUSE_IF(c->dtype != FLASH_E4M3 && (c->k_scale || c->v_scale), "k_scale and v_scale go with an e4m3 cache only");
  REFUSE_IF(c->page_size <= 0 || (c->page_size & (c->page_size - 1)) != 0 || c->page_size > kMostIndex,
            "page size must be a power of two (got %lld)", (long long)c->page_size);
  REFUSE_IF(c->num_pages <= 0 || c->num_pages > kMostIndex, "the cache must hold between 1 and 2^30 pages (got %lld)", (long long)c->num_pages);
  REFUSE_IF(c->sequences < 0 || c->sequences > kMostIndex || c->table_width < 0 || c->table_stride < 0 || c->table_stride > kMostStride,
            "page table of %lld x %lld entries, stride %lld", (long long)c->sequences, (long long)c->table_width, (long long)c->table_stride);
  REFUSE_IF(c->table_width > kMostIndex / c->page_size, "page table reaches %lld positions; 2^30 are the most",
            (long long)(c->table_width * c->page_size));
  REFUSE_IF(c->page_stride < 0 || c->page_stride > kMostStride, "cache: strides must not be negative");
  const int64_t elem = c->dtype == FLASH_E4M3 ? 1 : 2, align = 8 * elem;
  CHECK(check_rows("cache", nullptr, c->head_stride, c->kv_heads, c->slot_stride, c->page_size, elem, align));
  REFUSE_IF(c->num_pages > 1 && c->page_stride % 8 != 0, "cache: rows must start on %lld-byte boundaries (page stride %lld)", (long long)align,
            (long long)c->page_stride);
  if (memory) {
    REFUSE_IF(!c->k || !c->v, "null cache pointer");
    REFUSE_IF(((uintptr_t)c->k | (uintptr_t)c->v) % (uintptr_t)align != 0, "cache: rows must start on %lld-byte boundaries", (long long)align);
    REFUSE_IF((!c->page_table && c->table_width > 0) || !c->seq_lens, "null page table or lengths");
  }
  return FLASH_HIP_OK;
}
flash_hip::Pages pages_of(const flash_paged_cache* c, int64_t elem) {
  int shift = 0;
  while (((int64_t)1 << shift) < c->page_size) ++shift;
  return flash_hip::Pages{c->page_stride * elem, c->slot_stride * elem, (int32_t)c->num_pages, (int32_t)(c->table_width * c->page_size), shift};
}

// ---- decoding ---------------------------------------------------------------------------------------------------
using DecodeParams = flash_hip::paged::Params;

constexpr uint32_t kDecodeWorkgroups = flash_hip::paged::kMostWorkgroups;
// Workspace: room for two parts of every workgroup at the largest tile, then a ticket for each triple.  The tickets' place
// does not depend on the shape: parts of one call never lie where another call looks for zeros.
constexpr int64_t kPartRows = (int64_t)2 * kDecodeWorkgroups * 16, kPartBytes = kPartRows * (128 * 4 + 8);
static_assert(kPartBytes == FLASH_DECODE_PARTS_BYTES, "include/flash_hip.h names the part of the workspace that need not be zero");

struct DecodePlan {
  int tile_d;
  uint32_t workgroups;
  int64_t bytes;  // 0: no sequence can be cut
};
int plan_decode(const flash_decode_args* a, const flash_paged_cache* c, bool memory, DecodePlan* plan) {
  REFUSE_IF(!a, "null flash_decode_args");
  CHECK(check_cache(c, a->dtype, memory));
  CHECK(check_heads(a->q_heads, c->kv_heads, c->d));
  CHECK(check_scale(a->softmax_scale));
  CHECK(check_rows("q", memory ? a->q : nullptr, a->q_batch_stride, c->sequences, a->q_head_stride, a->q_heads, 2, 16));
  CHECK(check_rows("out", memory ? a->o : nullptr, a->o_batch_stride, c->sequences, a->o_head_stride, a->q_heads, 2, 16));
  CHECK(check_written("out", a->o_batch_stride, c->sequences, a->o_head_stride, a->q_heads, c->d));
  if (memory && c->sequences > 0) REFUSE_IF(!a->q || !a->o, "null tensor pointer");
  const int64_t group = a->q_heads / c->kv_heads;
  plan->tile_d = c->d <= 64 ? 64 : 128;
  const bool cache8 = c->dtype == FLASH_E4M3;
  const int64_t unit = (plan->tile_d == 64 || cache8) ? flash_hip::paged::kUnit<64, false> : flash_hip::paged::kUnit<128, false>;
  const int64_t reach = c->table_width * c->page_size;
  const int64_t most = reach <= unit ? 1 : (reach + unit - 1) / unit;  // units of a sequence
  const int64_t triples = c->sequences * c->kv_heads * ((group + 15) / 16);
  REFUSE_IF(triples * most >= (int64_t)1 << 31 || c->sequences * a->q_heads >= (int64_t)1 << 31, "batch of %lld sequences is too large", (long long)c->sequences);
  plan->workgroups = (uint32_t)(triples * most < kDecodeWorkgroups ? triples * most : kDecodeWorkgroups);
  plan->bytes = most > 1 && triples > 0 ? kPartBytes + (triples * 4 + 15) / 16 * 16 : 0;
  return FLASH_HIP_OK;
}

template <int D, int EK, bool CACHE8>
int launch_decode(const DecodeParams& p, hipStream_t stream) {
  namespace pg = flash_hip::paged;
  const bool page16 = p.pages.page_shift >= 4 && 16 * p.pages.slot_stride < ((int64_t)1 << 31);
  auto kernel = p.d == D ? (page16 ? pg::decode_kernel<D, EK, CACHE8, true, true> : pg::decode_kernel<D, EK, CACHE8, true, false>)
                         : (page16 ? pg::decode_kernel<D, EK, CACHE8, false, true> : pg::decode_kernel<D, EK, CACHE8, false, false>);
  hipLaunchKernelGGL(kernel, dim3(p.workgroups), dim3(pg::kThreads), 0, stream, p);
  return launched("flash_decode_paged");
}
template <int D>
int launch_decode(const DecodeParams& p, int dtype, bool cache8, hipStream_t stream) {
  using namespace flash_hip::direct;
  if (dtype == FLASH_F16) return cache8 ? launch_decode<D, kHalf, true>(p, stream) : launch_decode<D, kHalf, false>(p, stream);
  return cache8 ? launch_decode<D, kBfloat, true>(p, stream) : launch_decode<D, kBfloat, false>(p, stream);
}

// ---- packed prompts -----------------------------------------------------------------------------------------------
int64_t direct_tiles(const flash_hip::packed::Params& p) { return (int64_t)p.total_q / flash_hip::packed::kDirectRows + p.sequences; }
template <int D, int EK>
int launch_packed_direct(flash_hip::packed::Params p, hipStream_t stream) {
  namespace pk = flash_hip::packed;
  p.extra = 1;
  p.tiles = (uint32_t)direct_tiles(p);
  const dim3 grid(p.tiles, (uint32_t)p.heads);
  if (p.d == D) {
    hipLaunchKernelGGL((pk::packed_direct_kernel<D, EK, true>), grid, dim3(256), 0, stream, p);
  } else {
    hipLaunchKernelGGL((pk::packed_direct_kernel<D, EK, false>), grid, dim3(256), 0, stream, p);
  }
  return launched("flash_fwd_packed");
}

// The kernel's arguments, for what flash_fwd_packed takes.  Without `memory` the sizes and strides alone are looked at.
int plan_packed(const flash_packed_args* a, bool memory, flash_hip::packed::Params* out) {
  REFUSE_IF(!a, "null flash_packed_args");
  CHECK(check_16bit(a->dtype));
  CHECK(check_heads(a->q_heads, a->kv_heads, a->d));
  CHECK(check_scale(a->softmax_scale));
  REFUSE_IF(a->causal != 0 && a->causal != 1, "causal must be 0 or 1 (got %d)", a->causal);
  REFUSE_IF(a->sequences < 0 || a->sequences > kMostIndex || a->total_q < 0 || a->total_q > kMostIndex || a->total_k < 0 || a->total_k > kMostIndex,
            "sequences and rows must be between 0 and 2^30 (got %lld sequences, %lld queries, %lld keys)", (long long)a->sequences,
            (long long)a->total_q, (long long)a->total_k);
  if (a->sequences == 0 || a->total_q == 0) return FLASH_HIP_OK;
  REFUSE_IF(memory && (!a->q || !a->o || ((!a->k || !a->v) && a->total_k > 0)), "null tensor pointer");
  REFUSE_IF(memory && (!a->cu_seqlens_q || !a->cu_seqlens_k), "null cu_seqlens");
  CHECK(check_rows("q", memory ? a->q : nullptr, a->q_token_stride, a->total_q, a->q_head_stride, a->q_heads, 2, 16));
  CHECK(check_rows("k", memory ? a->k : nullptr, a->k_token_stride, a->total_k, a->k_head_stride, a->kv_heads, 2, 16));
  CHECK(check_rows("v", memory ? a->v : nullptr, a->v_token_stride, a->total_k, a->v_head_stride, a->kv_heads, 2, 16));
  CHECK(check_rows("out", memory ? a->o : nullptr, a->o_token_stride, a->total_q, a->o_head_stride, a->q_heads, 2, 16));
  CHECK(check_written("out", a->o_token_stride, a->total_q, a->o_head_stride, a->q_heads, a->d));
  flash_hip::packed::Params& p = *out;
  p.q = (const char*)a->q;
  p.k = (const char*)a->k;
  p.v = (const char*)a->v;
  p.o = (char*)a->o;
  p.cu_q = a->cu_seqlens_q;
  p.cu_k = a->cu_seqlens_k;
  p.q_token = a->q_token_stride * 2;
  p.q_head = a->q_head_stride * 2;
  p.k_token = a->k_token_stride * 2;
  p.k_head = a->k_head_stride * 2;
  p.v_token = a->v_token_stride * 2;
  p.v_head = a->v_head_stride * 2;
  p.o_token = a->o_token_stride * 2;
  p.o_head = a->o_head_stride * 2;
  p.sequences = (int32_t)a->sequences;
  p.total_q = (int32_t)a->total_q;
  p.total_k = (int32_t)a->total_k;
  p.heads = (int32_t)a->q_heads;
  p.kv_heads = (int32_t)a->kv_heads;
  p.d = (int32_t)a->d;
  p.causal = a->causal;
  p.scale_log2 = a->softmax_scale * 1.44269504088896340736f;
  // (many short sequences times heads pass the pipelined kernel's grid first; the other one has the heads in a dimension of their own)
  REFUSE_IF(!flash_hip::packed_mfma_takes(p) && !flash_hip::grid_fits((uint64_t)direct_tiles(p), 256),
            "%lld sequences of %lld rows in all are too many for one call", (long long)a->sequences, (long long)a->total_q);
  return FLASH_HIP_OK;
}

}  // namespace

extern "C" {

int64_t flash_decode_paged_workspace_bytes(const flash_decode_args* args, const flash_paged_cache* cache) {
  DecodePlan plan;
  return plan_decode(args, cache, false, &plan) == FLASH_HIP_OK ? plan.bytes : -1;
}

int flash_decode_paged(const flash_decode_args* a, const flash_paged_cache* c, void* workspace, int64_t workspace_bytes, void* hip_stream) {
  DecodePlan plan;
  CHECK(plan_decode(a, c, true, &plan));
  REFUSE_IF(plan.bytes > 0 && (!workspace || workspace_bytes < plan.bytes), "workspace of %lld bytes is too small: %lld needed",
            (long long)(workspace ? workspace_bytes : 0), (long long)plan.bytes);
  REFUSE_IF((uintptr_t)workspace % 16 != 0, "workspace must be 16-byte aligned");
  if (c->sequences == 0) return FLASH_HIP_OK;
  const int64_t elem = c->dtype == FLASH_E4M3 ? 1 : 2;
  DecodeParams p{};
  p.q = (const char*)a->q;
  p.o = (char*)a->o;
  p.lse = a->lse;
  p.k = (const char*)c->k;
  p.v = (const char*)c->v;
  p.table = c->page_table;
  p.lens = c->seq_lens;
  p.k_scale = c->k_scale;
  p.v_scale = c->v_scale;
  p.part_o = (float*)workspace;
  p.part_ml = p.part_o + kPartRows * 128;
  p.tickets = (uint32_t*)((char*)workspace + kPartBytes);
  p.q_batch = a->q_batch_stride * 2;
  p.q_head = a->q_head_stride * 2;
  p.o_batch = a->o_batch_stride * 2;
  p.o_head = a->o_head_stride * 2;
  p.pages = pages_of(c, elem);
  p.head_stride = c->head_stride * elem;
  p.table_stride = c->table_stride;
  p.batch = (int32_t)c->sequences;
  p.kv_heads = (int32_t)c->kv_heads;
  p.group = (int32_t)(a->q_heads / c->kv_heads);
  p.d = (int32_t)c->d;
  p.qblocks = (p.group + 15) / 16;
  p.workgroups = plan.workgroups;
  p.scale_log2 = a->softmax_scale * 1.44269504088896340736f;
  const hipStream_t stream = (hipStream_t)hip_stream;
  return plan.tile_d == 64 ? launch_decode<64>(p, a->dtype, elem == 1, stream)
                           : launch_decode<128>(p, a->dtype, elem == 1, stream);
}

int flash_cache_append(const flash_append_args* a, const flash_paged_cache* c, void* hip_stream) {
  namespace ap = flash_hip::append;
  REFUSE_IF(!a, "null flash_append_args");
  CHECK(check_cache(c, a->dtype, true));
  CHECK(check_heads(c->kv_heads, c->kv_heads, c->d));
  REFUSE_IF(a->tokens < 0 || !flash_hip::grid_fits((uint64_t)a->tokens / ap::kMostTokens + 1, ap::kThreads),
            "between 0 and %lld tokens (got %lld)", (1ll << 32) / ap::kThreads * ap::kMostTokens - ap::kMostTokens - 1, (long long)a->tokens);
  REFUSE_IF(!a->cu_seqlens && a->tokens != c->sequences, "without cu_seqlens one token per sequence is needed (got %lld tokens, %lld sequences)",
            (long long)a->tokens, (long long)c->sequences);
  REFUSE_IF(flash_hip::rows_meet({c->num_pages, c->page_stride}, {c->kv_heads, c->head_stride}, {c->page_size, c->slot_stride}, c->d),
            "cache: rows must not overlap in memory (strides %lld, %lld, %lld)", (long long)c->page_stride, (long long)c->head_stride, (long long)c->slot_stride);
  if (a->tokens == 0 || c->sequences == 0) return FLASH_HIP_OK;
  REFUSE_IF(!a->k || !a->v, "null tensor pointer");
  CHECK(check_rows("k", a->k, a->k_token_stride, a->tokens, a->k_head_stride, c->kv_heads, 2, 16));
  CHECK(check_rows("v", a->v, a->v_token_stride, a->tokens, a->v_head_stride, c->kv_heads, 2, 16));
  const int64_t elem = c->dtype == FLASH_E4M3 ? 1 : 2;
  ap::Params p{};
  p.k = (const char*)a->k;
  p.v = (const char*)a->v;
  p.k_cache = (char*)c->k;
  p.v_cache = (char*)c->v;
  p.table = c->page_table;
  p.lens = c->seq_lens;
  p.cu = a->cu_seqlens;
  p.k_scale = c->k_scale;
  p.v_scale = c->v_scale;
  p.k_token = a->k_token_stride * 2;
  p.k_head = a->k_head_stride * 2;
  p.v_token = a->v_token_stride * 2;
  p.v_head = a->v_head_stride * 2;
  p.pages = pages_of(c, elem);
  p.head_stride = c->head_stride * elem;
  p.table_stride = c->table_stride;
  p.batch = (int32_t)c->sequences;
  p.tokens_total = (int32_t)a->tokens;
  p.kv_heads = (int32_t)c->kv_heads;
  p.d = (int32_t)c->d;
  // about four workgroups a compute unit
  const int64_t each = (a->tokens + 1023) / 1024;
  p.tokens = (int32_t)(each < ap::kMostTokens ? each : ap::kMostTokens);
  const dim3 grid((uint32_t)((a->tokens + p.tokens - 1) / p.tokens));
  const hipStream_t stream = (hipStream_t)hip_stream;
  if (elem == 2) {
    hipLaunchKernelGGL((ap::append_kernel<flash_hip::direct::kHalf, false>), grid, dim3(ap::kThreads), 0, stream, p);  // moves bits
  } else if (a->dtype == FLASH_F16) {
    hipLaunchKernelGGL((ap::append_kernel<flash_hip::direct::kHalf, true>), grid, dim3(ap::kThreads), 0, stream, p);
  } else {
    hipLaunchKernelGGL((ap::append_kernel<flash_hip::direct::kBfloat, true>), grid, dim3(ap::kThreads), 0, stream, p);
  }
  return launched("flash_cache_append");
}

int64_t flash_fwd_packed_workspace_bytes(const flash_packed_args* args) {
  flash_hip::packed::Params p{};
  if (plan_packed(args, false, &p) != FLASH_HIP_OK) return -1;
  return p.total_q > 0 ? flash_hip::packed_mfma_workspace(p) : 0;
}
int flash_fwd_packed(const flash_packed_args* a, void* workspace, int64_t workspace_bytes, void* hip_stream) {
  flash_hip::packed::Params p{};
  CHECK(plan_packed(a, true, &p));
  if (p.total_q == 0) return FLASH_HIP_OK;
  if (workspace) {
    const int64_t need = flash_hip::packed_mfma_workspace(p);
    REFUSE_IF(workspace_bytes < need, "workspace of %lld bytes is too small: %lld needed", (long long)workspace_bytes, (long long)need);
    REFUSE_IF((uintptr_t)workspace % 16 != 0, "workspace must be 16-byte aligned");
  }
  const hipStream_t stream = (hipStream_t)hip_stream;
  if (flash_hip::packed_mfma_takes(p)) return flash_hip::launch_packed_mfma(p, a->dtype == FLASH_BF16, workspace, stream);
  using namespace flash_hip::direct;
  if (a->d <= 64) return a->dtype == FLASH_F16 ? launch_packed_direct<64, kHalf>(p, stream) : launch_packed_direct<64, kBfloat>(p, stream);
  return a->dtype == FLASH_F16 ? launch_packed_direct<128, kHalf>(p, stream) : launch_packed_direct<128, kBfloat>(p, stream);
}

}  // extern "C"
