// Launch of the pipelined kernel for packed prompts.  Unlike the other unit that compiles the kernel's body this one is compiled
// with NaNs: masked places may hold them, and rows that meet one are computed again here, with plain arithmetic on it.
#define FLASH_M16_HONOR_NANS 1
#include "../../include/flash_hip.h"

#include <hip/hip_runtime.h>

#include <atomic>

#include "attn_packed_mfma.hpp"
#include "host.hpp"

namespace flash_hip {

namespace {

using Kernel = void (*)(const packed::Params);

template <Kernel KERNEL, int LDS>
int launch(const packed::Params& p, hipStream_t stream) {
  constexpr uint32_t kLds = (uint32_t)LDS;
  static std::atomic<uint64_t> done{0};  // one bit per device: the kernel's LDS size has been set there
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return set_error(FLASH_HIP_ERR_RUNTIME, "hipGetDevice failed: %s", hipGetErrorString(e));
  const bool cached = dev >= 0 && dev < 64;
  if (!cached || !((done.load(std::memory_order_acquire) >> dev) & 1u)) {
    e = hipFuncSetAttribute((const void*)KERNEL, hipFuncAttributeMaxDynamicSharedMemorySize, (int)kLds);
    if (e != hipSuccess) return set_error(FLASH_HIP_ERR_LDS, "Failed to set dynamic shared memory size %u: %s", kLds, hipGetErrorString(e));
    if (cached) done.fetch_or((uint64_t)1 << dev, std::memory_order_release);
  }
  hipLaunchKernelGGL(KERNEL, dim3(p.items * (uint32_t)p.parts), dim3(m16::kThreads), kLds, stream, p);
  e = hipGetLastError();
  if (e != hipSuccess) return set_error(FLASH_HIP_ERR_RUNTIME, "flash_fwd_packed: kernel launch failed: %s", hipGetErrorString(e));
  return FLASH_HIP_OK;
}

template <typename TO>
struct HalfOut {
  using type = TO;
};
template <>
struct HalfOut<m16::bf16_out> {
  using type = m16h::bf16_out;
};

// Long sequences with work for every compute unit take the 256-row items: each K/V tile is fetched and read from LDS by half
// as many waves.  Shorter ones take the 128-row items, two workgroups to a compute unit, of which one computes while
// the other starts or ends.  Measured, 128-row / 256-row, us: 32 heads of 128 over 8, 16 x 512 rows 67 / 74, 8 x 1024
// 88 / 97, 4 x 2048 139 / 141, 2 x 4096 243 / 239, 8192 457 / 442, 16384 1775 / 1719; 32 heads of 64, 8 x 1024 56 / 66,
// 2 x 4096 152 / 154, 8192 288 / 282; 973 rows of 16 heads of 64 45 / 67 (not cut, see parts_of).
bool take_half(const packed::Params& p) {
  return (int64_t)p.total_k < (int64_t)4096 * p.sequences || (int64_t)p.total_q / m16::kPackedRows * p.heads < 512;
}
// The grid's tiles: a sequence has at most two more than whole ones among its rows, its last one and, where its numbers of
// queries and keys differ and the diagonal is cut, its first one.
int extra_tiles(const packed::Params& p) { return p.causal && !(p.cu_q == p.cu_k && p.total_q == p.total_k) ? 2 : 1; }
void set_grid(packed::Params& p, int64_t rows, int extra) {
  p.extra = extra;
  p.tiles = (uint32_t)(p.total_q / rows + (int64_t)p.extra * p.sequences);
  p.items = (uint32_t)packed_grid(p.tiles, (uint32_t)p.heads, (uint32_t)p.kv_heads);
  p.parts = 1;
}
// Fewer 128-row items than compute units, with enough keys to cut: the keys of an item are dealt to several workgroups, as
// many as fill the chip (two on each of 256 compute units) by what there may be of items.  Measured, cut / whole, us: 128 rows over 32768 keys, 8 heads of 128, 69 / 451; 256 over 8192, 32 heads,
// 57 / 115; 4096 rows, 4 heads, 41.5 / 60.6; 973 rows of three sequences, 16 heads of 64, 30 / 45; with an item for every
// compute unit there is nothing to gain: 4096 rows, 8 heads, 64 / 62, 1024 over 8192, 32 heads, 124.6 / 123.
int parts_of(const packed::Params& p, int extra) {
  constexpr int64_t kUnits = 256, kMostSlots = 4 * kUnits;
  if (!take_half(p) || p.total_k < 2 * m16h::kPartTiles * kBc) return 1;
  packed::Params h = p;
  set_grid(h, m16h::kPackedRows, extra);
  const int64_t items = ((int64_t)p.total_q / m16h::kPackedRows + p.sequences) * p.heads;
  if (items >= kUnits) return 1;
  const int64_t wanted = (2 * kUnits + items - 1) / items, room = kMostSlots / h.items;
  static_assert(kMostSlots / 2 * 4 <= FLASH_PACKED_TICKET_BYTES, "a ticket for each item that is cut");
  const int64_t parts = wanted < room ? wanted : room;
  return (int)(parts < 1 ? 1 : (parts < m16h::kMostParts ? parts : m16h::kMostParts));
}
// floats of a part of an item: its rows of O^T, and their reference and sum
int64_t part_floats(const packed::Params& p) { return (int64_t)m16h::kPackedRows * ((p.d <= 64 ? 64 : 128) + 2); }

template <int D, typename TO>
int launch(packed::Params p, void* workspace, hipStream_t stream) {
  using TH = typename HalfOut<TO>::type;
  if (take_half(p)) {
    const int extra = extra_tiles(p), parts = workspace ? parts_of(p, extra) : 1;
    set_grid(p, m16h::kPackedRows, extra);
    if (parts > 1) {
      p.parts = parts;
      p.tickets = (uint32_t*)workspace;
      p.part_o = (float*)((char*)workspace + FLASH_PACKED_TICKET_BYTES);
      p.part_ml = p.part_o + (int64_t)p.items * parts * m16h::kPackedRows * D;
      return p.causal ? launch<m16h::attn_fwd_kernel_packed<D, TH, true, true>, m16h::kPackedLds<D>>(p, stream)
                      : launch<m16h::attn_fwd_kernel_packed<D, TH, false, true>, m16h::kPackedLds<D>>(p, stream);
    }
    return p.causal ? launch<m16h::attn_fwd_kernel_packed<D, TH, true, false>, m16h::kPackedLds<D>>(p, stream)
                    : launch<m16h::attn_fwd_kernel_packed<D, TH, false, false>, m16h::kPackedLds<D>>(p, stream);
  }
  set_grid(p, m16::kPackedRows, extra_tiles(p));
  return p.causal ? launch<m16::attn_fwd_kernel_packed<D, TO, true, false>, m16::kPackedLds<D>>(p, stream)
                  : launch<m16::attn_fwd_kernel_packed<D, TO, false, false>, m16::kPackedLds<D>>(p, stream);
}

}  // namespace

// (the grids of cut items have at most 1024 workgroups, see parts_of)
static_assert(m16::kThreads == m16h::kThreads, "one limit of the grid");
bool packed_mfma_takes(const packed::Params& p) {
  const int64_t most = (int64_t)kOob / m16::kPackedRows;  // a row's bytes: 256 of them stay below kOob
  const int64_t tiles = (int64_t)p.total_q / (take_half(p) ? m16h::kPackedRows : m16::kPackedRows) + (int64_t)extra_tiles(p) * p.sequences;
  return p.q_token <= most && p.o_token <= most && p.k_token <= most && p.v_token <= most && tiles < ((int64_t)1 << 31) &&
         grid_fits(packed_grid((uint64_t)tiles, (uint32_t)p.heads, (uint32_t)p.kv_heads), m16::kThreads);
}

// By sizes alone: room for the call whether its keys are cut like its queries (the same offsets, known at the launch) or not.
int64_t packed_mfma_workspace(const packed::Params& p) {
  if (!packed_mfma_takes(p)) return 0;
  int64_t most = 0;
  for (int extra = p.causal && p.total_q != p.total_k ? 2 : 1; extra <= (p.causal ? 2 : 1); ++extra) {
    const int parts = parts_of(p, extra);
    if (parts == 1) continue;
    packed::Params h = p;
    set_grid(h, m16h::kPackedRows, extra);
    const int64_t bytes = FLASH_PACKED_TICKET_BYTES + (int64_t)h.items * parts * part_floats(p) * 4;
    most = bytes > most ? bytes : most;
  }
  return most;
}

int launch_packed_mfma(const packed::Params& p, bool bf16, void* workspace, hipStream_t stream) {
  if (p.d <= 64) return bf16 ? launch<64, m16::bf16_out>(p, workspace, stream) : launch<64, f16>(p, workspace, stream);
  return bf16 ? launch<128, m16::bf16_out>(p, workspace, stream) : launch<128, f16>(p, workspace, stream);
}

}  // namespace flash_hip
