// Launch of the pipelined kernel for packed prompts.  Compiled without regard to NaN like the kernels whose body it
// shares (fmaxf of matrix results must be one instruction); what may be NaN here is looked at through its bits.
#include "../../include/flash_hip.h"

#include <hip/hip_runtime.h>

#include <atomic>

#include "attn_packed_mfma.hpp"
#include "host.hpp"

namespace flash_hip {

namespace {

template <int D, typename TO, bool CAUSAL>
int launch(packed::Params p, hipStream_t stream) {
  constexpr uint32_t kLds = (uint32_t)m16::Cfg<D>::kLdsBytes;
  static std::atomic<uint64_t> done{0};  // one bit per device: the kernel's LDS size has been set there
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return set_error(FLASH_HIP_ERR_RUNTIME, "hipGetDevice failed: %s", hipGetErrorString(e));
  const bool cached = dev >= 0 && dev < 64;
  if (!cached || !((done.load(std::memory_order_acquire) >> dev) & 1u)) {
    e = hipFuncSetAttribute((const void*)m16::attn_fwd_kernel_packed<D, TO, CAUSAL>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)kLds);
    if (e != hipSuccess) return set_error(FLASH_HIP_ERR_LDS, "Failed to set dynamic shared memory size %u: %s", kLds, hipGetErrorString(e));
    if (cached) done.fetch_or((uint64_t)1 << dev, std::memory_order_release);
  }
  hipLaunchKernelGGL((m16::attn_fwd_kernel_packed<D, TO, CAUSAL>), dim3(p.tiles * (uint32_t)p.heads), dim3(m16::kThreads), kLds, stream, p);
  e = hipGetLastError();
  if (e != hipSuccess) return set_error(FLASH_HIP_ERR_RUNTIME, "flash_fwd_packed: kernel launch failed: %s", hipGetErrorString(e));
  return FLASH_HIP_OK;
}

template <int D, typename TO>
int launch(const packed::Params& p, hipStream_t stream) {
  return p.causal ? launch<D, TO, true>(p, stream) : launch<D, TO, false>(p, stream);
}

}  // namespace

bool packed_mfma_takes(const packed::Params& p) {
  const int64_t most = (int64_t)kOob / m16::kPackedRows;  // a row's bytes: 256 of them stay below kOob
  const int64_t tiles = (int64_t)p.total_q / m16::kPackedRows + 2 * (int64_t)p.sequences;
  return p.q_token <= most && p.o_token <= most && p.k_token <= most && p.v_token <= most && tiles * p.heads < ((int64_t)1 << 31);
}

int launch_packed_mfma(packed::Params p, bool bf16, hipStream_t stream) {
  // a sequence has at most two tiles more than whole ones among its rows (its first one may be short, and its last one)
  p.tiles = (uint32_t)(p.total_q / m16::kPackedRows + 2 * p.sequences);
  if (p.d <= 64) return bf16 ? launch<64, m16::bf16_out>(p, stream) : launch<64, f16>(p, stream);
  return bf16 ? launch<128, m16::bf16_out>(p, stream) : launch<128, f16>(p, stream);
}

}  // namespace flash_hip
