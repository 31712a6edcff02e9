// Writes the keys and values of new tokens into the pages of a cache.
//
// Token t (row t of k and v) of sequence b, cu[b] <= t < cu[b + 1], goes to position lens[b] - (cu[b + 1] - t): `lens`
// counts the new tokens already.  A copy, or x -> e4m3(clamp(x / scale)) with one scale per head; bound by HBM,
// 2 * d * kv_heads * (2 + bytes of a cache element) bytes a token.  A workgroup takes `tokens` consecutive ones:
// their targets are looked up once (the sequence by bisection of cu, in LDS where it fits) and every lane then moves
// chunks of 8 elements, 16-byte loads, with consecutive lanes on consecutive chunks of a token's row.
// Measured: 8509 tokens of 13 prompts, 8 heads of 128, 16-bit: 13-14 us, 4.9-5.3 TB/s read and written (a large copy: 4.6),
// into e4m3 19 us; 16 single tokens into an e4m3 cache: 3.3 us, a launch and a chain of three loads.
// Tokens outside every sequence, positions beyond the table and pages outside the cache are not written.
#pragma once

#include "attn_direct.hpp"
#include "serving_index.hpp"

namespace flash_hip {
namespace append {

using namespace direct;

constexpr int kThreads = 256;
constexpr int kMostTokens = 32;   // per workgroup
constexpr int kCuInLds = 2048;    // offsets kept in LDS

struct Params {
  const char* k;
  const char* v;
  char* k_cache;
  char* v_cache;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* cu;  // null: token t belongs to sequence t
  const float* k_scale;
  const float* v_scale;
  int64_t k_token, k_head, v_token, v_head;       // bytes
  Pages pages;
  int64_t head_stride;                            // bytes
  int64_t table_stride;                           // entries
  int32_t batch, tokens_total, kv_heads, d;
  int32_t tokens;                                 // per workgroup
};

// The nearest e4m3 values, ties to even, of values beyond +-448 the largest; NaN stays NaN
__device__ __forceinline__ float within_e4m3(float x) { return x != x ? x : fminf(fmaxf(x, -448.f), 448.f); }
__device__ __forceinline__ uint32_t to_e4m3(float a, float b, float c, float e) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(within_e4m3(a), within_e4m3(b), 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(within_e4m3(c), within_e4m3(e), w, true);
}

template <int EK, bool CACHE8>
__global__ __launch_bounds__(kThreads) void append_kernel(const Params p) {
#if defined(__HIP_DEVICE_COMPILE__)
  __shared__ int32_t sh_cu[kCuInLds + 1];
  __shared__ int64_t sh_at[kMostTokens];  // bytes from the cache's start, -1: nowhere
  const int32_t t0 = (int32_t)blockIdx.x * p.tokens;
  const int32_t count = p.tokens_total - t0 < p.tokens ? p.tokens_total - t0 : p.tokens;
  const bool in_lds = p.cu && p.batch <= kCuInLds;
  if (in_lds) {
    for (int32_t i = threadIdx.x; i <= p.batch; i += kThreads) sh_cu[i] = p.cu[i];
    __syncthreads();
  }
  if ((int32_t)threadIdx.x < count) {
    const int32_t t = t0 + (int32_t)threadIdx.x;
    int32_t b = t, behind = 1;  // rows of the sequence from this one on
    if (p.cu) {
      auto cu = [&](int32_t i) { return in_lds ? sh_cu[i] : p.cu[i]; };
      b = sequence_of(cu, p.batch, t);
      behind = b >= 0 ? cu(b + 1) - t : 0;
    }
    int64_t at = -1;
    if (b >= 0 && b < p.batch) {
      const int32_t pos = new_position(p.pages, p.lens[b], behind);
      if (pos >= 0) at = position_offset(p.pages, p.table[(int64_t)b * p.table_stride + (pos >> p.pages.page_shift)], pos);
    }
    sh_at[threadIdx.x] = at;
  }
  __syncthreads();
  const uint32_t per_head = (uint32_t)p.d / 8u, per_token = (uint32_t)p.kv_heads * per_head;
  const uint32_t chunks = (uint32_t)count * per_token;
  for (uint32_t x = threadIdx.x; x < 2 * chunks; x += kThreads) {
    const bool is_v = x >= chunks;
    const uint32_t y = is_v ? x - chunks : x;
    const uint32_t t = y / per_token, rest = y - t * per_token, h = rest / per_head, c = rest - h * per_head;
    const int64_t at = sh_at[t];
    if (at < 0) continue;
    const char* src = is_v ? p.v + (int64_t)(t0 + (int32_t)t) * p.v_token + (int64_t)h * p.v_head
                           : p.k + (int64_t)(t0 + (int32_t)t) * p.k_token + (int64_t)h * p.k_head;
    const u32x4 w = *(const u32x4*)(src + c * 16);
    char* dst = (is_v ? p.v_cache : p.k_cache) + at + (int64_t)h * p.head_stride;
    if constexpr (CACHE8) {
      const float* scales = is_v ? p.v_scale : p.k_scale;
      const float scale = scales ? scales[h] : 1.f;
      f32x2 f[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = unpack2<EK>(w[i]) / scale;
      *(u32x2*)(dst + c * 8) = u32x2{to_e4m3(f[0][0], f[0][1], f[1][0], f[1][1]), to_e4m3(f[2][0], f[2][1], f[3][0], f[3][1])};
    } else {
      *(u32x4*)(dst + c * 16) = w;
    }
  }
#endif
}

}  // namespace append
}  // namespace flash_hip
