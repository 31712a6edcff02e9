// Attention of one new token of every sequence over a paged key-value cache, split over the cache's length, and
// the join of the parts.  What a wave does with its keys is in attn_direct.hpp.
//
// What bounds it: the cache is read once, 2 * d * (bytes of an element) per key and K/V head, against
// 4 * d * (heads per K/V head) operations: at 8 query heads per K/V head and 16-bit values 16 operations a
// byte, two orders of magnitude below what the matrix cores could do in that time.  The kernel is made to keep
// loads in flight.  Measured: 8 sequences of 1024-2048, 96 heads of 128, fp16: 117 us, 6.0 TB/s; 32 ragged ones of 0-8192, 32
// heads over 8: 63 us, 5.1 TB/s; one of 130001: 99 us, 5.4 TB/s; e4m3, 16 of 7000-16384, 64 heads over 8: 82 us, 5.1 TB/s;
// one of 1023: 8.1 us, two chains of memory latency.
//
// Work split.  Sequence b of length n_b is cut into U_b = max(1, ceil(n_b / kUnit)) units; all units of all
// (sequence, K/V head, query block) triples stand in one line, b outermost, and workgroup w takes the units
// [w c, (w + 1) c) of it, c = ceil(total / workgroups).  Every workgroup then reads the same number of keys
// whatever the lengths are, and nothing about them has to be known on the host, so that a captured graph stays
// valid while they grow.  Every wave finds the line's length and the workgroup's place in it from the lengths
// themselves (a scan over 64 of them per step).  A workgroup that holds all units of a triple writes its output;
// otherwise it leaves (o, m, l) in the workspace and takes a ticket of the triple; whoever takes the last one adds
// the parts up, in the line's order, so that the result does not depend on timing, and resets the tickets.  Nobody waits.
#pragma once

#include "attn_direct.hpp"
#include "serving_index.hpp"

namespace flash_hip {
namespace paged {

using namespace direct;

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kMostWorkgroups = 768;  // three to each of 256 compute units

struct Params {
  const char* q;
  char* o;
  float* lse;  // may be null
  const char* k;
  const char* v;
  const int32_t* table;
  const int32_t* lens;
  const float* k_scale;  // per K/V head, null: 1
  const float* v_scale;
  float* part_o;         // [2 * workgroups][16][D]
  float* part_ml;        // [2 * workgroups][16][2]
  uint32_t* tickets;     // one for each triple; zero, and left zero
  int64_t q_batch, q_head, o_batch, o_head;     // bytes
  Pages pages;                                   // K and V alike
  int64_t head_stride;                           // bytes
  int64_t table_stride;                          // entries
  int32_t batch, kv_heads, group;                // group: query heads per K/V head
  int32_t d;
  int32_t qblocks;                               // blocks of 16 query heads per K/V head
  uint32_t workgroups;
  float scale_log2;                              // softmax scale * log2 e
};

// keys of a unit: every wave of the workgroup takes one step
template <int D, bool CACHE8>
constexpr int kSub = (D == 64 || CACHE8) ? 2 : 1;
template <int D, bool CACHE8>
constexpr int kUnit = kWaves * 32 * kSub<D, CACHE8>;

__device__ __forceinline__ int32_t length_of(const Params& p, int32_t b) { return cache_length(p.pages, p.lens[b]); }
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); }

// K and V are read once: without a place in the caches a large read runs at 6.4-6.6 TB/s on this chip, with one at 5.7-5.9
// (512 MB and 1 GB, 8 and 16 KB of every wave in flight, in order or not).
template <typename T>
__device__ __forceinline__ T stream(const T* p) {
  return __builtin_nontemporal_load(p);
}

template <int D, int EK, bool CACHE8, bool FULL, bool PAGE16>
__global__ __launch_bounds__(kThreads, 3) void decode_kernel(const Params p) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int NS = kSub<D, CACHE8>;
  constexpr int kUnitKeys = kUnit<D, CACHE8>;
  using S = Step<D, EK, CACHE8, NS>;
  constexpr int kRowFloats = D + 4;  // rows of the waves' sums, shifted by four banks each
  // the waves' sums; later the weights of a triple's parts (at most `workgroups` of them, for 8 rows)
  constexpr int kShFloats = kWaves * 16 * kRowFloats > 8 * kMostWorkgroups ? kWaves * 16 * kRowFloats : 8 * kMostWorkgroups;
  __shared__ __attribute__((aligned(16))) float sh[kShFloats];
  __shared__ __attribute__((aligned(16))) f32x4 sh_sum[kThreads];
  __shared__ float sh_ml[kWaves][16][2];
  __shared__ float sh_l[8];
  __shared__ uint32_t sh_ticket;
  float(&sh_o)[kWaves][16][kRowFloats] = *(float(*)[kWaves][16][kRowFloats]) & sh[0];

  // Parts go to memory and come from there past the L2s, which the XCDs do not share (sc0 sc1: system scope).  A release
  // and an acquire at agent scope write back and drop whole L2s instead: 174 us where this takes 63 (32 ragged sequences).
  constexpr int kThrough = 17;
  const __amdgpu_buffer_rsrc_t part_o = __builtin_amdgcn_make_buffer_rsrc(p.part_o, 0, (int)(p.workgroups * 2u * 16u * D * 4u), 0x00020000);
  const __amdgpu_buffer_rsrc_t part_ml = __builtin_amdgcn_make_buffer_rsrc(p.part_ml, 0, (int)(p.workgroups * 2u * 16u * 8u), 0x00020000);

  const int lane = threadIdx.x & 63;
  const int wave = (int)uniform(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;

  // ---- this workgroup's piece of the line -------------------------------------------------------------
  const uint32_t vheads = (uint32_t)(p.kv_heads * p.qblocks);
  auto units_at = [&](int32_t b0) __attribute__((always_inline)) {
    return b0 + lane < p.batch ? units_of(length_of(p, b0 + lane), kUnitKeys) * vheads : 0u;
  };
  uint32_t own = units_at(0), sum = wave_scan(own);
  uint32_t total = (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
  for (int32_t b0 = 64; b0 < p.batch; b0 += 64) total += (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(units_at(b0)), 63);
  const uint32_t c = units_each(total, p.workgroups);
  const uint32_t r_begin = blockIdx.x * c;
  if (r_begin >= total) return;
  const uint32_t r_end = r_begin + c < total ? r_begin + c : total;
  int32_t b = 0;
  uint32_t first = 0;  // units of the line before sequence b
  for (int32_t b0 = 0;;) {
    const uint64_t past = __builtin_amdgcn_ballot_w64(first + sum > r_begin);
    if (past != 0) {
      const int at = __builtin_ctzll(past);
      b = b0 + at;
      first += (uint32_t)__builtin_amdgcn_readlane((int)(sum - own), at);
      break;
    }
    first += (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
    b0 += 64;
    own = units_at(b0);
    sum = wave_scan(own);
  }
  int32_t len = (int32_t)uniform((uint32_t)length_of(p, b));
  uint32_t units = units_of(len, kUnitKeys);
  uint32_t vh = (r_begin - first) / units;
  uint32_t u0 = (r_begin - first) - vh * units;

  for (uint32_t r = r_begin; r < r_end;) {
    const uint32_t left = r_end - r;
    const uint32_t u1 = units - u0 < left ? units : u0 + left;
    const int32_t kvh = (int32_t)(vh / (uint32_t)p.qblocks), qb = (int32_t)(vh - (uint32_t)(kvh * p.qblocks));
    const int32_t row0 = qb * 16;  // first query head inside the group
    const int32_t rows = p.group - row0 < 16 ? p.group - row0 : 16;

    // queries of the block, zeros for the heads that do not exist
    u32x4 qf[S::kKS];
    const char* src = p.q + (int64_t)b * p.q_batch + (int64_t)(kvh * p.group + row0 + (n < rows ? n : 0)) * p.q_head;
#pragma unroll
    for (int ks = 0; ks < S::kKS; ++ks) {
      const int col = FULL ? S::column(ks, g) : q_column(CACHE8, ks, g, p.d);
      const bool there = n < rows && (FULL || col >= 0);
      const u32x4 x = *(const u32x4*)(src + (there ? col * 2 : 0));
      qf[ks] = there ? x : u32x4{0u, 0u, 0u, 0u};
    }
    const float sc = p.scale_log2 * (CACHE8 && p.k_scale ? p.k_scale[kvh] : 1.f);
    const char* kh = p.k + (int64_t)kvh * p.head_stride;
    const char* vv = p.v + (int64_t)kvh * p.head_stride;
    const uint32_t slot_stride = (uint32_t)p.pages.slot_stride;
    const int32_t* row_of_table = p.table + (int64_t)b * p.table_stride;

    // Place in the cache of the lane's key in this wave's step of unit u: its page's entry, then bytes (-1: no such key,
    // or an entry outside the cache).
    auto page_of = [&](uint32_t u) __attribute__((always_inline)) -> int32_t {
      const int32_t key = (int32_t)u * kUnitKeys + wave * S::kKeys + lane;
      return (lane < S::kKeys && key < len && u < u1) ? row_of_table[key >> p.pages.page_shift] : -1;
    };
    // (wave-uniform) which keys of the step exist; `at`: where they lie, the start of the cache for the others, which are
    // read from there and masked
    auto place = [&](uint32_t u, int32_t page, int64_t& at) __attribute__((always_inline)) -> uint64_t {
      const int64_t x = position_offset(p.pages, page, (int32_t)u * kUnitKeys + wave * S::kKeys + lane);
      at = x < 0 ? 0 : x;
      return __builtin_amdgcn_ballot_w64(x >= 0);
    };
    // Row of a key: with pages of at least 16 positions every 16-key tile lies in one page, whose start is a scalar
    auto tile_start = [&](int64_t at, int t) __attribute__((always_inline)) -> int64_t {
      const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)at, 16 * t);
      const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)((uint64_t)at >> 32), 16 * t);
      return (int64_t)(((uint64_t)hi << 32) | lo);
    };
    // (offsets inside a page, opaque so that they stay 32-bit registers beside a scalar base)
    uint32_t k_row = (uint32_t)n * slot_stride, v_row[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v_row[j] = (uint32_t)(4 * g + j) * slot_stride + (FULL || n * S::kE < p.d ? (uint32_t)(n * S::kE * S::kElem) : 0u);
    // A load never leaves its row: 16 bytes of 8-bit values may be 8 columns more than the row has from there on.  Such a load
    // begins earlier, and the query's elements stand beside the columns that it holds (q_column).
    auto load_k = [&](typename S::KBlock& k, int64_t at) __attribute__((always_inline)) {
      if constexpr (PAGE16) asm volatile("" : "+v"(k_row));
      if constexpr (!FULL && CACHE8) {
        if (p.d == 8) {  // rows shorter than a load
#pragma unroll
          for (int t = 0; t < 2 * NS; ++t) {
            const char* src = PAGE16 ? kh + tile_start(at, t) + k_row : kh + __shfl(at, 16 * t + n);
            const u32x2 x = stream((const u32x2*)src);
#pragma unroll
            for (int i = 0; i < S::kKLoads; ++i) k[t][i] = u32x4{x[0], x[1], 0u, 0u};
          }
          return;
        }
      }
#pragma unroll
      for (int t = 0; t < 2 * NS; ++t) {
        const char* src = PAGE16 ? kh + tile_start(at, t) : kh + __shfl(at, 16 * t + n);
#pragma unroll
        for (int i = 0; i < S::kKLoads; ++i) {
          if constexpr (PAGE16 && FULL) {
            k[t][i] = stream((const u32x4*)(src + (k_row + (uint32_t)(S::load_column(0, g) * S::kElem)) + S::load_column(i, 0) * S::kElem));
          } else {
            const int col = S::load_column(i, g), from = FULL ? col : row_load(col, 16 / S::kElem, p.d);
            k[t][i] = stream((const u32x4*)(src + ((PAGE16 ? k_row : 0u) + (uint32_t)(from * S::kElem))));
            // (infinite elements of a 16-bit row times a query's zero would be NaN; e4m3 has none)
            if constexpr (!FULL && !CACHE8) {
              if (col >= p.d) k[t][i] = u32x4{0u, 0u, 0u, 0u};
            }
          }
        }
      }
    };
    auto load_v = [&](typename S::VBlock& v, int64_t at) __attribute__((always_inline)) {
      if constexpr (PAGE16) asm volatile("" : "+v"(v_row[0]), "+v"(v_row[1]), "+v"(v_row[2]), "+v"(v_row[3]));
#pragma unroll
      for (int s = 0; s < NS; ++s) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if constexpr (PAGE16) {
            v[s][j] = stream((const typename S::VWord*)(vv + tile_start(at, 2 * s + j / 4) + v_row[j % 4]));
          } else {
            v[s][j] = stream((const typename S::VWord*)(vv + __shfl(at, S::v_key(s, g, j)) + (FULL || n * S::kE < p.d ? n * S::kE * S::kElem : 0)));
          }
        }
      }
    };

    // A step's K and V are fetched together at its beginning, the pages' entries a step ahead: 16 KB in flight per wave at
    // d = 128, and the registers leave room for three waves on a SIMD.
    typename S::State st;
    auto attend = [&](auto careful) __attribute__((always_inline)) {
      S::clear(st);
      int32_t page = page_of(u0);
      for (uint32_t u = u0; u < u1; ++u) {
        typename S::KBlock k;
        typename S::VBlock v;
        int64_t at;
        const uint64_t valid = place(u, page, at);
        page = page_of(u + 1);
        if (valid == 0) continue;
        load_k(k, at);
        load_v(v, at);
        typename S::Weights w;
        S::template weigh<false>(st, w, k, qf, valid, sc, lane);
        S::clear_missing(v, valid, lane);
        S::template accumulate<decltype(careful)::value>(st, w, v);
      }
    };
    attend(std::false_type{});
    // NaN may come from an infinite value (rare: the part is worked out again with care)
    if (S::holds_nan(st)) attend(std::true_type{});

    // ---- the four waves' parts --------------------------------------------------------------------------
    const bool complete = u0 == 0 && u1 == units;
    const uint32_t slot = part_slot(blockIdx.x, c, r - u0);
    const float vs = CACHE8 && p.v_scale ? p.v_scale[kvh] : 1.f;
    constexpr float kLower = 1.f / kRaise<EK>;  // (into the sum's inverse, apart from vs: their product may pass fp32's range)
    const float l = quad_sum(st.l);
    if (g == 0) {
      sh_ml[wave][n][0] = st.m;
      sh_ml[wave][n][1] = l;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int e = 0; e < S::kE; e += 4) {
        *(f32x4*)&sh_o[wave][n][S::kE * (4 * g + i) + e] =
            f32x4{st.o[e][i], st.o[e + 1][i], st.o[e + 2][i], st.o[e + 3][i]};
      }
    }
    __syncthreads();
    constexpr int kPieces = D / 4;
    for (int x = threadIdx.x; x < 16 * kPieces && x / kPieces < rows; x += kThreads) {
      const int row = x / kPieces, col = 4 * (x % kPieces);
      if (col < p.d) {
        float m = kMinusInf;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) m = fmaxf(m, sh_ml[w][row][0]);
        const float ref = m == kMinusInf ? 0.f : m;
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
        float l = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
          const float f = __builtin_amdgcn_exp2f(sh_ml[w][row][0] - ref);
          l += f * sh_ml[w][row][1];
          sum += f * *(const f32x4*)&sh_o[w][row][col];
        }
        if (complete) {
          const int32_t head = kvh * p.group + row0 + row;
          const float inv = l == 0.f ? 0.f : kLower / l, unit = l == 0.f ? 0.f : vs;
          *(u32x2*)(p.o + (int64_t)b * p.o_batch + (int64_t)head * p.o_head + col * 2) =
              u32x2{pack2<EK>(sum[0] * inv * unit, sum[1] * inv * unit), pack2<EK>(sum[2] * inv * unit, sum[3] * inv * unit)};
          if (p.lse && col == 0) {
            p.lse[(int64_t)b * p.kv_heads * p.group + head] = l == 0.f ? kMinusInf : (m + log2f(l)) * 0.693147180559945309f;
          }
        } else {
          const uint32_t at = slot * 16 + (uint32_t)row;
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, sum), part_o, (at * D + (uint32_t)col) * 4u, 0, kThrough);
          if (col == 0) __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(m), __float_as_uint(l)}, part_ml, at * 8u, 0, kThrough);
        }
      }
    }
    __syncthreads();

    // ---- the last workgroup of a triple to come here adds its parts up, in the line's order
    if (!complete) {
      const uint32_t start = r - u0, w0 = start / c, parts = (start + units - 1) / c - w0 + 1;
      uint32_t* const ticket = p.tickets + ((uint32_t)b * vheads + vh);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the part has reached memory
      __syncthreads();
      if (threadIdx.x == 0) sh_ticket = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __syncthreads();
      if (sh_ticket == parts - 1) {
        asm volatile("" ::: "memory");
        if (threadIdx.x == 0) __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        auto row_of = [&](uint32_t i, int row) __attribute__((always_inline)) { return part_slot(w0 + i, c, start) * 16 + (uint32_t)row; };
        // Loads past the caches take two microseconds: all of them go out together, the first ones of the sums even before
        // the weights are known.  Sums: four columns a thread; with few rows the parts are dealt to `sides` groups of
        // threads, TOGETHER parts a thread at a time.  (Indexes behind the last part read it again.)
        auto join_rows = [&](int q, auto together_tag, auto more_tag) __attribute__((always_inline)) {
          constexpr int kPieces = D / 4, kTogether = decltype(together_tag)::value, kMore = decltype(more_tag)::value;
          const int here = rows - 8 * q < 8 ? rows - 8 * q : 8, items = here * kPieces, sides = kThreads / items;
          const int x = (int)threadIdx.x % items, side = (int)threadIdx.x / items, r8 = x / kPieces, col = 4 * (x % kPieces);
          f32x4 part[kTogether];
          auto fetch = [&](uint32_t i0) __attribute__((always_inline)) {
#pragma unroll
            for (int k = 0; k < kTogether; ++k) {
              const uint32_t i = i0 + (uint32_t)(k * sides);
              part[k] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                                      part_o, (row_of(i < parts ? i : parts - 1, 8 * q + r8) * D + (uint32_t)col) * 4u, 0, kThrough));
            }
          };
          fetch((uint32_t)side);
          // weights of the parts: 32 lanes for each of 8 rows
          const int row = threadIdx.x / 32, sub = threadIdx.x % 32;
          const bool there = 8 * q + row < rows;
          float m = kMinusInf, l = 0.f;
          for (uint32_t i0 = sub; i0 < parts; i0 += 32 * kMore) {
            u32x2 ml[kMore];
#pragma unroll
            for (int k = 0; k < kMore; ++k) {
              const uint32_t i = i0 + 32u * (uint32_t)k;
              ml[k] = __builtin_amdgcn_raw_buffer_load_b64(part_ml, row_of(i < parts ? i : parts - 1, there ? 8 * q + row : 8 * q) * 8u, 0, kThrough);
            }
#pragma unroll
            for (int k = 0; k < kMore; ++k) {
              const uint32_t i = i0 + 32u * (uint32_t)k;
              if (i < parts) {
                const float mi = __uint_as_float(ml[k][0]), m_new = fmaxf(m, mi), ref = m_new == kMinusInf ? 0.f : m_new;
                sh[row * kMostWorkgroups + i] = mi;
                l = l * __builtin_amdgcn_exp2f(m - ref) + __uint_as_float(ml[k][1]) * __builtin_amdgcn_exp2f(mi - ref);
                m = m_new;
              }
            }
          }
          float top = m;
#pragma unroll
          for (int s = 1; s < 32; s <<= 1) top = fmaxf(top, __shfl_xor(top, s));
          const float ref = top == kMinusInf ? 0.f : top;
          l *= __builtin_amdgcn_exp2f(m - ref);
#pragma unroll
          for (int s = 1; s < 32; s <<= 1) l += __shfl_xor(l, s);
          for (uint32_t i = sub; i < parts; i += 32) sh[row * kMostWorkgroups + i] = __builtin_amdgcn_exp2f(sh[row * kMostWorkgroups + i] - ref);
          if (there && sub == 0) {
            sh_l[row] = l;
            if (p.lse) {
              p.lse[(int64_t)b * p.kv_heads * p.group + kvh * p.group + row0 + 8 * q + row] =
                  l == 0.f ? kMinusInf : (top + log2f(l)) * 0.693147180559945309f;
            }
          }
          __syncthreads();
          f32x4 acc = {0.f, 0.f, 0.f, 0.f};
          for (uint32_t i0 = (uint32_t)side; i0 < parts;) {
#pragma unroll
            for (int k = 0; k < kTogether; ++k) {
              const uint32_t i = i0 + (uint32_t)(k * sides);
              if (i < parts) acc += sh[r8 * kMostWorkgroups + i] * part[k];
            }
            i0 += (uint32_t)(kTogether * sides);
            if (i0 < parts) fetch(i0);
          }
          sh_sum[threadIdx.x] = acc;
          __syncthreads();
          if (side == 0 && col < p.d) {
            for (int s = 1; s < sides; ++s) acc += sh_sum[s * items + x];
            const float inv = sh_l[r8] == 0.f ? 0.f : kLower / sh_l[r8], unit = sh_l[r8] == 0.f ? 0.f : vs;
            *(u32x2*)(p.o + (int64_t)b * p.o_batch + (int64_t)(kvh * p.group + row0 + 8 * q + r8) * p.o_head + col * 2) =
                u32x2{pack2<EK>(acc[0] * inv * unit, acc[1] * inv * unit), pack2<EK>(acc[2] * inv * unit, acc[3] * inv * unit)};
          }
          __syncthreads();
        };
#pragma unroll 1
        for (int q = 0; 8 * q < rows; ++q) {
          if (parts <= 8) {
            join_rows(q, std::integral_constant<int, 4>{}, std::integral_constant<int, 1>{});
          } else {
            join_rows(q, std::integral_constant<int, 16>{}, std::integral_constant<int, 4>{});
          }
        }
      }
    }

    // ---- the next triple of the line ---------------------------------------------------------------------
    r += u1 - u0;
    u0 = 0;
    if (++vh == vheads) {
      vh = 0;
      if (r < r_end) {
        ++b;
        len = (int32_t)uniform((uint32_t)length_of(p, b));
        units = units_of(len, kUnitKeys);
      }
    }
  }
#endif
}

}  // namespace paged
}  // namespace flash_hip
