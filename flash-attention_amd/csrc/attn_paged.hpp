// Attention of one new token of every sequence over a paged key-value cache, split over the cache's length, and
// the join of the parts.  What a wave does with its keys is in attn_direct.hpp.
//
// What bounds it: the cache is read once, 2 * d * (bytes of an element) per key and K/V head, against
// 4 * d * (heads per K/V head) operations: at 8 query heads per K/V head and 16-bit values 16 operations a
// byte, two orders of magnitude below what the matrix cores could do in that time.  The kernel is made to keep
// loads in flight.
//
// Work split.  Sequence b of length n_b is cut into U_b = max(1, ceil(n_b / kUnit)) units; all units of all
// (sequence, K/V head, query block) triples stand in one line, b outermost, and workgroup w takes the units
// [w c, (w + 1) c) of it, c = ceil(total / workgroups).  Every workgroup then reads the same number of keys
// whatever the lengths are, and nothing about them has to be known on the host, so that a captured graph stays
// valid while they grow.  Every wave finds the line's length and the workgroup's place in it from the lengths
// themselves (a scan over 64 of them per step).  A workgroup that holds all units of a triple writes its output;
// otherwise it leaves (o, m, l) in the workspace and join_parts_kernel adds the parts up, in the line's order, so
// that the result does not depend on timing.
#pragma once

#include "attn_direct.hpp"
#include "serving_index.hpp"

#ifndef FLASH_DW
#define FLASH_DW 2
#endif
namespace flash_hip {
namespace paged {

using namespace direct;

constexpr int kThreads = 256;
constexpr int kWaves = 4;

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
  float* part_o;         // [2 * workgroups][rows][D]
  float* part_ml;        // [2 * workgroups][rows][2]
  int64_t q_batch, q_head, o_batch, o_head;     // bytes
  Pages pages;                                   // K and V alike
  int64_t head_stride;                           // bytes
  int64_t table_stride;                          // entries
  int32_t batch, kv_heads, group;                // group: query heads per K/V head
  int32_t d;
  int32_t qblocks;                               // blocks of 16 * NQ query heads per K/V head
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

// units of all sequences, and of those before sequence `upto`
struct Line {
  uint32_t total, before;
};
__device__ __forceinline__ Line measure_line(const Params& p, int32_t unit, int32_t upto, int lane) {
  Line r{0, 0};
  for (int32_t b0 = 0; b0 < p.batch; b0 += 64) {
    const int32_t b = b0 + lane;
    const uint32_t u = b < p.batch ? units_of(length_of(p, b), unit) : 0u;
    const uint32_t sum = wave_scan(u);
    if (upto >= b0 && upto < b0 + 64) r.before = r.total + uniform((uint32_t)__shfl((int)(sum - u), upto - b0));
    r.total += uniform((uint32_t)__shfl((int)sum, 63));
  }
  return r;
}

template <int D, int EK, bool CACHE8, int NQ, bool FULL, bool PAGE16>
__global__ __launch_bounds__(kThreads, FLASH_DW) void decode_kernel(const Params p) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int NS = kSub<D, CACHE8>;
  constexpr int kUnitKeys = kUnit<D, CACHE8>;
  using S = Step<D, EK, CACHE8, NS, NQ>;
  constexpr int kRowFloats = D + 4;  // rows of the join buffer, shifted by four banks each
  __shared__ __attribute__((aligned(16))) float sh_o[kWaves][16][kRowFloats];
  __shared__ float sh_ml[kWaves][NQ * 16][2];

  const int lane = threadIdx.x & 63;
  const int wave = (int)uniform(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;

  // ---- this workgroup's piece of the line -------------------------------------------------------------
  const uint32_t vheads = (uint32_t)(p.kv_heads * p.qblocks);
  const uint32_t total = measure_line(p, kUnitKeys, -1, lane).total * vheads;
  const uint32_t c = units_each(total, p.workgroups);
  const uint32_t r_begin = blockIdx.x * c;
  if (r_begin >= total) return;
  const uint32_t r_end = r_begin + c < total ? r_begin + c : total;
  int32_t b = 0;
  uint32_t first = 0;  // units of the line before sequence b
  for (int32_t b0 = 0; b0 < p.batch; b0 += 64) {
    const uint32_t u = b0 + lane < p.batch ? units_of(length_of(p, b0 + lane), kUnitKeys) * vheads : 0u;
    const uint32_t sum = wave_scan(u);
    const uint64_t past = __builtin_amdgcn_ballot_w64(first + sum > r_begin);
    if (past != 0) {
      const int at = __builtin_ctzll(past);
      b = b0 + at;
      first += uniform((uint32_t)__shfl((int)(sum - u), at));
      break;
    }
    first += uniform((uint32_t)__shfl((int)sum, 63));
  }
  int32_t len = (int32_t)uniform((uint32_t)length_of(p, b));
  uint32_t units = units_of(len, kUnitKeys);
  uint32_t vh = (r_begin - first) / units;
  uint32_t u0 = (r_begin - first) - vh * units;

  for (uint32_t r = r_begin; r < r_end;) {
    const uint32_t left = r_end - r;
    const uint32_t u1 = units - u0 < left ? units : u0 + left;
    const int32_t kvh = (int32_t)(vh / (uint32_t)p.qblocks), qb = (int32_t)(vh - (uint32_t)(kvh * p.qblocks));
    const int32_t row0 = qb * (16 * NQ);                                // first query head inside the group
    const int32_t rows = p.group - row0 < 16 * NQ ? p.group - row0 : 16 * NQ;

    // queries of the block, zeros for the heads that do not exist
    u32x4 qf[NQ][S::kKS];
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      const int row = 16 * q + n;
      const char* src = p.q + (int64_t)b * p.q_batch + (int64_t)(kvh * p.group + row0 + (row < rows ? row : 0)) * p.q_head;
#pragma unroll
      for (int ks = 0; ks < S::kKS; ++ks) {
        const int col = S::column(ks, g);
        const bool there = row < rows && (FULL || col < p.d);
        const u32x4 x = *(const u32x4*)(src + (there ? col * 2 : 0));
        qf[q][ks] = there ? x : u32x4{0u, 0u, 0u, 0u};
      }
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
    auto load_k = [&](typename S::KBlock& k, int64_t at) __attribute__((always_inline)) {
#pragma unroll
      for (int t = 0; t < 2 * NS; ++t) {
        const char* src = PAGE16 ? kh + tile_start(at, t) : kh + __shfl(at, 16 * t + n);
        const uint32_t row = PAGE16 ? (uint32_t)n * slot_stride : 0u;
#pragma unroll
        for (int i = 0; i < S::kKLoads; ++i) {
          const int col = S::load_column(i, g);
          const bool in = FULL || col < p.d;
          k[t][i] = *(const u32x4*)(src + (row + (uint32_t)((in ? col : 0) * S::kElem)));
          if constexpr (!FULL) {
            // (an 8-bit load holds 16 columns, of which the last 8 may lie behind the row)
            if (!in) k[t][i] = u32x4{0u, 0u, 0u, 0u};
            if constexpr (CACHE8) {
              if (in && col + 8 >= p.d) k[t][i][2] = k[t][i][3] = 0u;
            }
          }
        }
      }
    };
    auto load_v = [&](typename S::VBlock& v, int64_t at) __attribute__((always_inline)) {
      const bool in = FULL || n * S::kE < p.d;
      const uint32_t col = (uint32_t)(in ? n * S::kE * S::kElem : 0);
#pragma unroll
      for (int s = 0; s < NS; ++s) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if constexpr (PAGE16) {
            const uint32_t row = (uint32_t)(4 * g + j % 4) * slot_stride;
            v[s][j] = *(const typename S::VWord*)(vv + tile_start(at, 2 * s + j / 4) + (row + col));
          } else {
            v[s][j] = *(const typename S::VWord*)(vv + __shfl(at, S::v_key(s, g, j)) + col);
          }
        }
      }
    };

    // K is fetched a step ahead, V at the step's beginning: 16 KB in flight per wave at any time at d = 128
    typename S::State st;
    auto attend = [&](auto careful) __attribute__((always_inline)) {
      S::clear(st);
      typename S::KBlock k, k_next;
      int64_t at, at_next;
      uint64_t valid = place(u0, page_of(u0), at), valid_next;
      int32_t page = page_of(u0 + 1);
      load_k(k, at);
      for (uint32_t u = u0; u < u1; ++u) {
        typename S::VBlock v;
        load_v(v, at);
        const bool more = u + 1 < u1;
        if (more) {
          valid_next = place(u + 1, page, at_next);
          load_k(k_next, at_next);
          page = page_of(u + 2);
        }
        if (valid != 0) {
          typename S::Weights w;
          S::template weigh<false>(st, w, k, qf, valid, sc, lane);
          S::clear_missing(v, valid, lane);
          S::template accumulate<decltype(careful)::value>(st, w, v);
        }
        if (more) {
#pragma unroll
          for (int t = 0; t < 2 * NS; ++t) {
#pragma unroll
            for (int i = 0; i < S::kKLoads; ++i) k[t][i] = k_next[t][i];
          }
          at = at_next;
          valid = valid_next;
        }
      }
    };
    attend(std::false_type{});
    // NaN may come from an infinite value (rare: the part is worked out again with care)
    if (S::holds_nan(st)) attend(std::true_type{});

    // ---- the four waves' parts, 16 queries at a time -----------------------------------------------------
    const bool complete = u0 == 0 && u1 == units;
    const uint32_t slot = part_slot(blockIdx.x, c, r - u0);
    const float vs = CACHE8 && p.v_scale ? p.v_scale[kvh] : 1.f;
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      const float l = quad_sum(st.l[q]);
      if (g == 0) {
        sh_ml[wave][16 * q + n][0] = st.m[q];
        sh_ml[wave][16 * q + n][1] = l;
      }
    }
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int e = 0; e < S::kE; e += 4) {
          *(f32x4*)&sh_o[wave][n][S::kE * (4 * g + i) + e] =
              f32x4{st.o[q][e][i], st.o[q][e + 1][i], st.o[q][e + 2][i], st.o[q][e + 3][i]};
        }
      }
      __syncthreads();
      constexpr int kPieces = D / 4;
      for (int x = threadIdx.x; x < 16 * kPieces; x += kThreads) {
        const int row = x / kPieces, col = 4 * (x % kPieces);
        if (16 * q + row < rows && col < p.d) {
          float m = kMinusInf;
#pragma unroll
          for (int w = 0; w < kWaves; ++w) m = fmaxf(m, sh_ml[w][16 * q + row][0]);
          const float ref = m == kMinusInf ? 0.f : m;
          f32x4 sum = {0.f, 0.f, 0.f, 0.f};
          float l = 0.f;
#pragma unroll
          for (int w = 0; w < kWaves; ++w) {
            const float f = __builtin_amdgcn_exp2f(sh_ml[w][16 * q + row][0] - ref);
            l += f * sh_ml[w][16 * q + row][1];
            sum += f * *(const f32x4*)&sh_o[w][row][col];
          }
          if (complete) {
            const int32_t head = kvh * p.group + row0 + 16 * q + row;
            const float inv = l == 0.f ? 0.f : vs / l;
            *(u32x2*)(p.o + (int64_t)b * p.o_batch + (int64_t)head * p.o_head + col * 2) =
                u32x2{pack2<EK>(sum[0] * inv, sum[1] * inv), pack2<EK>(sum[2] * inv, sum[3] * inv)};
            if (p.lse && col == 0) {
              p.lse[(int64_t)b * p.kv_heads * p.group + head] = l == 0.f ? kMinusInf : (m + log2f(l)) * 0.693147180559945309f;
            }
          } else {
            const uint64_t at = (uint64_t)slot * (16 * NQ) + (uint32_t)(16 * q + row);
            *(f32x4*)(p.part_o + at * D + col) = sum;
            if (col == 0) *(f32x2*)(p.part_ml + at * 2) = f32x2{m, l};
          }
        }
      }
      __syncthreads();
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

// One workgroup per sequence and query head: the parts of its triple, if there are several, in the line's order.
// 32 lanes (16 at D = 64) hold a row, the others other parts of it.
template <int D, int EK, bool CACHE8, int NQ>
__global__ __launch_bounds__(kThreads) void join_parts_kernel(const Params p) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int kPieces = D / 4, kSides = kThreads / kPieces;
  __shared__ __attribute__((aligned(16))) float sh_o[kSides][D];
  __shared__ float sh_ml[kSides][2];
  const int lane = threadIdx.x & 63;
  const int32_t heads = p.kv_heads * p.group;
  const int32_t b = (int32_t)(blockIdx.x / (uint32_t)heads), head = (int32_t)blockIdx.x - b * heads;
  const int32_t kvh = head / p.group, in_group = head - kvh * p.group;
  const uint32_t vheads = (uint32_t)(p.kv_heads * p.qblocks);
  constexpr int kUnitKeys = kUnit<D, CACHE8>;
  const Line line = measure_line(p, kUnitKeys, b, lane);
  const uint32_t units = units_of((int32_t)uniform((uint32_t)length_of(p, b)), kUnitKeys);
  const uint32_t c = units_each(line.total * vheads, p.workgroups);
  const uint32_t start = line.before * vheads + (uint32_t)(kvh * p.qblocks + in_group / (16 * NQ)) * units;
  const uint32_t w0 = start / c, w1 = (start + units - 1) / c;
  if (w0 == w1) return;  // one workgroup had it all and wrote the output
  const int side = threadIdx.x / kPieces, col = 4 * (threadIdx.x % kPieces);
  float m = kMinusInf, l = 0.f;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  for (uint32_t w = w0 + (uint32_t)side; w <= w1; w += kSides) {
    const uint32_t slot = part_slot(w, c, start);
    const uint64_t at = (uint64_t)slot * (16 * NQ) + (uint32_t)(in_group % (16 * NQ));
    const f32x2 ml = *(const f32x2*)(p.part_ml + at * 2);
    const f32x4 x = col < p.d ? *(const f32x4*)(p.part_o + at * D + col) : f32x4{0.f, 0.f, 0.f, 0.f};
    const float m_new = fmaxf(m, ml[0]), ref = m_new == kMinusInf ? 0.f : m_new;
    const float keep = __builtin_amdgcn_exp2f(m - ref), add = __builtin_amdgcn_exp2f(ml[0] - ref);
    sum = sum * keep + x * add;
    l = l * keep + ml[1] * add;
    m = m_new;
  }
  *(f32x4*)&sh_o[side][col] = sum;
  if (col == 0) {
    sh_ml[side][0] = m;
    sh_ml[side][1] = l;
  }
  __syncthreads();
  if (side == 0 && col < p.d) {
#pragma unroll
    for (int s = 1; s < kSides; ++s) m = fmaxf(m, sh_ml[s][0]);
    const float ref = m == kMinusInf ? 0.f : m;
    l = 0.f;
    sum = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < kSides; ++s) {
      const float f = __builtin_amdgcn_exp2f(sh_ml[s][0] - ref);
      l += f * sh_ml[s][1];
      sum += f * *(const f32x4*)&sh_o[s][col];
    }
    const float inv = l == 0.f ? 0.f : (CACHE8 && p.v_scale ? p.v_scale[kvh] : 1.f) / l;
    *(u32x2*)(p.o + (int64_t)b * p.o_batch + (int64_t)head * p.o_head + col * 2) =
        u32x2{pack2<EK>(sum[0] * inv, sum[1] * inv), pack2<EK>(sum[2] * inv, sum[3] * inv)};
    if (p.lse && col == 0) p.lse[(int64_t)b * heads + head] = l == 0.f ? kMinusInf : (m + log2f(l)) * 0.693147180559945309f;
  }
#endif
}

}  // namespace paged
}  // namespace flash_hip
