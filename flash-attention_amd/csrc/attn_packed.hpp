// Attention over packed prompts: sequences of different lengths one behind the other, grouped heads, causal or not.
//
// Sequence b has queries cu_q[b] .. cu_q[b + 1] - 1 and keys cu_k[b] .. cu_k[b + 1] - 1; its query i sees key j when
// j <= i + (keys - queries), i.e. the last query sees the last key.  A query that sees no key gets zeros.
//
// The number of query tiles of a call is known to the device only; the grid holds total_q / rows and one or two for each
// sequence of them for every head, which is enough whatever the lengths are, and every wave finds its sequence by itself.
#pragma once

#include "attn_direct.hpp"
#include "serving_index.hpp"

namespace flash_hip {
namespace packed {

struct Params {
  const char* q;
  const char* k;
  const char* v;
  char* o;
  const int32_t* cu_q;
  const int32_t* cu_k;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, o_token, o_head;  // bytes
  int32_t sequences, total_q, total_k, heads, kv_heads, d;
  int32_t causal;
  uint32_t tiles;     // query tiles of the grid, per head
  uint32_t items;     // workgroups of the grid for one part of every item
  int32_t extra;      // tiles that a sequence may have beyond count / rows
  int32_t parts;      // most parts of an item (1: items are not cut)
  float* part_o;      // [items * parts][4 waves][query blocks][D / 16][64 lanes][4]
  float* part_ml;     // [items * parts][rows][2]
  uint32_t* tickets;  // [items]; zero, and left zero
  float scale_log2;   // softmax scale * log2 e
};

// A tile of query rows: its sequence's place in q and k, and its first row there
struct Tile {
  int32_t q0, nq, k0, nk, row;
  bool there;
};
// The tiles of all sequences in a row, `rows` query rows each; `extent(queries, keys)`: rows that those of a sequence
// cover together.  Every wave works this out for itself: up to 64 sequences by one scan.  More of them have tile numbers with
// gaps (first_tile), among which a search finds the sequence in two or three steps; numbers in a gap are workgroups that end
// at once.  (A scan over all sequences in every workgroup took 4096 prompts of 16 rows, 32 heads of 128, 11.7 ms where this takes 1.84.)
template <typename Extent>
struct TileLine {
  const Params& p;
  int32_t rows;
  int lane;
  const Extent& extent;

  struct Chunk {
    Range q, k;
    uint32_t own, sum;  // tiles of the lane's sequence, and of all sequences up to it
  };
  __device__ __forceinline__ Chunk chunk(int32_t b0) const {
    Chunk c{{0, 0}, {0, 0}, 0, 0};
    const int32_t b = b0 + lane;
    if (b < p.sequences) {
      c.q = sequence_rows(p.cu_q[b], p.cu_q[b + 1], p.total_q);
      c.k = sequence_rows(p.cu_k[b], p.cu_k[b + 1], p.total_k);
    }
    c.own = (uint32_t)((extent(c.q.count, c.k.count) + rows - 1) / rows);
    c.sum = direct::wave_scan(c.own);
    return c;
  }
  // `c`: the first chunk.  The number of tiles (of tile numbers, with many sequences), cut to the grid's (offsets that run
  // backwards could make more of them)
  __device__ __forceinline__ uint32_t length(const Chunk& c) const {
    const uint32_t n = (uint32_t)__builtin_amdgcn_readlane((int)c.sum, 63);
    return p.sequences <= 64 && n < p.tiles ? n : p.tiles;
  }
  __device__ __forceinline__ Tile tile(uint32_t at, Chunk c) const {
    uint32_t nth;  // of the sequence's tiles
    int l;         // lane that knows the sequence
    if (p.sequences <= 64) {
      const uint64_t past = __builtin_amdgcn_ballot_w64(c.sum > at);
      if (past == 0) return Tile{0, 0, 0, 0, 0, false};
      l = __builtin_ctzll(past);
      nth = at - (uint32_t)__builtin_amdgcn_readlane((int)(c.sum - c.own), l);
    } else {
      // the last sequence whose first number is not behind `at`, 64 probes a step
      int32_t b = 0;
      for (int32_t count = p.sequences; count > 1;) {
        const int32_t step = (count + 63) / 64, mine = lane * step;
        const bool before = mine < count && first_tile(p.cu_q[b + mine], p.total_q, (uint32_t)rows, (uint32_t)p.extra, b + mine) <= at;
        const uint64_t all = __builtin_amdgcn_ballot_w64(before);
        if (all == 0) return Tile{0, 0, 0, 0, 0, false};
        const int32_t skip = (63 - __builtin_clzll(all)) * step;
        b += skip;
        count = count - skip < step ? count - skip : step;
      }
      l = 0;
      const uint32_t first = first_tile(p.cu_q[b], p.total_q, (uint32_t)rows, (uint32_t)p.extra, b);
      c = chunk(b);
      nth = at - first;
      if (at < first || nth >= (uint32_t)__builtin_amdgcn_readlane((int)c.own, 0)) return Tile{0, 0, 0, 0, 0, false};
    }
    auto of = [&](int32_t x) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(x, l); };
    return Tile{of(c.q.start), of(c.q.count), of(c.k.start), of(c.k.count), (int32_t)nth * rows, true};
  }
};

// 16 query rows of one head by one wave, K and V straight from memory (attn_direct.hpp).  Rows outside the sequence
// (row0 may be negative) are left out.
template <int D, int EK, bool FULL>
__device__ __forceinline__ void attend_rows(const Params& p, const Tile& t, int32_t row0, int32_t head, int lane) {
  using namespace direct;
  using S = Step<D, EK, false, 1>;
  if (row0 >= t.nq || row0 + 15 < 0) return;
  const int n = lane & 15, g = lane >> 4;
  const int32_t kvh = head / (p.heads / p.kv_heads);
  const int32_t row = row0 + n;
  u32x4 qf[S::kKS];
  const bool mine = (uint32_t)row < (uint32_t)t.nq;
  const char* src = p.q + (int64_t)(t.q0 + (mine ? row : 0)) * p.q_token + (int64_t)head * p.q_head;
#pragma unroll
  for (int ks = 0; ks < S::kKS; ++ks) {
    const int col = S::column(ks, g);
    const bool there = mine && (FULL || col < p.d);
    const u32x4 x = *(const u32x4*)(src + (there ? col * 2 : 0));
    qf[ks] = there ? x : u32x4{0u, 0u, 0u, 0u};
  }
  // keys the lane's query sees, and those the last row of the 16 does
  const int32_t sees = visible_keys(row, t.nq, t.nk, p.causal);
  const int32_t end = visible_keys(row0 + 15 < t.nq ? row0 + 15 : t.nq - 1, t.nq, t.nk, p.causal);
  typename S::State st;
  S::clear(st);
  const char* kh = p.k + (int64_t)t.k0 * p.k_token + (int64_t)kvh * p.k_head;
  const char* vh = p.v + (int64_t)t.k0 * p.v_token + (int64_t)kvh * p.v_head;
  for (int32_t key0 = 0; key0 < end; key0 += S::kKeys) {
    typename S::KBlock k;
    typename S::VBlock v;
    const uint64_t valid = end - key0 >= S::kKeys ? 0xffffffffull : (1ull << (end - key0)) - 1;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int32_t key = key0 + 16 * i + n;
      const char* a = kh + (int64_t)(key < end ? key : key0) * p.k_token;
#pragma unroll
      for (int x = 0; x < S::kKLoads; ++x) {
        const int col = S::load_column(x, g);
        const bool in = FULL || col < p.d;
        k[i][x] = *(const u32x4*)(a + (in ? col * 2 : 0));
        if (!in) k[i][x] = u32x4{0u, 0u, 0u, 0u};
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int32_t key = key0 + S::v_key(0, g, j);
      const bool in = FULL || n * S::kE < p.d;
      v[0][j] = *(const typename S::VWord*)(vh + (int64_t)(key < end ? key : key0) * p.v_token + (in ? n * S::kE * 2 : 0));
    }
    S::clear_missing(v, valid, lane);
    typename S::Weights w;
    S::template weigh<true>(st, w, k, qf, valid, p.scale_log2, lane, sees - key0);
    S::accumulate_limited(st, w, v, lane, sees - key0);
  }
  const float l = quad_sum(st.l);
  const float inv = l == 0.f ? 0.f : 1.f / kRaise<EK> / l;
  if (!mine) return;
  char* dst = p.o + (int64_t)(t.q0 + row) * p.o_token + (int64_t)head * p.o_head;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int col = S::kE * (4 * g + i);
    if (FULL || col < p.d) {
      typename S::VWord w;
      if constexpr (S::kE == 8) {
        w = u32x4{pack2<EK>(st.o[0][i] * inv, st.o[1][i] * inv), pack2<EK>(st.o[2][i] * inv, st.o[3][i] * inv),
                  pack2<EK>(st.o[4][i] * inv, st.o[5][i] * inv), pack2<EK>(st.o[6][i] * inv, st.o[7][i] * inv)};
      } else {
        w = u32x2{pack2<EK>(st.o[0][i] * inv, st.o[1][i] * inv), pack2<EK>(st.o[2][i] * inv, st.o[3][i] * inv)};
      }
      *(typename S::VWord*)(dst + col * 2) = w;
    }
  }
}

}  // namespace packed

// the pipelined kernel (flash_packed.hip): whether it takes a call, the workspace with which it can cut items (0: it would
// not), and its launch
__attribute__((visibility("hidden"))) bool packed_mfma_takes(const packed::Params& p);
__attribute__((visibility("hidden"))) int64_t packed_mfma_workspace(const packed::Params& p);
__attribute__((visibility("hidden"))) int launch_packed_mfma(const packed::Params& p, bool bf16, void* workspace, hipStream_t stream);

namespace packed {

constexpr int kDirectRows = 64;  // 4 waves x 16

template <int D, int EK, bool FULL>
__global__ __launch_bounds__(256) void packed_direct_kernel(const Params p) {
#if defined(__HIP_DEVICE_COMPILE__)
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  auto extent = [](int32_t nq, int32_t) { return nq; };
  const TileLine<decltype(extent)> line{p, kDirectRows, lane, extent};
  const Tile t = line.tile(blockIdx.x, line.chunk(0));
  const int32_t row0 = t.row + wave * 16;
  if (!t.there || row0 >= t.nq) return;
  attend_rows<D, EK, FULL>(p, t, row0, (int32_t)blockIdx.y, lane);
#endif
}

}  // namespace packed
}  // namespace flash_hip
