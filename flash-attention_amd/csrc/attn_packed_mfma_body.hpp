// The pipelined kernel for packed prompts, once per wave layout: included by attn_packed_mfma.hpp with FLASH_M16_NS set to
// the layout's namespace (see there).
//
// Rings.  Tile t's K (64 keys) lies in slot (t + lead) % 3 of the K ring, block b of V (32 keys) in slot (b + 2 lead) %
// kVBlocks of the V ring.  Iteration t multiplies V blocks 2t - 1 and 2t and reads K up to the start of block 2t + 3; it
// fetches V blocks 2t + 1 and 2t + 2 and K tile t + 2.  Four V blocks are enough for that; `lead` makes the end of an item
// (its diagonal) begin in slot 0, so that every slot is a constant of the code.

namespace flash_hip {
namespace FLASH_M16_NS {

constexpr int kPackedRows = 64 * kQ16;
constexpr int kVBlocks = FLASH_PACKED_V_BLOCKS;
constexpr int kPeriod = kVBlocks == 4 ? 6 : 3;  // tiles after which both rings are where they were
template <int D>
constexpr int kPackedLds = kRing * Cfg<D>::kTileBytes + kVBlocks * Cfg<D>::kBlkBytes;

// How far (in exp2 units) a row's largest weight stands above 1 when its reference moves.  fp16 has no bits below 2^-24, and
// a long tail behind one leading key consists of small weights: they are raised by 2^7, which with the 2^8 that the
// reference may lag behind stays below 65504 and keeps weights down to 2^-31 of the largest.  (bfloat16 reaches as
// far down as fp32.)  Where |reference| is so large that fp32 has no room for the lift, rounding makes it up to twice
// as much or nothing: below 2^15 all the same.
template <int EK>
constexpr float kLift = EK == kF16 ? 7.f : 0.f;
template <int EK>
constexpr float kLiftOfThreshold = kLift<EK> / (kDeferLog2 + kLift<EK>);

// A tile iteration: tile t with (t + lead) % kPeriod = SLOT.  Q0 is the first query block that sees tile t, QK_B the first
// one that sees tile t + 1, PV_A the first one that saw tile t - 1; MASK_A and MASK_B the block whose scores of tile t
// (second half) and tile t + 1 (first half) are masked; QK_NEXT: there is a tile t + 1, STAGE_K: a tile t + 2.
constexpr int kNoMask = -1, kMaskAll = -2;
template <int SLOT_, int Q0_, int QK_B_, int PV_A_, int MASK_A_, int MASK_B_, bool STAGE_K_, bool QK_NEXT_>
struct TilePlan {
  static constexpr int SLOT = SLOT_, Q0 = Q0_, QK_B = QK_B_, PV_A = PV_A_, MASK_A = MASK_A_, MASK_B = MASK_B_;
  static constexpr bool STAGE_K = STAGE_K_, QK_NEXT = QK_NEXT_;
};
// tile T of the diagonal
template <int T>
using DiagonalPlan = TilePlan<T % kPeriod, T, (T + 1 < kQ16 ? T + 1 : T), (T > 0 ? T - 1 : 0), T, (T + 1 < kQ16 ? T + 1 : kNoMask), (T + 2 < kQ16),
                              (T + 1 < kQ16)>;

// A part of an item: the tiles [first, behind) of its keys.  SPLIT kernels cut items with many tiles where there are too few
// of them to fill the chip: every part leaves its sums, and the last one to do so adds them up, in their order.  A part's
// start, end and join cost about as much as 10 tiles: 64 rows of 32 heads over 2048 keys take 26 us with parts of 8 tiles and
// more, 31 with 12, 34 uncut; but a whole prompt of 2048 rows, 8 heads, 35, 31.5 and 34; and of 8 x 1024 17.6, 15.9 and 15.1.
constexpr int kMostParts = 16, kPartTiles = 12;  // parts of an item at most, tiles of a part at least
struct Part {
  int parts, first, behind;
};
// Item of workgroup `place` of those that work on part `nth` (workgroup i runs on XCD i % 8, and there are a multiple of 8
// items): the parts of an item go to different XCDs.
__device__ __forceinline__ uint32_t item_of_part(uint32_t place, uint32_t nth) { return place ^ (nth & 7u); }
template <int D, typename TO, bool CAUSAL, bool SPLIT>
__device__ __forceinline__ bool packed_item(const packed::Params& p, packed::Item item, const Part& part, char* smem_raw);

template <int D, typename TO, bool CAUSAL, bool SPLIT>
__global__ __launch_bounds__(kThreads, kQ16 == 2 ? 2 : 1) void attn_fwd_kernel_packed(const packed::Params p) {
#if defined(__HIP_DEVICE_COMPILE__)
  extern __shared__ __attribute__((aligned(16))) char smem_raw[];
  bool again;
  {
    Part part{1, 0, 0};
    const uint32_t nth = SPLIT ? blockIdx.x / p.items : 0;  // number of the part
    const packed::Item item = packed::find_item(p, SPLIT ? item_of_part(blockIdx.x - nth * p.items, nth) : blockIdx.x, kPackedRows, CAUSAL, (int)(threadIdx.x & 63));
    if (!item.it.there) return;
    // rows that see no key: at most the first ones of a sequence with more queries than keys
    again = item.it.nk == 0 || item.a0 < 0;
    if (!again) {
      part.behind = CAUSAL ? item.a0 / kBc + kQ16 : (item.it.nk - 1) / kBc + 1;  // tiles of the item
      if constexpr (SPLIT) {
        const int tiles = part.behind, wanted = tiles / kPartTiles;
        part.parts = wanted < 1 ? 1 : (wanted < p.parts ? wanted : p.parts);
        if ((int)nth >= part.parts) return;
        part.first = (int)nth * tiles / part.parts;
        part.behind = ((int)nth + 1) * tiles / part.parts;
      }
      again = packed_item<D, TO, CAUSAL, SPLIT>(p, item, part, smem_raw);
    } else if (nth > 0) {
      return;
    }
  }
  if (again) {
    // (rare: the arguments are read again here, rather than kept in registers all the while)
    const packed::Params* late = (const packed::Params*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(late));
    int lane = (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
    asm volatile("" : "+v"(lane));
    const packed::Item item = packed::find_item(*late, SPLIT ? item_of_part(blockIdx.x % late->items, blockIdx.x / late->items) : blockIdx.x, kPackedRows, CAUSAL, lane);
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
#pragma unroll 1
    for (int q = 0; q < kQ16; ++q) {
      packed::attend_rows<D, kElemKindOf<TO> == kBF16 ? direct::kBfloat : direct::kHalf, false>(*late, item.it, item.row0 + 64 * q + 16 * wave,
                                                                                                item.head, lane);
    }
  }
#endif
}

// The item, or a part of it, on the pipelined body.  True: this wave's rows hold NaN or infinities and so do the values of
// its diagonal.
template <int D, typename TO, bool CAUSAL, bool SPLIT>
__device__ __forceinline__ bool packed_item(const packed::Params& p, packed::Item item, const Part& part, char* smem_raw) {
#if defined(__HIP_DEVICE_COMPILE__)
  using C = Cfg<D>;
  constexpr int EK = kElemKindOf<TO>;
  constexpr int kKS = C::kKS, kDv16 = C::kDv16, kTileBytes = C::kTileBytes, kBlkBytes = C::kBlkBytes;
  constexpr int kPiecesPerWave = C::kPiecesPerWave;
  lds_char* const smem = (lds_char*)smem_raw;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n16 = lane & 15;
  const int g = lane >> 4;
  const int d = p.d;
  if constexpr (SPLIT) {
    // the keys in front of the part are not there for anything below
    item.it.k0 += part.first * kBc;
    item.it.nk -= part.first * kBc;
    item.a0 -= part.first * kBc;
  }
  const packed::Tile& it = item.it;
  const int32_t head = item.head, kvh = item.kvh, row0 = item.row0, a0 = item.a0;
  const int32_t seen = CAUSAL ? a0 - row0 : 0;  // keys that a row sees, less its number and one
  // Tiles in front of the end: the diagonal's kQ16 (rows that do not exist make some of them idle), or the last one,
  // which may be partly there
  const int full = SPLIT ? part.behind - part.first - (CAUSAL ? kQ16 : 1) : (CAUSAL ? a0 / kBc : (it.nk - 1) / kBc);
  const int lead = (kPeriod - full % kPeriod) % kPeriod;
  // (finite: a scale below 1e-37 must not make the lift infinite)
  const ScaleSplit sc{p.scale_log2, fminf((kDeferLog2 + kLift<EK>) / p.scale_log2, 3e38f)};

  const char* const qb = p.q + ((int64_t)it.q0 + row0) * p.q_token + (int64_t)head * p.q_head;
  char* const ob = p.o + ((int64_t)it.q0 + row0) * p.o_token + (int64_t)head * p.o_head;
  const char* const kb = p.k + (int64_t)it.k0 * p.k_token + (int64_t)kvh * p.k_head;
  const char* const vb = p.v + (int64_t)it.k0 * p.v_token + (int64_t)kvh * p.v_head;
  const uint32_t q_row = (uint32_t)p.q_token, o_row = (uint32_t)p.o_token;
  const uint32_t k_row = (uint32_t)p.k_token, v_row = (uint32_t)p.v_token;
  // (offsets beyond the item's rows are kOob; the launcher sees to it that kOob lies behind them)
  const __amdgpu_buffer_rsrc_t q_rs = __builtin_amdgcn_make_buffer_rsrc((void*)qb, 0, kOob, 0x00020000);
  const __amdgpu_buffer_rsrc_t o_rs = __builtin_amdgcn_make_buffer_rsrc((void*)ob, 0, kOob, 0x00020000);

  lds_char* const k_ring = smem;
  lds_char* const v_ring = smem + kRing * kTileBytes;

  // staging: as in attn_fwd_kernel_m16; a descriptor covers the rows of one tile that exist, so that rows behind the
  // sequence read as zeros and 32 bits suffice at every length
  uint32_t k_off[kPiecesPerWave], v_off[kPiecesPerWave];
#pragma unroll
  for (int i = 0; i < kPiecesPerWave; ++i) {
    const int ci = (wave * kPiecesPerWave + i) * 64 + lane;
    const int row = ci / C::kChunks;
    const int src = (ci % C::kChunks) ^ swz<D>(row);
    k_off[i] = (src * 8 < d) ? (uint32_t)row * k_row + (uint32_t)src * 16u : kOob;
    v_off[i] = (src * 8 < d) ? (uint32_t)row * v_row + (uint32_t)src * 16u : kOob;
  }
  // (base and size of what exists of `rows` rows from row `first` on)
  auto rows_srd = [&](const char* base, uint32_t row_bytes, int first, int rows) __attribute__((always_inline)) {
    const int left = it.nk - first, n = left < rows ? left : rows;
    return make_srd(base + (int64_t)first * row_bytes, n > 0 ? (uint32_t)(n - 1) * row_bytes + (uint32_t)d * 2u : 0u);
  };
  // piece i of this wave: 1 KiB of the tile, or of the pair of V blocks (the waves of each half of the workgroup have one)
  const int half = wave / (kWaves / 2);
  auto k_piece = [&](const srd_t srd, int slot, int i) __attribute__((always_inline)) {
    const uint32_t lds_base = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(k_ring + slot * kTileBytes + (wave * kPiecesPerWave + i) * 1024));
    dma_piece(srd, k_off[i], lds_base);
  };
  auto v_piece = [&](const srd_t srd, int slot0, int slot1, int i) __attribute__((always_inline)) {
    const uint32_t lds_base = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(
        v_ring + (half ? slot1 : slot0) * kBlkBytes + ((wave - half * (kWaves / 2)) * kPiecesPerWave + i) * 1024));
    dma_piece(srd, v_off[i], lds_base);
  };
  auto staged_barrier = [&]() __attribute__((always_inline)) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  };

  // ---- Q fragments ------------------------------------------------------------------------------------------
  f16x8 qf[kQ16][kKS];
  const int row_n = row0 + 16 * wave + n16;  // the lane's row in query block 0
#pragma unroll
  for (int q = 0; q < kQ16; ++q) {
    const bool there = (uint32_t)(row_n + 64 * q) < (uint32_t)it.nq;
#pragma unroll
    for (int ks = 0; ks < kKS; ++ks) {
      const int col = 8 * (ks + kKS * g);
      const uint32_t off = (there && col < d) ? (uint32_t)(64 * q + 16 * wave + n16) * q_row + (uint32_t)col * 2u : kOob;
      qf[q][ks] = __builtin_bit_cast(f16x8, __builtin_amdgcn_raw_buffer_load_b128(q_rs, off, 0, 0));
    }
  }
  {
    // K tiles 0 and 1, and V block 0 as the second one of the pair (-1, 0)
    srd_t k0_srd = rows_srd(kb, k_row, 0, kBc), v0_srd = rows_srd(vb, v_row, 0, kBc / 2);
    const int v_slot = 2 * lead % kVBlocks;
    settle_scalars(k0_srd, v0_srd);
#pragma unroll
    for (int i = 0; i < kPiecesPerWave; ++i) k_piece(k0_srd, lead % 3, i);
    if (half) {
#pragma unroll
      for (int i = 0; i < kPiecesPerWave; ++i) {
        const uint32_t lds_base = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(
            v_ring + v_slot * kBlkBytes + ((wave - kWaves / 2) * kPiecesPerWave + i) * 1024));
        dma_piece(v0_srd, v_off[i] == kOob ? kOob : v_off[i] - (uint32_t)(kBc / 2) * v_row, lds_base);
      }
    }
    srd_t k1_srd = rows_srd(kb, k_row, kBc, kBc);
    settle_scalars(k1_srd);
#pragma unroll
    for (int i = 0; i < kPiecesPerWave; ++i) k_piece(k1_srd, (lead + 1) % 3, i);
    // step 0 multiplies P(-1) = 0 with V block -1: make that finite
    for (int i = tid * 16; i < kBlkBytes; i += kThreads * 16) {
      *FLASH_LDS_CAST(u32x4, v_ring + (v_slot == 0 ? kVBlocks - 1 : v_slot - 1) * kBlkBytes + i) = u32x4{0u, 0u, 0u, 0u};
    }
  }
  f32x4 o[kQ16][kDv16];
#pragma unroll
  for (int q = 0; q < kQ16; ++q) {
#pragma unroll
    for (int ks = 0; ks < kKS; ++ks) asm volatile("" : "+a"(qf[q][ks]));
#pragma unroll
    for (int b = 0; b < kDv16; ++b) {
#pragma unroll
      for (int i = 0; i < 4; ++i) o[q][b][i] = 0.f;
      asm volatile("" : "+a"(o[q][b]));
    }
  }
  const LaneAddr<D> la = make_lane_addr<D>(lane, k_ring, v_ring);
  const QueryLimit limit_causal{row_n + seen + 1};
  const auto limit = [&]() __attribute__((always_inline)) {
    if constexpr (CAUSAL) return limit_causal; else return (int)it.nk;
  }();

  staged_barrier();

  // ---- prologue: S(0), its row maximum, the first K fragments of block 1 -------------------------------------
  f32x4 sA[2][kQ16], sB[2][kQ16];
  f16x8 pA[kQ16], pB[kQ16];
  f16x8 ka[4];
#pragma unroll
  for (int q = 0; q < kQ16; ++q) {
#pragma unroll
    for (int j = 0; j < 8; ++j) pB[q][j] = (f16)0.f;
    asm volatile("" : "+v"(pB[q]));
  }
  const uint32_t k_first = (uint32_t)(lead % 3 * kTileBytes);
#pragma unroll
  for (int f = 0; f < 4; ++f) ka[f] = read_k<D>(k_first, la, f / kKS, f % kKS);
#pragma unroll
  for (int f = 0; f < 2 * kKS; ++f) {
#pragma unroll
    for (int q = 0; q < kQ16; ++q) {
      if (f % kKS == 0) {
        mfma_s_first0<EK>(sA[f / kKS][q], ka[f % 4], qf[q][f % kKS]);
      } else {
        mfma_s<true, EK>(sA[f / kKS][q], ka[f % 4], qf[q][f % kKS]);
      }
    }
    if (f + 4 < 2 * kKS) {
      ka[f % 4] = read_k<D>(k_first, la, (f + 4) / kKS, (f + 4) % kKS);
    } else {
      ka[f % 4] = read_k<D>(k_first + (uint32_t)kBlkBytes, la, (f + 4 - 2 * kKS) / kKS, (f + 4) % kKS);
    }
  }
  drain_s(sA);
  State st[kQ16];
  float mx_all = 0.f;
  uint64_t vote = 0;
  f32x4 bias[kQ16];
  f32x4 lsum[kQ16];
  uint64_t pending = 0;
#pragma unroll
  for (int q = 0; q < kQ16; ++q) {
    mask_tile(sA[0][q], 0, key_limit(limit, q), lane);
    mask_tile(sA[1][q], 16, key_limit(limit, q), lane);
    float mx = fmaxf(fmaxf(sA[0][q][0], sA[0][q][1]), fmaxf(sA[0][q][2], sA[0][q][3]));
    mx = fmaxf(mx, fmaxf(fmaxf(sA[1][q][0], sA[1][q][1]), fmaxf(sA[1][q][2], sA[1][q][3])));
    const float mc = quad_lane_max(mx, lane) - kLiftOfThreshold<EK> * sc.thr;  // every row sees key 0
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sA[0][q][i] -= mc;
      sA[1][q][i] -= mc;
      bias[q][i] = -mc;
    }
    st[q].mc = mc;
#pragma unroll
    for (int i = 0; i < 4; ++i) lsum[q][i] = 0.f;
    pin_lsum<D>(lsum[q], q);
    st[q].alpha = 1.f;
  }
  bias_ready(bias);

  // ---- tile iterations: two steps each ---------------------------------------------------------------------------
  auto tile_iter = [&](auto plan, int t) __attribute__((always_inline)) {
    using F = decltype(plan);
    constexpr int S = F::SLOT, kV0 = (2 * S + kVBlocks - 1) % kVBlocks, kV1 = 2 * S % kVBlocks, kV2 = (2 * S + 1) % kVBlocks, kV3 = (2 * S + 2) % kVBlocks;
    srd_t k_srd, v_srd = rows_srd(vb, v_row, t * kBc + kBc / 2, F::QK_NEXT ? kBc : kBc / 2);
    if constexpr (F::STAGE_K) {
      k_srd = rows_srd(kb, k_row, (t + 2) * kBc, kBc);
      settle_scalars(k_srd, v_srd);
    } else {
      settle_scalars(v_srd);
    }
    auto hook1 = [&](int n) __attribute__((always_inline)) {
      constexpr int kSpacing = (2 * kKS + kDv16) * kQ16 / (2 * kPiecesPerWave);
      if (n % kSpacing == 1) {
        const int i = n / kSpacing;
        if (i < kPiecesPerWave) {
          v_piece(v_srd, kV2, kV3, i);
        } else if (i < 2 * kPiecesPerWave) {
          if constexpr (F::STAGE_K) k_piece(k_srd, (S + 2) % 3, i - kPiecesPerWave);
        }
      }
    };
    auto hook2 = [&](int) __attribute__((always_inline)) {};
    constexpr uint32_t k_cur = (uint32_t)(S % 3 * kTileBytes), k_nxt = (uint32_t)((S + 1) % 3 * kTileBytes);
    constexpr uint32_t v_cur = (uint32_t)(kV1 * kBlkBytes), v_prv = (uint32_t)(kV0 * kBlkBytes);
    pipeline_step<D, true, F::QK_NEXT, F::MASK_A != kNoMask, kPvAccumulate, EK, true, F::Q0, F::Q0, F::PV_A, (F::MASK_A < 0 ? -1 : F::MASK_A)>(
        hook1, k_cur + kBlkBytes, v_prv, k_nxt, la, bias, qf, ka, o, sA, sB, pB, pA, mx_all, lsum, sc, pending, vote, t * kBc + 32,
        limit, lane);
    step_end<kDv16, true, false, true>(o, st, mx_all, lsum, bias, sB, pending, vote, sc, lane, kLiftOfThreshold<EK>);
    pipeline_step<D, F::QK_NEXT, F::QK_NEXT, F::MASK_B != kNoMask, kPvAccumulate, EK, true, F::QK_B, F::Q0, F::Q0, (F::MASK_B < 0 ? -1 : F::MASK_B)>(
        hook2, k_nxt, v_cur, k_nxt + kBlkBytes, la, bias, qf, ka, o, sB, sA, pA, pB, mx_all, lsum, sc, pending, vote, (t + 1) * kBc, limit, lane);
    step_end<kDv16, F::QK_NEXT, false, true>(o, st, mx_all, lsum, bias, sA, pending, vote, sc, lane, kLiftOfThreshold<EK>);
    staged_barrier();
  };
  constexpr int kEndMask = CAUSAL ? 0 : kMaskAll;  // of the end's first tile (idle in front of the other tiles)
  if (full > 0) {
    // (the first trip begins in the slot of tile 0)
    for (int t = -lead;;) {
      if (t >= 0) tile_iter(TilePlan<0, 0, 0, 0, kNoMask, kNoMask, true, true>{}, t);
      ++t;
      if (t >= 0) tile_iter(TilePlan<1, 0, 0, 0, kNoMask, kNoMask, true, true>{}, t);
      ++t;
      if constexpr (kPeriod == 6) {
        if (t >= 0) tile_iter(TilePlan<2, 0, 0, 0, kNoMask, kNoMask, true, true>{}, t);
        ++t;
        if (t >= 0) tile_iter(TilePlan<3, 0, 0, 0, kNoMask, kNoMask, true, true>{}, t);
        ++t;
        if (t >= 0) tile_iter(TilePlan<4, 0, 0, 0, kNoMask, kNoMask, true, true>{}, t);
        ++t;
      }
      tile_iter(TilePlan<kPeriod - 1, 0, 0, 0, kNoMask, kEndMask, true, true>{}, t);
      if (++t == full) break;
    }
  }
  // The end's tiles.  (Of a part that is not the last one these are like the others, so that all query blocks run through
  // all of them, with masks that leave such a part's scores as they are: a second end beside the diagonal's made the
  // compiler spill 216 registers.)
  if constexpr (SPLIT && CAUSAL) {
    static_assert(kQ16 == 2, "two tiles");
    tile_iter(TilePlan<0, 0, 0, 0, 0, kMaskAll, false, true>{}, full);
    tile_iter(TilePlan<1, 0, 0, 0, kMaskAll, kNoMask, false, false>{}, full + 1);
  } else if constexpr (CAUSAL) {
    tile_iter(DiagonalPlan<0>{}, full);
    tile_iter(DiagonalPlan<1>{}, full + 1);
    if constexpr (kQ16 == 4) {
      tile_iter(DiagonalPlan<2>{}, full + 2);
      tile_iter(DiagonalPlan<3>{}, full + 3);
    }
  } else {
    tile_iter(TilePlan<0, 0, 0, 0, kMaskAll, kNoMask, false, false>{}, full);
  }

  // ---- the second product of the last block -----------------------------------------------------------------------
  constexpr int kLastQ = CAUSAL && !SPLIT ? kQ16 - 1 : 0, kLastSlot = ((CAUSAL ? 2 * kQ16 : 2) - 1) % kVBlocks;
  drain_o(o);
#pragma unroll
  for (int b = 0; b < kDv16; ++b) {
    const f16x8 vf = read_v<D>((uint32_t)(kLastSlot * kBlkBytes), la, b);
#pragma unroll
    for (int q = kLastQ; q < kQ16; ++q) mfma_o<true, EK>(o[q][b], vf, pB[q]);
  }
  drain_o(o);
  drain_lsum<D>(lsum);

  // ---- epilogue ----------------------------------------------------------------------------------------------
  // (the lane's number again, from the hardware: nothing of it is kept through the iterations)
  int lane_e = (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
  asm volatile("" : "+v"(lane_e));
  const int n_e = lane_e & 15, g_e = lane_e >> 4;
  bool odd = false;
  // two neighbouring tiles of O^T of query block q, as 8 consecutive columns of one of them per lane
  auto store_pair = [&](int q, int b, const f32x4& x, const f32x4& y, float inv) __attribute__((always_inline)) {
    const bool there = (uint32_t)(row0 + 16 * wave + n_e + 64 * q) < (uint32_t)it.nq;
    const f32x4 xs = x * inv, ys = y * inv;
    const u32x2 xu = {pack2<EK>(xs[0], xs[1]), pack2<EK>(xs[2], xs[3])};
    const u32x2 yu = {pack2<EK>(ys[0], ys[1]), pack2<EK>(ys[2], ys[3])};
    u32x4 out;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      auto r = __builtin_amdgcn_permlane16_swap(xu[w], yu[w], false, false);
      out[w] = r[0];
      out[2 + w] = r[1];
    }
    const int dv = 16 * (b + (g_e & 1)) + 8 * (g_e >> 1);
    const uint32_t off = (there && dv < d) ? (uint32_t)(64 * q + 16 * wave + n_e) * o_row + (uint32_t)dv * 2u : kOob;
    __builtin_amdgcn_raw_buffer_store_b128(out, o_rs, off, 0, 0);
    if constexpr (CAUSAL) odd |= there && packed::holds_not_finite<EK == kBF16>(out);
  };
  if (!SPLIT || __builtin_expect(part.parts == 1, 1)) {  // (expected: else O^T moves to other registers here, and spills)
#pragma unroll
    for (int q = 0; q < kQ16; ++q) {
      const float inv = __builtin_amdgcn_rcpf(quad_lane_sum(lsum[q][0], lane_e));
#pragma unroll
      for (int b = 0; b < kDv16; b += 2) store_pair(q, b, o[q][b], o[q][b + 1], inv);
    }
  } else if constexpr (SPLIT) {
    // Parts go to memory and come from there past the L2s (sc0 sc1), which the XCDs do not share; the last one to take a
    // ticket adds them up in their order.
    constexpr int kThrough = 17;
    constexpr uint32_t kPartFloats = (uint32_t)(kPackedRows * D);
    // (the arguments are read again here, rather than kept in registers through the iterations)
    const packed::Params* late = (const packed::Params*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(late));
    const uint32_t nth = blockIdx.x / late->items, number = item_of_part(blockIdx.x - nth * late->items, nth);
    const uint32_t slots = late->items * (uint32_t)late->parts;
    const __amdgpu_buffer_rsrc_t part_o = __builtin_amdgcn_make_buffer_rsrc(late->part_o, 0, (int)(slots * kPartFloats * 4u), 0x00020000);
    const __amdgpu_buffer_rsrc_t part_ml = __builtin_amdgcn_make_buffer_rsrc(late->part_ml, 0, (int)(slots * (uint32_t)kPackedRows * 8u), 0x00020000);
    const uint32_t slot0 = number * (uint32_t)late->parts;
    // (a scalar: byte offset of the wave's values in a part)
    auto o_at = [&](uint32_t slot, int q, int b) __attribute__((always_inline)) {
      return (int)((slot * kPartFloats + (uint32_t)(((wave * kQ16 + q) * kDv16 + b) * 64 * 4)) * 4u);
    };
    auto ml_at = [&](uint32_t slot, int q) __attribute__((always_inline)) {
      return (slot * (uint32_t)kPackedRows + (uint32_t)(64 * q + 16 * wave + n_e)) * 8u;
    };
#pragma unroll
    for (int q = 0; q < kQ16; ++q) {
      const float l = quad_lane_sum(lsum[q][0], lane_e);
#pragma unroll
      for (int b = 0; b < kDv16; ++b) {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o[q][b]), part_o, lane_e * 16, o_at(slot0 + nth, q, b), kThrough);
      }
      if (g_e == 0) {
        __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(st[q].mc * sc.c), __float_as_uint(l)}, part_ml,
                                              ml_at(slot0 + nth, q), 0, kThrough);
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    uint32_t* const said = (uint32_t*)smem_raw;  // (the rings are done with)
    if (tid == 0) *said = __hip_atomic_fetch_add(late->tickets + number, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (*said != (uint32_t)part.parts - 1) return false;
    asm volatile("" ::: "memory");
    if (tid == 0) __hip_atomic_store(late->tickets + number, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const int parts = part.parts;
    // reference and sum of a row in part `first` + g_e, or in the last part
    auto load_ml = [&](int q, int first) __attribute__((always_inline)) {
      const int i = first + g_e < parts ? first + g_e : parts - 1;
      return __builtin_amdgcn_raw_buffer_load_b64(part_ml, ml_at(slot0 + (uint32_t)i, q), 0, kThrough);
    };
#pragma unroll 1
    for (int q = 0; q < kQ16; ++q) {
      float m = -INFINITY;
#pragma unroll 1
      for (int first = 0; first < parts; first += 4) m = fmaxf(m, __uint_as_float(load_ml(q, first)[0]));
      m = quad_lane_max(m, lane_e);
      constexpr int kTogether = 4;  // tiles of O^T that are fetched together, of four parts
#pragma unroll 1
      for (int b0 = 0; b0 < kDv16; b0 += kTogether) {
        f32x4 sum[kTogether];
        float l = 0.f;
#pragma unroll
        for (int b = 0; b < kTogether; ++b) sum[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
        for (int first = 0; first < parts; first += 4) {
          const u32x2 ml = load_ml(q, first);
          f32x4 x[kTogether][4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t slot = slot0 + (uint32_t)(first + i < parts ? first + i : parts - 1);
#pragma unroll
            for (int b = 0; b < kTogether; ++b) {
              x[b][i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(part_o, lane_e * 16, o_at(slot, q, b0 + b), kThrough));
            }
          }
          const float w = first + g_e < parts ? fast_exp2(__uint_as_float(ml[0]) - m) : 0.f;
          l += first + g_e < parts ? w * __uint_as_float(ml[1]) : 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float wi = __shfl(w, 16 * i + n_e);
#pragma unroll
            for (int b = 0; b < kTogether; ++b) {
              if (first + i < parts) sum[b] += x[b][i] * wi;
            }
          }
        }
        const float inv = __builtin_amdgcn_rcpf(quad_lane_sum(l, lane_e));
#pragma unroll
        for (int b = 0; b < kTogether; b += 2) store_pair(q, b0 + b, sum[b], sum[b + 1], inv);
      }
    }
  }
  if constexpr (CAUSAL) {
    if (__builtin_amdgcn_ballot_w64(odd) != 0) {
      bool found = false;
      for (int32_t x = a0 * C::kChunks + lane_e; x < (a0 + kPackedRows) * C::kChunks; x += 64) {
        const int32_t key = x / C::kChunks, c = x % C::kChunks;
        if (key < it.nk && c * 8 < d) found |= packed::holds_not_finite<EK == kBF16>(*(const u32x4*)(vb + (int64_t)key * p.v_token + c * 16));
      }
      return __builtin_amdgcn_ballot_w64(found) != 0;
    }
  }
#endif  // __HIP_DEVICE_COMPILE__
  return false;
}

}  // namespace FLASH_M16_NS
}  // namespace flash_hip
