// Packed prompts on the pipelined kernel body (attn_fwd_mfma16_body.hpp: four waves, K and V through LDS rings).  One work
// item = 128 or 256 query rows of one sequence and head.
//
// What bounds it: 4 d operations for each visible (query, key) pair, on the matrix cores; K and V are read from the L2s by
// every item.  One prompt of 16384 rows, 32 heads of 128 over 8, bf16: 1.71 ms, 1290 TFLOP/s (8192^3 library product on the
// same chip: 1261); 13 ragged ones of 0 to 2048 rows 122 us (floor 80; the matrix cores are busy 43 % of the time: starts and ends of items).
//
// The causal square is cut where the matrix tiles are: an item's first row is placed so that its last visible key ends
// a 64-key tile (the first item of a sequence may be shorter).  Wave w holds, as query block q, the rows
// 64 q + 16 w .. + 15 of the item, so that in the last tiles (the diagonal, four at 256 rows) tile T is seen in part by block T of
// every wave, whole by the blocks behind it and not at all by those before it: the steps of tile T leave the first T
// blocks out and mask one, with the same work for every wave.  The diagonal then costs 2.5 tiles of matrix time
// instead of 4 (rows in consecutive blocks per wave would make the last wave do all four).
//
// P enters the second product rounded to the tensors' 16-bit type (half a step of each weight), as in the operators for equal
// lengths: a second product for what the rounding leaves would cost a third of the rate.  Its sum l is taken of the rounded
// weights.
//
// Values of keys that some rows of a tile do not see are multiplied by 0 there; where they are infinite or NaN that is
// wrong, and such rows come out as NaN.  A wave whose output holds one looks at the values of its diagonal tiles and, if
// they hold one, computes its rows again on the path that keeps them apart (attend_rows).
//
// Two layouts (attn_packed_mfma_body.hpp):
//   m16   64 query rows per wave, 256 per item, one workgroup per compute unit;
//   m16h  32 query rows per wave, 128 per item, two workgroups per compute unit (80 KB of LDS each at d = 128: three K
//         tiles and four half tiles of V), whose starts and ends overlap with each other's matrix work.
#pragma once

#include "attn_fwd_mfma16.hpp"
#include "attn_packed.hpp"

#define FLASH_M16_NS m16h
#define FLASH_M16_ROWS 32
#define FLASH_M16_WAVES 4
#include "attn_fwd_mfma16_body.hpp"
#undef FLASH_M16_NS
#undef FLASH_M16_ROWS
#undef FLASH_M16_WAVES

namespace flash_hip {
namespace packed {

// How far in front of a sequence's first row its first item begins (see above).
__device__ __forceinline__ int32_t packed_shift(int32_t nq, int32_t nk, bool causal) {
  return causal ? (nk - nq) & (kBc - 1) : 0;
}

// any of the packed 16-bit values infinite or NaN
template <bool BF16>
__device__ __forceinline__ bool holds_not_finite(const u32x4& w) {
  constexpr uint32_t kExponent = BF16 ? 0x7f80u : 0x7c00u;
  bool any = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    any |= (w[i] & kExponent) == kExponent || ((w[i] >> 16) & kExponent) == kExponent;
  }
  return any;
}

// The workgroup's item.  K/V heads are taken in batches that hold at least four query heads.  The 8 XCDs form teams of f,
// as many teams as divide the number of batches, and a team works its batches off one after the other, each XCD every
// f-th tile, from the last row to the first (the longest items first): the readers of a head's K and V share an L2 or a
// few, and every XCD gets its share of long and short items.  For every tile come the batch's query heads: an
// XCD hands its workgroups to its four shader engines in turn, whether they have room or not, so four items of one
// length in a row keep them evenly loaded (with the eight tiles of one head in a row instead, causal, 1024 rows, 96
// heads, a compute unit was busy 70 % of the time: one engine got the longest item and the fifth of every head).
struct Item {
  Tile it;
  int32_t head, kvh;
  int32_t row0;  // first row inside the sequence, may be negative
  int32_t a0;    // keys seen by all rows of the item, a multiple of 64; negative: some rows see none
};
__device__ __forceinline__ Item find_item(const Params& p, uint32_t id, int32_t rows, bool causal, int lane) {
  Item x;
  auto extent = [&](int32_t nq, int32_t nk) __attribute__((always_inline)) { return nq > 0 ? nq + packed_shift(nq, nk, causal) : 0; };
  const TileLine<decltype(extent)> line{p, rows, lane, extent};
  const auto c = line.chunk(0);
  const ItemPlace at = item_place(id, line.length(c), (uint32_t)p.heads, (uint32_t)p.kv_heads);
  x.it.there = at.there;
  if (!at.there) return x;
  x.head = (int32_t)at.head;
  x.kvh = (int32_t)(at.head / (uint32_t)(p.heads / p.kv_heads));
  x.it = line.tile(at.tile, c);
  x.row0 = x.it.row - packed_shift(x.it.nq, x.it.nk, causal);
  x.a0 = causal ? x.row0 + x.it.nk - x.it.nq : 0;
  return x;
}

}  // namespace packed
}  // namespace flash_hip

#define FLASH_M16_NS m16
#define FLASH_PACKED_V_BLOCKS 6
#include "attn_packed_mfma_body.hpp"
#undef FLASH_M16_NS
#undef FLASH_PACKED_V_BLOCKS

#define FLASH_M16_NS m16h
#define FLASH_PACKED_V_BLOCKS 4
#include "attn_packed_mfma_body.hpp"
#undef FLASH_M16_NS
#undef FLASH_PACKED_V_BLOCKS
