// Index arithmetic of the serving kernels: plain functions of the lengths, offsets and page tables that the kernels
// find in device memory.  They decide what is read and written whatever those hold, and compile for the host as well,
// where tests walk them through every kind of content.
#pragma once

#include <cstdint>

#if defined(__HIP__)
#define FLASH_INDEX __host__ __device__ __forceinline__
#else
#define FLASH_INDEX inline
#endif

namespace flash_hip {

FLASH_INDEX int32_t within(int32_t x, int32_t low, int32_t high) { return x < low ? low : (x > high ? high : x); }

// Workgroups that one dimension of a grid can have: the runtime refuses 2^32 threads and more along it
FLASH_INDEX bool grid_fits(uint64_t workgroups, uint32_t threads) { return workgroups < (1ull << 32) / threads; }

// ---- rows that are written ----------------------------------------------------------------------------------------
// Rows of `d` elements at every sum of i * stride, 0 <= i < count, over up to three dimensions.
struct RowDim {
  int64_t count, stride;
};
// elements from the first row of a dimension to its last one, up to 2^61
FLASH_INDEX int64_t row_reach(RowDim x) {
  constexpr int64_t kMost = (int64_t)1 << 61;
  return x.stride > 0 && x.count - 1 > kMost / x.stride ? kMost : (x.count - 1) * x.stride;
}
// Whether two of the rows share an element: dimensions whose strides reach over all that the smaller ones span do not add
// to that, nor do two that interleave without meeting.  (A third one that interleaves with both counts as meeting.)
FLASH_INDEX bool rows_meet(RowDim a, RowDim b, RowDim c, int64_t d) {
  RowDim dims[3] = {a, b, c};
  for (int i = 0; i < 3; ++i) {
    if (dims[i].count < 1) return false;  // no rows
    if (dims[i].count == 1) dims[i].stride = 0;
    for (int j = i; j > 0 && dims[j].stride < dims[j - 1].stride; --j) {
      const RowDim x = dims[j];
      dims[j] = dims[j - 1];
      dims[j - 1] = x;
    }
  }
  int64_t span = d;  // of the dimensions so far
  for (int i = 0; i < 3; ++i) {
    if (dims[i].count == 1) continue;
    if (dims[i].stride < span) {
      const int inner = i - 1;
      if (dims[i].stride < d || inner < 0 || span != d + row_reach(dims[inner])) return true;
      // two dimensions: rows i * outer + j * inner are apart if no multiple of the outer stride comes closer than d to one of
      // the inner stride
      const int64_t step = dims[inner].stride, most = dims[inner].count - 1;
      for (int64_t n = 1; n < dims[i].count && n * dims[i].stride < span; ++n) {
        const int64_t at = n * dims[i].stride, below = at / step < most ? at / step : most;
        if (at - below * step < d || (below < most && (below + 1) * step - at < d)) return true;
      }
    }
    span += row_reach(dims[i]);
  }
  return false;
}

// ---- packed sequences -------------------------------------------------------------------------------------------
struct Range {
  int32_t start, count;
};
// rows of the sequence between two neighbouring entries of cu_seqlens, cut to the tensor's `total` rows
FLASH_INDEX Range sequence_rows(int32_t from, int32_t to, int32_t total) {
  const int32_t start = within(from, 0, total);
  return Range{start, within(to, start, total) - start};
}
// Tiles of `rows` query rows for many sequences: numbers with gaps, which need no sum over the sequences in front.  Sequence b,
// whose rows start at `start`, takes those from here to the next sequence's: at least count / rows + `extra` of them.
FLASH_INDEX uint32_t first_tile(int32_t start, int32_t total, uint32_t rows, uint32_t extra, int32_t b) {
  return (uint32_t)within(start, 0, total) / rows + extra * (uint32_t)b;
}
// keys that row `row` of a sequence with nq queries and nk keys sees
FLASH_INDEX int32_t visible_keys(int32_t row, int32_t nq, int32_t nk, bool causal) {
  return causal ? within(row + (nk - nq) + 1, 0, nk) : nk;
}
// The sequence that row t belongs to: the last one that starts at or before t (empty ones share their start with the
// one behind them); -1: none starts there.  The result is below `sequences` for any content.
template <typename Offsets>
FLASH_INDEX int32_t sequence_of(const Offsets& cu, int32_t sequences, int32_t t) {
  int32_t lo = 0, hi = sequences;
  while (lo < hi) {
    const int32_t mid = lo + (hi - lo) / 2;
    if (cu(mid) <= t) {
      lo = mid + 1;
    } else {
      hi = mid;
    }
  }
  return lo - 1;
}

// Which query tile and head workgroup `id` of a grid of packed_grid(...) works on, of `tiles` tiles that there are; every
// pair comes once.  (The order is explained with the kernel that uses it.)
struct ItemPlace {
  uint32_t tile, head;
  bool there;
};
struct ItemTeams {
  uint32_t batch, batches, teams, members;  // K/V heads a batch; XCDs of a team
};
FLASH_INDEX ItemTeams item_teams(uint32_t heads, uint32_t kv_heads) {
  const uint32_t group = heads / kv_heads, batch = group >= 4 ? 1 : (group == 1 ? 4 : 2), batches = (kv_heads + batch - 1) / batch;
  const uint32_t divisor = batches & (0u - batches), teams = divisor < 8 ? divisor : 8;
  return ItemTeams{batch, batches, teams, 8 / teams};
}
FLASH_INDEX uint64_t packed_grid(uint64_t tiles, uint32_t heads, uint32_t kv_heads) {
  const ItemTeams t = item_teams(heads, kv_heads);
  return 8ull * (t.batches / t.teams) * ((tiles + t.members - 1) / t.members) * t.batch * (heads / kv_heads);
}
FLASH_INDEX ItemPlace item_place(uint32_t id, uint32_t tiles, uint32_t heads, uint32_t kv_heads) {
  const ItemTeams t = item_teams(heads, kv_heads);
  const uint32_t group = heads / kv_heads, xcd = id & 7u, place = id >> 3;
  const uint32_t team = xcd & (t.teams - 1), member = xcd / t.teams;
  // tiles of this XCD: one of every `members`, back and forth, so that their lengths add up alike
  const uint32_t rounds = tiles / t.members, rest = tiles - rounds * t.members;
  const uint32_t mine = rounds + (((rounds & 1) ? t.members - 1 - member : member) < rest ? 1 : 0);
  const uint32_t each = mine * t.batch * group;
  if (each == 0 || place >= each * (t.batches / t.teams)) return ItemPlace{0, 0, false};
  const uint32_t nth = place / each, kv0 = (team + nth * t.teams) * t.batch, left = kv_heads - kv0;
  const uint32_t here = (left < t.batch ? left : t.batch) * group, in_batch = place - nth * each, round = in_batch / here;
  const uint32_t slot = round * t.members + ((round & 1) ? t.members - 1 - member : member);
  return ItemPlace{tiles - 1 - slot, kv0 * group + (in_batch - round * here), round < mine};
}

// ---- the paged cache --------------------------------------------------------------------------------------------
struct Pages {
  int64_t page_stride, slot_stride;  // bytes
  int32_t num_pages, max_keys, page_shift;
};
// byte offset of position `pos` inside a head of the cache, -1 for a page index outside it
FLASH_INDEX int64_t position_offset(const Pages& c, int32_t page, int32_t pos) {
  if ((uint32_t)page >= (uint32_t)c.num_pages) return -1;
  return (int64_t)page * c.page_stride + (int64_t)(pos & ((1 << c.page_shift) - 1)) * c.slot_stride;
}
// Position of a token that stands `behind` rows (itself among them) before the end of its sequence of length `len`;
// -1: outside the table
FLASH_INDEX int32_t new_position(const Pages& c, int32_t len, int32_t behind) {
  const int64_t pos = (int64_t)len - behind;
  return behind > 0 && pos >= 0 && pos < c.max_keys ? (int32_t)pos : -1;
}
FLASH_INDEX int32_t cache_length(const Pages& c, int32_t len) { return within(len, 0, c.max_keys); }

// ---- columns of a cache row that a lane loads, of d (a multiple of 8) ------------------------------------------------
// first of the 8 head-dim elements that lane group g multiplies in k-step ks; a 16-byte load of an 8-bit row holds
// those of two k-steps
FLASH_INDEX int32_t k_column(bool cache8, int32_t ks, int32_t g) { return cache8 ? 64 * (ks / 2) + 16 * g + 8 * (ks & 1) : 32 * ks + 8 * g; }
// Where a load of `width` elements (at most d) begins for a lane that wants those from `column` on: inside the row at both
// ends.  What it holds in front of `column` others multiply already, or, where column >= d, all of it: no query element
// goes with that.
FLASH_INDEX int32_t row_load(int32_t column, int32_t width, int32_t d) { return column + width <= d ? column : d - width; }
// The query elements that lane group g multiplies the 8 elements of k-step ks with: those from here on, -1: zeros.
FLASH_INDEX int32_t q_column(bool cache8, int32_t ks, int32_t g, int32_t d) {
  const int32_t wide = cache8 && d >= 16 ? 16 : 8, first = k_column(cache8, wide == 16 ? ks & ~1 : ks, g);
  const int32_t mine = row_load(first, wide, d) + (wide == 16 ? 8 * (ks & 1) : 0);
  return mine >= first ? mine : -1;
}

// ---- the line of units that decoding workgroups divide among themselves --------------------------------------
// units of a sequence of n keys; an empty one has a unit too, which writes its zeros
FLASH_INDEX uint32_t units_of(int32_t n, int32_t unit) { return n <= unit ? 1u : (uint32_t)((n - 1) / unit + 1); }
// units of every workgroup but the last ones
FLASH_INDEX uint32_t units_each(uint32_t total, uint32_t workgroups) { return (total - 1) / workgroups + 1; }
// Place in the workspace for workgroup w's part of the triple that starts at unit `start` of the line: a workgroup
// holds at most two parts, of the triple it begins with and of the one it ends with.
FLASH_INDEX uint32_t part_slot(uint32_t w, uint32_t each, uint32_t start) { return 2u * w + (w * each < start ? 1u : 0u); }

}  // namespace flash_hip
