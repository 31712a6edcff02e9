// Host walk through the index arithmetic of the serving kernels (csrc/serving_index.hpp): every offset that the
// kernels form from lengths, offsets and page tables stays inside the tensors whatever those hold, and the units
// that decoding workgroups take cover every sequence once.
#include <climits>
#include <cstdio>
#include <cstdlib>
#include <set>
#include <vector>

#include "../../flash-attention_amd/csrc/serving_index.hpp"

using namespace flash_hip;

#define EXPECT(x)                                                  \
  do {                                                             \
    if (!(x)) {                                                    \
      printf("line %d: %s does not hold\n", __LINE__, #x);         \
      exit(1);                                                     \
    }                                                              \
  } while (0)

static uint64_t state = 88172645463325252ull;
static uint32_t rnd() {
  state ^= state << 13;
  state ^= state >> 7;
  state ^= state << 17;
  return (uint32_t)(state >> 16);
}
static int32_t strange() {
  static const int32_t all[] = {0, 1, -1, INT_MIN, INT_MAX, INT_MAX - 1, 7, 64, 1000, -64};
  return rnd() % 3 ? all[rnd() % 10] : (int32_t)rnd();
}

static void packed_rows() {
  for (int n = 0; n < 200000; ++n) {
    const int32_t total = rnd() % 3 ? (int32_t)(rnd() % 300) : (1 << 30);
    const Range r = sequence_rows(strange(), strange(), total);
    EXPECT(r.start >= 0 && r.count >= 0 && (int64_t)r.start + r.count <= total);
  }
  for (int nq = 0; nq < 20; ++nq) {
    for (int nk = 0; nk < 20; ++nk) {
      for (int i = 0; i < nq; ++i) {
        int seen = 0;
        for (int j = 0; j < nk; ++j) seen += j <= i + nk - nq;
        EXPECT(visible_keys(i, nq, nk, true) == seen && visible_keys(i, nq, nk, false) == nk);
      }
    }
  }
}

// every (tile, head) pair is the work of exactly one workgroup of the grid, also when fewer tiles exist than the grid
// was made for
static void prompt_items() {
  for (uint32_t kv = 1; kv <= 40; ++kv) {
    for (uint32_t group : {1u, 2u, 3u, 4u, 5u, 8u, 17u}) {
      for (uint32_t bound : {1u, 2u, 7u, 16u, 23u}) {
        for (uint32_t tiles = 0; tiles <= bound; tiles += bound > 7 ? 5 : 1) {
          const uint64_t grid = packed_grid(bound, kv * group, kv);
          EXPECT(grid % 8 == 0 && grid < 1u << 20);
          std::vector<int> seen((size_t)tiles * kv * group, 0);
          for (uint32_t id = 0; id < grid; ++id) {
            const ItemPlace x = item_place(id, tiles, kv * group, kv);
            if (!x.there) continue;
            EXPECT(x.tile < tiles && x.head < kv * group);
            seen[(size_t)x.tile * kv * group + x.head] += 1;
          }
          for (int n : seen) EXPECT(n == 1);
        }
      }
    }
  }
}

// the tile numbers of many sequences: in order, room for all of a sequence's tiles (its first one may begin up to 63 rows
// early where there is room for two more), and all of them inside the grid
static void tile_numbers() {
  for (int n = 0; n < 3000; ++n) {
    const int32_t seqs = 1 + (int32_t)(rnd() % 300);
    const uint32_t rows = n % 3 == 0 ? 64 : n % 3 == 1 ? 128 : 256, extra = 1 + (uint32_t)(n / 3 % 2);
    std::vector<int32_t> cu(seqs + 1);
    cu[0] = (int32_t)(rnd() % 500);
    for (int b = 0; b < seqs; ++b) cu[b + 1] = cu[b] + (int32_t)(rnd() % (rnd() % 4 ? 20 : 700));
    const int32_t total = cu[seqs] + (int32_t)(rnd() % 100);
    const uint32_t grid = (uint32_t)total / rows + extra * (uint32_t)seqs;
    for (int b = 0; b < seqs; ++b) {
      const uint32_t shift = extra == 2 ? rnd() % 64 : 0, count = (uint32_t)(cu[b + 1] - cu[b]);
      const uint32_t mine = count == 0 ? 0 : (count + shift + rows - 1) / rows;
      const uint32_t first = first_tile(cu[b], total, rows, extra, b), next = first_tile(cu[b + 1], total, rows, extra, b + 1);
      EXPECT(first + mine <= next && next <= grid);
    }
    for (int b = 0; b < seqs; ++b) EXPECT(first_tile(strange(), total, rows, extra, b) < grid + extra);
  }
}

static void token_targets() {
  for (int n = 0; n < 20000; ++n) {
    const int32_t seqs = 1 + (int32_t)(rnd() % 9);
    std::vector<int32_t> cu(seqs + 1);
    const bool sane = n % 2;
    cu[0] = sane ? (int32_t)(rnd() % 3) : strange();
    for (int b = 0; b < seqs; ++b) cu[b + 1] = sane ? cu[b] + (int32_t)(rnd() % 4) : strange();
    auto at = [&](int32_t i) {
      EXPECT(i >= 0 && i <= seqs);
      return cu[i];
    };
    for (int t = 0; t < 30; ++t) {
      const int32_t b = sequence_of(at, seqs, t);
      EXPECT(b >= -1 && b < seqs);
      if (!sane) continue;
      int want = -1;
      for (int s = 0; s < seqs; ++s) {
        if (cu[s] <= t && t < cu[s + 1]) want = s;
      }
      const bool inside = b >= 0 && at(b + 1) - t > 0;
      EXPECT(inside == (want >= 0) && (!inside || b == want));
    }
  }
}

static void cache_places() {
  for (int n = 0; n < 200000; ++n) {
    Pages c{};
    c.page_shift = (int32_t)(rnd() % 9);
    c.num_pages = 1 + (int32_t)(rnd() % 50);
    const int32_t width = (int32_t)(rnd() % 20), page = 1 << c.page_shift;
    c.max_keys = width * page;
    c.slot_stride = 16;
    c.page_stride = 16 * page;
    const int32_t len = cache_length(c, strange());
    EXPECT(len >= 0 && len <= c.max_keys);
    const int32_t pos = new_position(c, strange(), strange());
    EXPECT(pos >= -1 && pos < (c.max_keys ? c.max_keys : 1) && (pos < 0 || (pos >> c.page_shift) < width));
    const int32_t entry = strange();
    const int64_t off = position_offset(c, entry, pos < 0 ? 0 : pos);
    EXPECT(off == -1 || (off >= 0 && off + 16 <= (int64_t)c.num_pages * c.page_stride));
    EXPECT((off >= 0) == (entry >= 0 && entry < c.num_pages));
  }
  Pages far{(int64_t)1 << 22, 256, 1 << 30, 1 << 30, 14};
  EXPECT(position_offset(far, (1 << 30) - 1, 16383) == ((int64_t)1 << 52) - ((int64_t)1 << 22) + 16383 * 256);
}

// every unit of every triple is taken once, by the workgroups between the first and the last one of the triple, and no
// two parts share a place in the workspace
static void the_line() {
  for (int n = 0; n < 4000; ++n) {
    const uint32_t triples = 1 + rnd() % 40, workgroups = 1 + rnd() % 70, unit = 128;
    std::vector<uint32_t> units, start;
    uint32_t total = 0;
    for (uint32_t t = 0; t < triples; ++t) {
      const int32_t len = (int32_t)(rnd() % (rnd() % 4 ? 500 : 20000));
      const uint32_t u = units_of(len, (int32_t)unit);
      EXPECT(u >= 1 && (len <= 0 ? u == 1 : (uint64_t)u * unit >= (uint64_t)len && (uint64_t)(u - 1) * unit < (uint64_t)len));
      start.push_back(total);
      units.push_back(u);
      total += u;
    }
    const uint32_t each = units_each(total, workgroups);
    EXPECT((uint64_t)each * workgroups >= total);
    std::vector<uint32_t> taken(total, 0);
    std::set<uint32_t> slots;
    for (uint32_t w = 0; w < workgroups; ++w) {
      const uint32_t begin = w * each;
      if (begin >= total) continue;
      const uint32_t end = begin + each < total ? begin + each : total;
      uint32_t t = 0;
      while (t + 1 < triples && start[t + 1] <= begin) ++t;
      uint32_t u0 = begin - start[t];
      for (uint32_t r = begin; r < end;) {
        const uint32_t u1 = units[t] - u0 < end - r ? units[t] : u0 + (end - r);
        EXPECT(u1 > u0 && u1 <= units[t] && r - u0 == start[t]);
        for (uint32_t u = u0; u < u1; ++u) taken[start[t] + u] += 1;
        const uint32_t first = start[t] / each, last = (start[t] + units[t] - 1) / each;
        EXPECT((u0 == 0 && u1 == units[t]) == (first == last) && first <= w && w <= last);
        if (first != last) {
          const uint32_t slot = part_slot(w, each, start[t]);
          EXPECT(slot < 2 * workgroups && slots.insert(slot).second);
        }
        r += u1 - u0;
        u0 = 0;
        ++t;
      }
    }
    for (uint32_t u : taken) EXPECT(u == 1);
  }
  EXPECT(units_of(1 << 30, 128) == 1u << 23);
}

int main() {
  packed_rows();
  prompt_items();
  tile_numbers();
  token_targets();
  cache_places();
  the_line();
  printf("serving index arithmetic holds\n");
  return 0;
}
