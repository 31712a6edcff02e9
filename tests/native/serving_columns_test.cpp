// Host walk through the loads of decoding's cache rows (csrc/serving_index.hpp): for every head dim, tile and width of a
// cache element no load of K or V leaves its row at either end, and every column is multiplied once.  And through the
// rule for grids that the runtime takes.
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "../../flash-attention_amd/csrc/serving_index.hpp"

using namespace flash_hip;

#define EXPECT(x)                                                             \
  do {                                                                        \
    if (!(x)) {                                                               \
      printf("line %d, d = %d: %s does not hold\n", __LINE__, d, #x);         \
      exit(1);                                                                \
    }                                                                         \
  } while (0)

int main() {
  for (int d = 8; d <= 128; d += 8) {
    for (int cache8 = 0; cache8 < 2; ++cache8) {
      const int tile = d <= 64 ? 64 : 128, steps = tile / 32, wide = cache8 ? 16 : 8;
      // K: one 16-byte load for `wide` columns (8-byte ones where a row is shorter than that), each column of which goes
      // with a query element at most; over all lanes and steps every one does, once
      std::vector<int> used(d, 0);
      for (int g = 0; g < 4; ++g) {
        for (int ks = 0; ks < steps; ++ks) {
          const int width = wide <= d ? wide : 8, first = k_column(cache8, wide == 16 ? ks & ~1 : ks, g);
          EXPECT(wide == 8 || k_column(true, ks & ~1, g) + 8 * (ks & 1) == k_column(true, ks, g));
          const int from = width == wide ? row_load(first, width, d) : 0;  // (a short row is loaded whole)
          EXPECT(from >= 0 && from + width <= d);
          const int held = from + (width == 16 ? 8 * (ks & 1) : 0);         // first of the 8 elements that the step multiplies
          const int q = q_column(cache8, ks, g, d);
          EXPECT(q == -1 || (q == held && q + 8 <= d && q % 8 == 0));
          if (q < 0) continue;
          for (int e = 0; e < 8; ++e) used[q + e] += 1;
        }
      }
      for (int n : used) EXPECT(n == 1);
      // V: tile / 16 columns of each of 16 lanes, from column 0 for lanes behind the row
      const int mine = tile / 16;
      for (int n = 0; n < 16; ++n) {
        const int from = n * mine < d ? n * mine : 0;
        EXPECT(from + mine <= d);
      }
    }
  }
  for (int threads : {64, 256, 1024}) {
    const int d = threads;
    EXPECT(grid_fits(1, threads) && !grid_fits((1ull << 32) / threads, threads) && !grid_fits(1ull << 63, threads));
    EXPECT(grid_fits((1ull << 32) / threads - 1, threads) && ((1ull << 32) / threads - 1) * threads < 1ull << 32);
  }
  printf("loads stay inside their rows\n");
  return 0;
}
