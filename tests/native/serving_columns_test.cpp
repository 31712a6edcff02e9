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
      // K: one 16-byte load for `wide` columns (8-byte ones where a row is shorter than that)
      std::vector<int> used(d, 0);
      for (int g = 0; g < 4; ++g) {
        for (int ks = 0; ks < steps; ks += wide / 8) {
          const int column = k_column(cache8, ks, g), width = wide <= d ? wide : 8;
          EXPECT(!cache8 || k_column(true, ks + 1, g) == column + 8);
          for (int c = column; c < column + wide; c += width) {   // (once, but for rows of 8 elements)
            const RowLoad x = row_load(c, width, d);
            EXPECT(x.from >= 0 && x.from + width <= d);
            EXPECT(x.skip == 0 || x.skip == width || (wide == 16 && x.skip == 8));
            for (int e = x.skip; e < width; ++e) {
              EXPECT(x.from + e == c + e - x.skip);
              used[x.from + e] += 1;
            }
          }
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
