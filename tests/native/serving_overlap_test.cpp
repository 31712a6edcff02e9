// Host test of rows_meet (csrc/serving_index.hpp) against a count of every element.
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "../../flash-attention_amd/csrc/serving_index.hpp"

using namespace flash_hip;

static uint64_t state = 88172645463325252ull;
static uint32_t rnd() {
  state ^= state << 13;
  state ^= state >> 7;
  state ^= state << 17;
  return (uint32_t)(state >> 16);
}

int main() {
  long meet = 0, apart = 0, extra = 0;
  for (int n = 0; n < 400000; ++n) {
    const int dims = 1 + n % 3;
    const int64_t d = 1 + rnd() % 9;
    RowDim x[3] = {{1, 0}, {1, 0}, {1, 0}};
    for (int i = 0; i < dims; ++i) x[i] = RowDim{(int64_t)(rnd() % 6), (int64_t)(rnd() % (rnd() % 2 ? 60 : 200))};
    if (n % 5 == 0) {  // nested, as tensors are
      int64_t span = d;
      for (int i = 0; i < dims; ++i) {
        x[i].stride = span + rnd() % 3;
        span = x[i].stride * std::max<int64_t>(x[i].count, 1);
      }
    }
    std::vector<int64_t> all;
    for (int64_t i = 0; i < x[0].count; ++i)
      for (int64_t j = 0; j < x[1].count; ++j)
        for (int64_t k = 0; k < x[2].count; ++k)
          for (int64_t e = 0; e < d; ++e) all.push_back(i * x[0].stride + j * x[1].stride + k * x[2].stride + e);
    std::sort(all.begin(), all.end());
    const bool want = std::adjacent_find(all.begin(), all.end()) != all.end();
    std::swap(x[rnd() % 3], x[rnd() % 3]);
    const bool got = rows_meet(x[0], x[1], x[2], d);
    // never an overlap that is not seen; one too many only among three that interleave
    if (want && !got) return printf("overlap not seen, case %d\n", n), 1;
    if (got && !want) {
      if (dims < 3 || n % 5 == 0) return printf("overlap where there is none, case %d\n", n), 1;
      ++extra;
    }
    (got ? meet : apart) += 1;
  }
  if (meet < 1000 || apart < 1000 || extra > meet / 5) return printf("%ld %ld %ld\n", meet, apart, extra), 1;
  if (!rows_meet({1 << 30, 0}, {1, 0}, {1, 0}, 8) || rows_meet({1 << 30, (int64_t)1 << 20}, {65535, 16}, {1, 0}, 16)) return 1;
  // sizes that no memory holds
  for (int64_t big : {(int64_t)1 << 40, ((int64_t)1 << 40) - 8}) {
    if (rows_meet({1 << 30, big}, {1 << 30, 64}, {1, 0}, 64) != (((int64_t)1 << 36) > big)) return printf("large strides\n"), 1;
    if (!rows_meet({1 << 30, big}, {1 << 30, big}, {1 << 30, big}, 8)) return printf("large strides\n"), 1;
    if (!rows_meet({1 << 30, big}, {1 << 30, big + 8}, {1, 0}, 16)) return printf("large strides\n"), 1;
  }
  printf("rows that meet are found\n");
  return 0;
}
