// The lists of blocks that attention's workgroups keep in LDS, and their union
// (kv_lists.h), lane by lane over memory that holds what others left there.
#include <cstdint>
#include <cstdio>
#include <random>
#include <set>
#include <vector>

#include "kv_lists.h"

using namespace mlxvs::kern;

int main() {
  std::mt19937 rng(7);
  const auto pick = [&](int lo, int hi) { return (int)(lo + rng() % (uint32_t)(hi - lo + 1)); };
  int failures = 0;
  for (int run = 0; run < 4000; ++run) {
    const int n = run % 3 ? pick(1, 256) : pick(1, 8), stride = n + 1, tokens = pick(1, 3);
    const int cols = pick(1, run % 2 ? 5000 : 100);
    // block numbers that could be: of this table, past it, of later windows
    std::vector<int> lists(tokens * stride);
    for (int& x : lists) x = pick(0, cols + 3000);
    std::set<int> want;
    for (int t = 0; t < tokens; ++t) {
      const int own = pick(-1, cols + 2);
      int* list = lists.data() + t * stride;
      int count = 0;
      const bool few = pick(0, 1);
      for (int e = 0; e < n; ++e) {
        const int b = few && pick(0, 9) ? -1 : pick(-2, cols + 2);
        if (b >= 0 && b < cols && b <= own) want.insert(b);
        if (block_shows(b, cols, own)) list[count++] = b;
      }
      for (int lane = 0; lane < 64; ++lane) end_list(list, count, stride, lane);
    }
    std::set<int> got;
    for (int base = 0; base < cols + 5000; base += kWindow)
      for (int t = 0; t < tokens; ++t)
        for (int lane = 63; lane >= 0; --lane)
          blocks_in_window(lists.data() + t * stride, stride, lane, base, cols, [&](int b) {
            if (b < 0 || b >= kWindow) ++failures;
            got.insert(base + b);
          });
    if (got != want) ++failures;
    // a list that nothing ended still names no block past the table
    for (int lane = 0; lane < 64; ++lane) {
      std::vector<int> left(stride);
      for (int& x : left) x = pick(0, cols + 3000);
      for (int base = 0; base < cols + 5000; base += kWindow)
        blocks_in_window(left.data(), stride, lane, base, cols, [&](int b) {
          if (base + b >= cols) ++failures;
        });
    }
  }
  if (failures) {
    std::printf("%d failures\n", failures);
    return 1;
  }
  std::printf("all tests passed\n");
  return 0;
}
