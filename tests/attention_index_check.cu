// Host-side check of attention_flash.cuh's index arithmetic (no GPU needed):
// prints "ok", or the first case that is wrong.
#include <stdio.h>

#include <vector>

#include "attention_flash.cuh"

using namespace emx;

static int wrong(const char* what, long long a, long long b, long long c) {
  printf("%s: %lld %lld %lld\n", what, a, b, c);
  return 1;
}

// n / d for every n up to the product bound, or around multiples of d near it
static int check_div() {
  const unsigned ds[] = {1, 2, 3, 4, 5, 7, 8, 12, 16, 31, 33, 127, 128, 255, 1000, 4097, 65535, 65536};
  for (unsigned d : ds) {
    const SmallDiv s = SmallDiv::of(d);
    const long long most = d == 1 ? 0x7fffffffll : ((1ll << 32) - 1) / d;  // n * d < 2^32
    const long long limit = most < 0x7fffffffll ? most : 0x7fffffffll;
    for (long long n = 0; n <= limit && n < 100000; ++n)
      if (s.div((int)n) != n / d) return wrong("div", n, d, s.div((int)n));
    for (long long k = 0; k < 2000; ++k)
      for (long long e = -1; e <= 1; ++e) {
        const long long n = limit / d * d - k * d + e;
        if (n >= 0 && n <= limit && s.div((int)n) != n / d) return wrong("div", n, d, s.div((int)n));
      }
  }
  return 0;
}

// every (sequence, head, token) is one row of one tile
static int check_rows(int B, int HQ, int HKV, int TQ, int tile, bool all) {
  const int group = HQ / HKV, rows_all = TQ * group * (all ? B : 1);
  const SmallDiv g = SmallDiv::of(group), t = SmallDiv::of(TQ);
  std::vector<int> seen((size_t)B * HQ * TQ);
  for (int b = 0; b < (all ? 1 : B); ++b)
    for (int kvh = 0; kvh < HKV; ++kvh)
      for (int row0 = 0; row0 < rows_all; row0 += tile)
        for (int r = row0; r < rows_all && r < row0 + tile; ++r) {
          const RowId id = row_of(r, g, t, kvh, b, all);
          if (id.b < 0 || id.b >= B || id.h < kvh * group || id.h >= (kvh + 1) * group || id.t < 0 || id.t >= TQ)
            return wrong("row", r, kvh, b);
          ++seen[((size_t)id.b * HQ + id.h) * TQ + id.t];
        }
  for (size_t i = 0; i < seen.size(); ++i)
    if (seen[i] != 1) return wrong("seen", (long long)i, seen[i], all);
  return 0;
}

// the splits' tiles are 0 .. n - 1 in order, about the same number each
static int check_splits() {
  for (int splits = 1; splits <= 300; splits += splits < 20 ? 1 : 37)
    for (int n : {0, 1, 2, 5, 63, 64, 65, 1000, 1 << 20, (1 << 25) - 1}) {
      if (split_start(n, 0, splits) != 0 || split_start(n, splits, splits) != n) return wrong("ends", n, splits, 0);
      for (int s = 0; s < splits; ++s) {
        const int len = split_start(n, s + 1, splits) - split_start(n, s, splits);
        if (len < n / splits || len > n / splits + 1) return wrong("split", n, splits, s);
      }
    }
  return 0;
}

int main() {
  if (check_div() || check_splits()) return 1;
  const int shapes[][4] = {{3, 6, 2, 5}, {70, 8, 8, 1}, {2, 4, 1, 50}, {5, 12, 4, 3}, {1, 1, 1, 1}, {9, 128, 1, 7}, {40, 5, 1, 33}};
  for (auto& s : shapes)
    for (int tile : {8, 16, 128, 256})
      for (int all = 0; all < 2; ++all)
        if (check_rows(s[0], s[1], s[2], s[3], tile, all != 0)) return 1;
  printf("ok\n");
  return 0;
}
