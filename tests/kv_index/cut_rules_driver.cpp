// The rules by which attention is cut (kv_cut.h), with the kernels' own figures: parts fit what the workspace is sized for, stretches cover
// the span in multiples of a tile, and the borders of the rules are where they are said to be.
#include <cstdio>
#include <cstdlib>
#include <random>

#include "kv_cut.h"

using namespace amem;

static long cut_some, cut_part, shortest, unsteady;

static bool check(const Cut& cut, int pairs, int64_t span, int64_t longest, bool even) {
  const CutInto into = cut_last_round(cut, pairs, span, even);
  const int64_t parts = into.splits > 1 ? (int64_t)(pairs - into.whole) * into.splits : 0;
  bool fine = into.splits >= 1 && into.whole >= 0 && into.whole <= pairs && parts <= most_parts(cut, pairs, longest);
  if (into.splits == 1) {
    fine = fine && into.whole == pairs;
  } else {
    fine = fine && pairs - into.whole <= cut.fit && into.whole % cut.fit == 0 && into.stretch > 0 && into.stretch % 64 == 0 &&
           (int64_t)into.stretch * into.splits >= span && (int64_t)into.stretch * into.splits < (int64_t)1 << 31 && span >= cut.shorter;
    if (into.stretch <= 512) fine = fine && into.stretch % std::min(cut.least, cut.step) == 0;
    ++cut_some;
    cut_part += into.whole > 0;
    shortest += into.stretch == 128;
    unsteady += into.stretch % cut.step != 0;
  }
  if (!fine)
    printf("fit %d least %d pairs %d span %lld: whole %d splits %d stretch %d, room for %lld parts\n", cut.fit, cut.least, pairs, (long long)span,
           into.whole, into.splits, into.stretch, (long long)most_parts(cut, pairs, longest));
  return fine;
}

int main() {
  std::mt19937 r(5);
  auto pick = [&](int64_t lo, int64_t hi) { return (int64_t)(lo + r() % (uint64_t)(hi - lo + 1)); };
  const int shapes[][2] = {{128, 256}, {128, 768}, {256, 256}, {128, 512}};  // rows of a unit, workgroups that fit
  const int dims[] = {64, 128, 256};
  for (int i = 0; i < 600000; ++i) {
    const int head_dim = dims[r() % 3], blocks = (int)pick(1, head_dim == 64 ? 4 : 2);
    const int* shape = shapes[r() % 4];
    const Cut cut = i % 2 ? cut_of_few(head_dim, r() % 2, blocks) : cut_of_many(shape[0], shape[1]);
    const int pairs = (int)(i % 3 ? pick(1, 2000) : pick(1, 1 << 22));
    const int64_t span = i % 7 == 0 ? pick(0, (1 << 30) - 1) : i % 7 == 1 ? pick(0, 600) : i % 7 == 2 ? pick(370, 1100) : pick(0, 30000);
    const int64_t longest = std::min<int64_t>(span + pick(0, 5000), (1 << 30) - 1);  // a mask shortens the span
    if (!check(cut, pairs, span, longest, r() % 2)) return 1;
  }
  // each border of the span, for few pairs and for a round and a bit
  for (int head_dim : dims)
    for (int eight = 0; eight < 2; ++eight)
      for (int blocks = 1; blocks <= (head_dim == 64 ? 4 : 2); ++blocks)
        for (int pairs : {1, 2, 8, 32, 100, 300, 520, 800})
          for (int64_t span = 0; span <= 1100; ++span)
            if (!check(cut_of_few(head_dim, eight, blocks), pairs, span, span, true)) return 2;
  if (cut_some < 1000 || cut_part < 1000 || shortest < 1000 || unsteady < 1000) return 3;
  // contexts below 384 stay whole, longer ones of one sequence become stretches of 128
  const Cut cut = cut_of_few(128, true, 1);
  if (cut_last_round(cut, 8, 383, true).splits != 1 || cut_last_round(cut, 8, 384, true).stretch != 128) return 4;
  printf("ok\n");
}
