// Cuts of every kind (kv_cut.h): parts fit what the workspace is sized for, stretches cover the span, and whatever is not worth it stays whole.
#include <cstdio>
#include <cstdlib>
#include <random>

#include "kv_cut.h"

using namespace amem;

int main() {
  std::mt19937 r(7);
  auto pick = [&](int64_t lo, int64_t hi) { return (int64_t)(lo + r() % (uint64_t)(hi - lo + 1)); };
  long cut_some = 0, cut_part = 0;
  for (int i = 0; i < 400000; ++i) {
    const int fit = 256 * (int)pick(1, 3), bytes = 128 << pick(0, 3), blocks = (int)pick(1, 4);
    const Cut cut = i % 2 ? Cut{fit, 4, 2, 256, 256, 37, 39, 33, 79, 5500 / bytes, 12000 / bytes, 34 * blocks * 130 / bytes}
                          : Cut{fit, 2, 0, 512, 64, 66, 33, 0, 100, 0, 150, blocks > 2 ? 200 : 100};
    const int pairs = (int)(i % 3 ? pick(1, 2000) : pick(1, 1 << 22));
    const int64_t span = i % 7 == 0 ? pick(0, (1 << 30) - 1) : i % 7 == 1 ? pick(0, 300) : pick(0, 30000);
    const int64_t longest = std::min<int64_t>(span + pick(0, 5000), (1 << 30) - 1);  // a mask shortens the span
    const CutInto into = cut_last_round(cut, pairs, span, pick(0, 1));
    const int64_t parts = into.splits > 1 ? (int64_t)(pairs - into.whole) * into.splits : 0;
    bool fine = into.splits >= 1 && into.whole >= 0 && into.whole <= pairs && parts <= most_parts(cut, pairs, longest);
    if (into.splits == 1) fine = fine && into.whole == pairs;
    else
      fine = fine && pairs - into.whole <= fit && into.whole % fit == 0 && into.stretch > 0 && into.stretch % cut.step == 0 &&
             (int64_t)into.stretch * into.splits >= span && (int64_t)into.stretch * into.splits < (int64_t)1 << 31;
    if (!fine) {
      printf("fit %d pairs %d span %lld: whole %d splits %d stretch %d, room for %lld parts\n", fit, pairs, (long long)span, into.whole,
             into.splits, into.stretch, (long long)most_parts(cut, pairs, longest));
      return 1;
    }
    cut_some += into.splits > 1;
    cut_part += into.splits > 1 && into.whole;
  }
  if (cut_some < 1000 || cut_part < 1000) return 2;
  // few pairs of long contexts are cut; short contexts and full rounds are not
  const Cut cut = {512, 4, 2, 256, 256, 37, 39, 33, 79, 21, 46, 17};
  if (cut_last_round(cut, 8, 100000, true).splits < 16 || cut_last_round(cut, 8, 200, true).splits != 1 || cut_last_round(cut, 512, 8192, true).splits != 1 ||
      cut_last_round(cut, 520, 8192, true).whole != 512 || cut_last_round(cut, 520, 8192, false).splits != 1)
    return 3;
  printf("ok\n");
}
