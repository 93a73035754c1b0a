// Host test of attention's units (kv_index.h): whatever the offsets of the sequences' rows are, ascending or not, a unit's rows and heads
// are those of the tensors, the positions it sees are in the cache, and ascending offsets give every row once.
#include <stdio.h>
#include <stdlib.h>

#include <climits>
#include <random>
#include <vector>

#include "kv_index.h"

using namespace amem;

#define CHECK(x)                             \
  do {                                       \
    if (!(x)) {                              \
      printf("line %d: %s\n", __LINE__, #x); \
      exit(1);                               \
    }                                        \
  } while (0)

// What a wave of the kernels counts: 64 sequences at a time, all of those that are not above u, on to the next 64 if all were.
static int find(const KvBatch& b, int u, int tile, int group) {
  int count = 0;
  for (int s0 = 0; s0 < b.sequences; s0 += 64) {
    int n = 0;
    for (int s = s0; s < s0 + 64 && s < b.sequences; ++s) n += kv_unit_base(b, s, tile, 1, group) <= u;
    count += n;
    if (n < 64) break;
  }
  return count - 1;
}

static long negative = 0;

// All units of a call; `times`: how often each (token row, head of a group) came up.
static void units(const KvBatch& b, int group, int tile, bool causal, int window, std::vector<int>& times) {
  times.assign((size_t)b.tokens * group, 0);
  for (int index = 0; index < kv_units(b, tile, 1, group); ++index) {
    const int s = find(b, index, tile, group);
    if (s < 0) continue;
    CHECK(s < b.sequences);
    const KvSeq q = kv_seq(b, s);
    KvUnit u;
    const int of = index - kv_unit_base(b, s, tile, 1, group);
    negative += of < 0;
    if (!kv_unit_at(causal, window, group, tile, s, of, q, u)) continue;
    CHECK(u.rows >= 1 && u.rows <= tile && u.first >= 0 && u.first + u.rows <= q.n * group);
    int lo = INT_MAX, to = INT_MIN, all_from = 0, all_to = INT_MAX;
    for (int r = u.first; r < u.first + u.rows; ++r) {
      const int row = q.row + r / group, head = r % group;
      CHECK(row >= 0 && row < b.tokens && head >= 0 && head < group);
      ++times[(size_t)row * group + head];
      int from, end;
      kv_row_range(causal, window, q, r / group, from, end);
      CHECK(from >= 0 && end <= q.context);
      // as 64 bits have it
      const int64_t pos = (int64_t)q.context - q.n + r / group, far = window ? pos - window + 1 : 0;
      CHECK(from == (far > 0 ? far : 0) && end == (causal && pos + 1 < q.context ? pos + 1 : q.context));
      lo = from < lo ? from : lo;
      to = end > to ? end : to;
      all_from = from > all_from ? from : all_from;
      all_to = end < all_to ? end : all_to;
    }
    CHECK(u.lo == lo && u.to == to && u.all_from == all_from && u.all_to == all_to && u.from >= 0 && u.from <= lo && u.from % 64 == 0);
  }
}

int main() {
  std::vector<int> times;
  {  // offsets that fall: unit 7 is counted to a sequence that begins behind it
    const int cu[] = {0, 8, 15, 16, 16, 11, 14}, context[] = {20, 20, 20, 20, 20, 20};
    KvBatch b = {};
    b.cu_tokens = cu;
    b.context = context;
    b.sequences = 6;
    b.tokens = 16;
    b.max_context = 32;
    units(b, 4, 16, true, 0, times);
    CHECK(negative == 1);
  }
  std::mt19937 r(11);
  for (int round = 0; round < 6000; ++round) {
    const int seqs = 1 + r() % (round % 5 ? 9 : 150), most = 1 << (r() % 7), group = 1 + r() % 9;
    const bool wrong = round % 2;
    std::vector<int> cu(1, 0), context;
    for (int s = 0; s < seqs; ++s) {
      cu.push_back(cu.back() + r() % (most + 1));
      context.push_back(r() % 8 ? cu[s + 1] - cu[s] + r() % 300 : r() % 30);  // some are shorter than the new tokens
    }
    const int used = cu.back();
    KvBatch b = {};
    b.sequences = seqs;
    b.tokens = used + r() % 3;
    b.max_context = 500;
    if (wrong) {
      const int odd[] = {-1, INT_MIN, INT_MAX, b.tokens, b.tokens / 2, 0, 1};
      for (int i = 0; i < 6; ++i) {
        cu[r() % cu.size()] = i % 2 ? odd[r() % 7] : (int)(r() % (b.tokens + 1));
        context[r() % context.size()] = odd[r() % 7];
      }
    }
    b.cu_tokens = cu.data();
    b.context = context.data();
    const int windows[] = {0, 0, 1, 5, 64, 1000, INT_MAX, INT_MAX - 1};
    for (int tile : {16, 48, 128}) {
      units(b, group, tile, r() % 2, windows[r() % 8], times);
      if (!wrong)
        for (int i = 0; i < b.tokens * group; ++i) CHECK(times[i] == (i < used * group));
    }
  }
  CHECK(negative > 100);
  printf("ok\n");
  return 0;
}
