// Host test of kv_index.h: whatever lengths, offsets and page numbers device memory holds, the indexes that the
// kernels build from them stay inside the tensors, and the units of work cover every row and block once.
#include <stdio.h>
#include <stdlib.h>

#include <climits>
#include <random>
#include <vector>

#include "kv_index.h"

using namespace amem;

#define CHECK(x)                                             \
  do {                                                       \
    if (!(x)) {                                              \
      printf("line %d: %s\n", __LINE__, #x);                 \
      exit(1);                                               \
    }                                                        \
  } while (0)

static int find(const KvBatch& b, int u, int tile, int spare) {  // what a wave of the kernels counts
  int n = 0;
  while (n < b.sequences && kv_unit_base(b, n, tile, spare) <= u) ++n;
  return n - 1;
}

int main() {
  std::mt19937 r(7);
  for (int round = 0; round < 4000; ++round) {
    const int seqs = 1 + r() % 9, page_shift = r() % 8, tokens_most = 1 << (r() % 9);
    const bool wrong = round % 2;
    std::vector<int> cu(1, 0), context;
    for (int s = 0; s < seqs; ++s) {
      cu.push_back(cu.back() + r() % (tokens_most + 1));
      context.push_back(cu[s + 1] - cu[s] + r() % 300);
    }
    KvBatch b = {};
    b.sequences = seqs;
    b.tokens = cu.back() + r() % 3;
    b.table_pages = 1 + (tokens_most + 300) / (1 << page_shift);
    b.table_stride = b.table_pages + r() % 3;
    b.max_context = b.table_pages << page_shift;
    KvCache c = {};
    c.pages = 1 + r() % 50;
    c.kv_heads = 1 + r() % 4;
    c.page_shift = page_shift;
    c.block_shift = 4;
    c.slot_stride = 64;
    c.head_stride = (int64_t)c.slot_stride << page_shift;
    c.page_stride = c.head_stride * c.kv_heads;
    std::vector<int> table(seqs * b.table_stride);
    for (int& t : table) t = r() % c.pages;
    if (wrong) {
      const int odd[] = {-1, INT_MIN, INT_MAX, c.pages, b.tokens + 1, -c.pages, 1 << 30};
      for (int i = 0; i < 6; ++i) {
        table[r() % table.size()] = odd[r() % 7];
        cu[r() % cu.size()] = odd[r() % 7];
        context[r() % context.size()] = odd[r() % 7];
      }
    }
    b.page_table = table.data();
    b.context = context.data();
    b.cu_tokens = cu.data();
    const int64_t cache_bytes = c.pages * c.page_stride;
    std::vector<int> seen(b.tokens, 0);
    for (int s = 0; s < seqs; ++s) {
      const KvSeq q = kv_seq(b, s);
      CHECK(q.row >= 0 && q.n >= 0 && q.row + q.n <= b.tokens);
      CHECK(q.context >= 0 && q.context <= b.max_context);
      CHECK(wrong || !q.bad);
      for (int p = 0; p < q.context; p += 1 + r() % 40) {
        const int page = kv_page(c, b, s, p);
        CHECK(page >= -1 && page < c.pages);
        CHECK(wrong || page >= 0);
        if (page < 0) continue;
        const int64_t at = kv_offset(c, page, c.kv_heads - 1, p);
        CHECK(at >= 0 && at + c.slot_stride <= cache_bytes);
      }
    }
    for (int tile : {1, 8, 48, 64}) {  // tiles of rows
      std::vector<int> rows(b.tokens, 0);
      for (int u = 0; u < kv_units(b, tile, 1); ++u) {
        const int s = find(b, u, tile, 1);
        if (s < 0) continue;
        const KvSeq q = kv_seq(b, s);
        const int64_t first = (int64_t)(u - kv_unit_base(b, s, tile, 1)) * tile;
        for (int64_t j = first; j < first + tile && j < q.n; ++j) {
          CHECK(q.row + j >= 0 && q.row + j < b.tokens);
          ++rows[q.row + j];
        }
      }
      if (!wrong)
        for (int i = 0; i < b.tokens; ++i) CHECK(rows[i] == (i < cu.back()));
    }
    // blocks of cache positions
    std::vector<int> rows(b.tokens, 0);
    for (int u = 0; u < kv_units(b, 16, 2); ++u) {
      const int s = find(b, u, 16, 2);
      if (s < 0) continue;
      const KvSeq q = kv_seq(b, s);
      const int first = q.context - q.n > 0 ? q.context - q.n : 0;
      const int64_t start = ((int64_t)(first >> 4) + u - kv_unit_base(b, s, 16, 2)) << 4;
      if (q.bad || !q.n || start >= q.context) continue;
      for (int64_t p = start > first ? start : first; p < start + 16 && p < q.context; ++p) {
        const int64_t row = q.row + q.n - q.context + p;
        CHECK(row >= q.row && row < q.row + q.n);
        ++rows[row];
      }
    }
    if (!wrong)
      for (int i = 0; i < b.tokens; ++i) CHECK(rows[i] == (i < cu.back()));
  }
  // one length for all
  KvBatch b = {};
  b.sequences = 5;
  b.uniform = 3;
  b.tokens = 15;
  for (int s = 0; s <= 5; ++s) CHECK(kv_cu(b, s) == 3 * s);
  // far pages: 64 bits
  KvCache c = {};
  c.pages = 1 << 20;
  c.page_shift = 4;
  c.page_stride = 1 << 20;
  c.slot_stride = 256;
  CHECK(kv_offset(c, (1 << 20) - 1, 0, 15) == ((int64_t)((1 << 20) - 1) << 20) + 15 * 256);
  printf("ok\n");
  return 0;
}
