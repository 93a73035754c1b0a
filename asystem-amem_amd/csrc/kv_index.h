// Where the rows of a paged key/value cache are: the index arithmetic that the kernels of kv_*.hip share,
// in functions that a host compiler takes too, so that lengths and page numbers out of range can be
// tested without a GPU. Every index that comes from device memory is bounded here before it is used.
#ifndef AMEM_KV_INDEX_H_
#define AMEM_KV_INDEX_H_

#include <stdint.h>

#ifdef __HIPCC__
#define AMEM_HD __host__ __device__ __forceinline__
#else
#define AMEM_HD inline
#endif

namespace amem {

// Strides in bytes (scales: in floats).
struct KvCache {
  uint8_t* k;
  uint8_t* v;
  float* k_scale;
  float* v_scale;
  int64_t page_stride, head_stride, slot_stride;
  int64_t scale_page_stride, scale_head_stride;
  int pages, kv_heads;
  int page_shift;   // log2 of the slots of a page
  int block_shift;  // log2 of the slots that share a scale
};

struct KvBatch {
  const int* page_table;
  const int* context;
  const int* cu_tokens;  // null: every sequence has `uniform` rows
  int64_t table_stride;
  int sequences, table_pages, tokens, uniform;
  int max_context;
};

// A sequence of a call: rows [row, row + n), `context` tokens in the cache; bad: its context is out of range.
struct KvSeq {
  int row, n, context;
  bool bad;
};

AMEM_HD int kv_clamp(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }

AMEM_HD int kv_cu(const KvBatch& b, int s) {  // s in [0, sequences]
  if (!b.cu_tokens) return s * b.uniform;
  return kv_clamp(b.cu_tokens[s], 0, b.tokens);
}

AMEM_HD KvSeq kv_seq(const KvBatch& b, int s) {
  KvSeq q;
  q.row = kv_cu(b, s);
  const int end = kv_cu(b, s + 1);
  q.n = end > q.row ? end - q.row : 0;
  q.context = b.context[s];
  q.bad = q.context < 0 || q.context > b.max_context;  // the host holds max_context to the table's pages
  if (q.bad) q.context = 0;
  return q;
}

// What the page table has for position `p` (0 <= p < context of a sequence that is not bad): to be checked before it is used.
AMEM_HD int kv_table(const KvCache& c, const KvBatch& b, int s, int p) {
  return b.page_table[(int64_t)s * b.table_stride + (p >> c.page_shift)];
}

AMEM_HD int kv_checked(const KvCache& c, int page) { return page >= 0 && page < c.pages ? page : -1; }

// The page that holds position `p`, or -1.
AMEM_HD int kv_page(const KvCache& c, const KvBatch& b, int s, int p) { return kv_checked(c, kv_table(c, b, s, p)); }

// Byte offset of a slot's dims; `page` as kv_page gives it and not -1.
AMEM_HD int64_t kv_offset(const KvCache& c, int page, int head, int p) {
  return (int64_t)page * c.page_stride + (int64_t)head * c.head_stride +
         (int64_t)(p & ((1 << c.page_shift) - 1)) * c.slot_stride;
}

AMEM_HD int64_t kv_scale_offset(const KvCache& c, int page, int head, int p) {
  return (int64_t)page * c.scale_page_stride + (int64_t)head * c.scale_head_stride +
         ((p & ((1 << c.page_shift) - 1)) >> c.block_shift);
}

// Work is handed out in units of `tile` items (`per_row` items a row) without the host knowing the lengths: unit u
// belongs to the last sequence s with kv_unit_base(s) <= u. `spare` units more for each sequence cover what its first and
// last, partial tiles need (1 for tiles that start at its first item, 2 for tiles of its cache positions), so a call has at
// most kv_units() of them and some are empty. The host holds tokens * per_row to 2^27.
AMEM_HD int kv_unit_base(const KvBatch& b, int s, int tile, int spare, int per_row = 1) {
  return (int)((uint32_t)(kv_cu(b, s) * per_row) / (uint32_t)tile) + s * spare;
}
AMEM_HD int kv_units(const KvBatch& b, int tile, int spare, int per_row = 1) {
  return b.tokens * per_row / tile + b.sequences * spare;
}

// A unit of attention's rows: some rows of one sequence (row r is head r % group of new token r / group), and the positions they see.
struct KvUnit {
  int s, first, rows;  // the sequence, the first of its rows, how many
  int lo, to;          // positions that some row sees: [lo, to)
  int from;            // lo, down to a multiple of 64
  int all_from, all_to;  // positions that every row sees
};

// The positions [from, to) that the rows of a new token see.
AMEM_HD void kv_row_range(bool causal, int window, const KvSeq& q, int token, int& from, int& to) {
  const int pos = q.context - q.n + token;
  to = causal && pos + 1 < q.context ? pos + 1 : q.context;
  from = window && pos >= window ? pos - window + 1 : 0;  // any window, and positions below zero, without overflow
}

// Unit `index` of sequence s, `tile` rows long; false if there are no rows, as for an index below zero, which offsets that do not ascend give.
AMEM_HD bool kv_unit_at(bool causal, int window, int group, int tile, int s, int index, const KvSeq& q, KvUnit& u) {
  u.s = s;
  u.first = index * tile;
  u.rows = q.n * group - u.first;
  if (index < 0 || u.rows <= 0) return false;
  if (u.rows > tile) u.rows = tile;
  kv_row_range(causal, window, q, u.first / group, u.lo, u.all_to);
  kv_row_range(causal, window, q, (u.first + u.rows - 1) / group, u.all_from, u.to);
  u.from = u.lo & ~63;
  return true;
}

}  // namespace amem
#endif
