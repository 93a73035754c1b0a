// How attention deals out its work: units of rows that share a key/value head, and stretches of the positions they see.
#ifndef AMEM_KV_PARTS_H_
#define AMEM_KV_PARTS_H_

#include "kv_cut.h"
#include "kv_device.h"

namespace amem {

// How a call's rows and positions are dealt out.
struct Parts {
  int stretch;   // positions of a workgroup, a multiple of 64
  int units;
  // Pairs of a unit and a kv head are numbered heads first and the last units first. The first `whole` of them are not cut, each of
  // the others is, into at most `splits` stretches.
  int whole, splits;
  float* sums;   // [pair - whole][split][row][dim]; in multiples of kPartUnit where the cache has 8 bits
  float* stats;  // [pair - whole][split][row]{m, l}, m in units of log 2
};

namespace {

__device__ __forceinline__ void row_range(const KvAttend& a, const KvSeq& q, int token, int& from, int& to) {
  kv_row_range(a.causal, a.window, q, token, from, to);
}

__device__ __forceinline__ bool find_unit(const KvBatch& b, const KvAttend& a, int group, int tile, int index, KvSeq& q, KvUnit& u) {
  int s;
  if (b.cu_tokens) {
    s = find_sequence(b, index, tile, 1, group);
    if (s < 0) return false;
    index -= kv_unit_base(b, s, tile, 1, group);
  } else {
    const int each = (b.uniform * group - 1) / tile + 1;
    s = index / each;
    index -= s * each;
  }
  q = kv_seq(b, s);
  return kv_unit_at(a.causal, a.window, group, tile, s, index, q, u);
}

// The pair and the stretch that workgroup `index` has.
__device__ __forceinline__ void pair_of(const KvCache& c, const Parts& parts, int index, int& unit, int& kvh, int& split) {
  const int cut = parts.units * c.kv_heads - parts.whole;
  split = index < parts.whole ? 0 : (index - parts.whole) / cut;
  const int pair = index < parts.whole ? index : parts.whole + (index - parts.whole) % cut;
  unit = parts.units - 1 - pair / c.kv_heads;
  kvh = pair % c.kv_heads;
}

// Where the part of a pair's first stretch is kept, those of the others behind it; below zero if the pair is not cut.
__device__ __forceinline__ int64_t part_of(const KvCache& c, const Parts& parts, int unit, int kvh) {
  return ((int64_t)(parts.units - 1 - unit) * c.kv_heads + kvh - parts.whole) * parts.splits;
}

inline int units_of(const KvBatch& b, int group, int tile) {
  return b.cu_tokens ? kv_units(b, tile, 1, group) : b.sequences * ((b.uniform * group - 1) / tile + 1);
}

// Sets whole, splits and stretch.
inline void cut_pairs(const Cut& cut, const KvCache& c, int64_t span, bool even, Parts* parts) {
  const CutInto into = cut_last_round(cut, parts->units * c.kv_heads, span, even);
  parts->whole = into.whole;
  parts->splits = into.splits;
  parts->stretch = into.stretch;
}

// Bytes of a call's parts: `rows` of each, their sums, m and l.
inline uint64_t parts_bytes(const Cut& cut, int64_t pairs, int64_t span, int rows, int head_dim) {
  return (uint64_t)most_parts(cut, pairs, span) * rows * (head_dim + 2) * 4;
}

inline uint32_t workgroups(const KvCache& c, const Parts& parts) {
  return (uint32_t)parts.whole + (uint32_t)(parts.units * c.kv_heads - parts.whole) * parts.splits;
}

}  // namespace

// Joins the stretches of every row: kv_attention.hip. `tile`: a unit's rows; `lift`: what the kernel added to m; `sum_unit`: what the sums are multiples of.
hipError_t launch_join(const KvCache& c, const KvBatch& b, const KvAttend& a, const Parts& parts, int tile, float lift, float sum_unit, int head_dim, bool half, hipStream_t stream);

}  // namespace amem
#endif
