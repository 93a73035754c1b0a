// How attention deals out its work: units of rows that share a key/value head, and stretches of the positions they see.
#ifndef AMEM_KV_PARTS_H_
#define AMEM_KV_PARTS_H_

#include <algorithm>

#include "kv_device.h"

namespace amem {

// How a call's rows and positions are dealt out.
struct Parts {
  int stretch;   // positions of a workgroup, a multiple of 64
  int units;
  // Pairs of a unit and a kv head are numbered heads first and the last units first. The first `whole` of them are not cut, each of
  // the others is, into at most `splits` stretches.
  int whole, splits;
  float* sums;   // [pair - whole][split][row][dim]
  float* stats;  // [pair - whole][split][row]{m, l}, m in units of log 2
};

namespace {

// A unit: some rows of one sequence (row r is head r % group of new token r / group), and the positions they see.
struct Unit {
  int s, first, rows;  // the sequence, the first of its rows, how many
  int lo, to;          // positions that some row sees: [lo, to)
  int from;            // lo, down to a multiple of 64
  int all_from, all_to;  // positions that every row sees
};

__device__ __forceinline__ void row_range(const KvAttend& a, const KvSeq& q, int token, int& from, int& to) {
  const int pos = q.context - q.n + token;
  to = a.causal && pos + 1 < q.context ? pos + 1 : q.context;
  from = a.window && pos - a.window + 1 > 0 ? pos - a.window + 1 : 0;
}

// Unit `index` of sequence s, `tile` rows long; false if there are no rows.
__device__ __forceinline__ bool unit_at(const KvBatch& b, const KvAttend& a, int group, int tile, int s, int index, const KvSeq& q, Unit& u) {
  u.s = s;
  u.first = index * tile;
  u.rows = q.n * group - u.first;
  if (u.rows <= 0) return false;
  if (u.rows > tile) u.rows = tile;
  row_range(a, q, u.first / group, u.lo, u.all_to);
  row_range(a, q, (u.first + u.rows - 1) / group, u.all_from, u.to);
  u.from = u.lo & ~63;
  return true;
}

__device__ __forceinline__ bool find_unit(const KvBatch& b, const KvAttend& a, int group, int tile, int index, KvSeq& q, Unit& u) {
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
  return unit_at(b, a, group, tile, s, index, q, u);
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

// How pairs are cut. A round is as many workgroups as fit at once; what is cut is the last round, or the only one, where it is not
// full: into as many stretches of the same length as fill some rounds, if they end sooner. Costs are hundredths of positions.
struct Cut {
  int fit;               // workgroups that fit at once, a multiple of the 256 compute units
  int rounds, over;      // that the last round becomes, at most; up to `over` rounds may be overfull, since some pairs are shorter
  int least, step;       // positions of a stretch: about the fewest, and what they are a multiple of
  int base, each, load;  // workgroups take base + each * (those of a compute unit), and at least load * (all of them) / 100
  int fill;              // positions that pairs have on average, in percent of the longest one's
  int start, join;       // positions: what a stretch costs beside its own, and the join
  int part;              // each part's sums, written and read once more
};

// As many stretches as a context is cut into, at most.
inline int most_splits(const Cut& cut, int64_t span) { return (int)std::min<int64_t>((span + cut.least / 2) / cut.least, cut.rounds * cut.fit); }

inline int units_of(const KvBatch& b, int group, int tile) {
  return b.cu_tokens ? kv_units(b, tile, 1, group) : b.sequences * ((b.uniform * group - 1) / tile + 1);
}

// Sets whole, splits and stretch. `even`: pairs see about as many positions each, at most `span`; else the last round is left as
// it is, since the short ones fill it.
inline void cut_last_round(const Cut& cut, int pairs, int64_t span, bool even, Parts* parts) {
  const int last = pairs <= cut.fit ? pairs : even ? pairs % cut.fit : 0, most = most_splits(cut, span);
  auto time = [&](int count, int loads) { return (int64_t)std::max(cut.base + cut.each * ((count + 255) / 256), cut.load * loads / 100); };
  parts->splits = 1;
  int64_t least = time(last, last * cut.fill / 100) * (span + cut.start / 4);
  for (int i = 0; last && i <= cut.rounds + cut.over; ++i) {
    // a compute unit's worth, rounds, and rounds that are overfull
    const int slots = i == 0 ? 256 : i <= cut.rounds ? i * cut.fit : (i - cut.rounds) * cut.fit + last - 1;
    const int splits = std::min(slots / last, most);
    if (splits < 2) continue;
    const int count = last * (100 + (splits - 1) * cut.fill) / 100, rest = count % cut.fit;
    const int64_t all = count / cut.fit * time(cut.fit, cut.fit) + (rest ? time(rest, rest) : 0);
    const int64_t cost = all * (span / splits + cut.start) + 100 * (int64_t)cut.join + (int64_t)count * cut.part;
    if (cost >= least) continue;
    least = cost;
    parts->splits = splits;
  }
  parts->whole = parts->splits > 1 ? pairs - last : pairs;
  parts->stretch = (int)(((span + parts->splits - 1) / parts->splits + cut.step - 1) / cut.step * cut.step);
}

// Bytes of the parts of a call, for any mask.
inline uint64_t parts_bytes(const Cut& cut, int64_t pairs, int64_t span, int rows, int head_dim) {
  const int64_t splits = most_splits(cut, span);
  return splits < 2 ? 0 : (uint64_t)(std::min<int64_t>(std::min<int64_t>(pairs, cut.fit) * splits, cut.rounds * cut.fit) * rows) * (head_dim + 2) * 4;
}

inline uint32_t workgroups(const KvCache& c, const Parts& parts) {
  return (uint32_t)parts.whole + (uint32_t)(parts.units * c.kv_heads - parts.whole) * parts.splits;
}

}  // namespace

// Joins the stretches of every row: kv_attention.hip. `tile`: a unit's rows; `lift`: what the kernel added to m.
hipError_t launch_join(const KvCache& c, const KvBatch& b, const KvAttend& a, const Parts& parts, int tile, float lift, int head_dim, bool half, hipStream_t stream);

}  // namespace amem
#endif
