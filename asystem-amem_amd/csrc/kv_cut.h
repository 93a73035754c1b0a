// Into how many stretches the positions of attention's pairs (of a unit of rows and a key/value head) are cut, on the host.
#ifndef AMEM_KV_CUT_H_
#define AMEM_KV_CUT_H_

#include <stdint.h>

#include <algorithm>

namespace amem {

// How pairs are cut. A round is as many workgroups as fit at once; what is cut is the last round, or the only one, where it is not
// full: into as many stretches of the same length as fill some rounds, if they end sooner. Costs are hundredths of positions.
struct Cut {
  int fit;               // workgroups that fit at once, a multiple of the 256 compute units
  int rounds, over;      // that the last round becomes, at most; up to `over` rounds may be overfull, since some pairs are shorter
  int least, step;       // positions of a stretch: about the fewest, and what they are a multiple of; up to 512 of them: of `least`
  int base, each, load;  // workgroups take base + each * (those of a compute unit), and at least load * (all of them) / 100
  int fill;              // positions that pairs have on average, in percent of the longest one's
  int start, join;       // positions: what a stretch costs beside its own, and the join
  int part;              // each part's sums, written and read once more
  int shorter = 0;       // positions: what is shorter is not cut
};

// Few rows, `blocks` of 16 of them. Workgroups are bound by what a compute unit can load, or all of them by the memory. The figures are fitted to times of 25
// calls with 1 to 32 stretches (8 to 512 pairs, contexts of 2000 to 131072, equal and not), 4 % above the best on average. Uncut, and
// cut (us): 128 dims of e4m3, 33 sequences of 1000 to 4000 positions 50 and 44; 65 of 4000 126 and 102; 3 of 30000 270 and 40.
inline Cut cut_of_few(int head_dim, bool eight, int blocks) {
  const int fit = head_dim == 256 && (!eight || blocks > 1) ? 256 : head_dim == 64 && !eight && blocks == 1 ? 768 : 512;
  const int bytes = head_dim * (eight ? 2 : 4);  // of a position
  // Stretches of what four waves take at once: with 256 everywhere a token of 1000 positions takes 10.4 us instead of 9.7, 16.6 instead of 14.0 with 256
  // dims in 16 bits; multiples of 256 for longer stretches: 24 tokens of 4000 positions 45 us, and 49 in multiples of 128.
  // One token of 256 positions takes 6.9 us uncut and 8.4 cut, of 300 9.0 and 9.5, of 500 10.4 in two stretches and 9.2 in four.
  const int least = head_dim == 64 && eight && blocks == 1 ? 256 : 128;
  return {fit, 4, 2, least, 256, 37, 39, 33, 79, 5500 / bytes, 12000 / bytes, 34 * blocks * (head_dim + 2) / bytes, 384};
}

// Many rows, `rows` of a unit. Two workgroups of a compute unit take 4/3 of the time of one, three 5/3; a part of 128 rows costs about a position's work
// once all compute units write theirs. Uncut, and cut (us): 32 heads over 8, 128 dims, 16 bits, 1200 rows of 8192 positions 254 and
// 226; 4500 of 16384 1262 and 1062; 256 dims, 8 bits, 1100 rows of 16000 positions 1290 and 674.
inline Cut cut_of_many(int rows, int fit) { return {fit, 2, 0, 512, 64, 66, 33, 0, 100, 0, 150, rows * 100 / 128}; }

// The first `whole` pairs stay whole, each of the others becomes at most `splits` stretches of `stretch` positions.
struct CutInto {
  int whole, splits, stretch;
};

// As many stretches as a context is cut into, at most.
inline int most_splits(const Cut& cut, int64_t span) {
  return span < cut.shorter ? 1 : (int)std::min<int64_t>((span + cut.least / 2) / cut.least, cut.rounds * cut.fit);
}

// `even`: pairs see about as many positions each, at most `span`; else the last round is left as it is, since the short ones fill it.
inline CutInto cut_last_round(const Cut& cut, int pairs, int64_t span, bool even) {
  const int last = pairs <= cut.fit ? pairs : even ? pairs % cut.fit : 0, most = most_splits(cut, span);
  auto time = [&](int count, int loads) { return (int64_t)std::max(cut.base + cut.each * ((count + 255) / 256), cut.load * loads / 100); };
  CutInto into = {pairs, 1, 0};
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
    const int64_t length = (span + splits - 1) / splits;
    const int step = length <= 512 ? std::min(cut.least, cut.step) : cut.step;
    into = {pairs - last, splits, (int)((length + step - 1) / step * step)};
  }
  return into;
}

// Parts of a call, at most, whatever its mask (which only shortens the span).
inline int64_t most_parts(const Cut& cut, int64_t pairs, int64_t span) {
  const int64_t splits = most_splits(cut, span);
  return splits < 2 ? 0 : std::min<int64_t>(std::min<int64_t>(pairs, cut.fit) * splits, cut.rounds * cut.fit);
}

}  // namespace amem
#endif
