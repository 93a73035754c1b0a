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
