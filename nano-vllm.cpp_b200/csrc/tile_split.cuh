// tile_split.cuh -- an even split of a ragged batch's key tiles over a grid.
//
// A unit is one (sequence, kv head [, row tile]) and has the key tiles of its
// sequence, at least one (a unit without keys still writes its rows), after a
// fixed number of empty places for what a unit costs besides its tiles.  The
// units' places, sequence after sequence, form one line that is cut into equal
// runs of `per` places, one run per CTA: every CTA has the same work however
// ragged the contexts are, a unit whose tiles lie inside a run needs no merge,
// and a run touches at most two units that others share.  (A line of tiles
// alone gave runs of many short units to some CTAs: 8-bit decode of 23 sequences
// of 1 to 9,001 tokens took 47 us; with the places, and merges by whole warps,
// 27.)  A unit's part from the first CTA that has tiles of it is that CTA's
// last, every later one's its first; hence two places for partials per CTA.
// Each CTA finds its run from the context lengths themselves (no host work, so a
// captured launch follows new lengths), every warp for itself (no barrier).
#pragma once

#include "common.cuh"

namespace nvattn {
namespace tilesplit {

// (Places are 32-bit: the launchers refuse a batch whose host bounds allow
// kMaxPlaces or more, and 64-bit divisions cost a short launch half a
// microsecond.)
constexpr long long kMaxPlaces = 1ll << 30;

struct Run {
  int begin, end;  // places of this CTA's run
  int per;         // places per CTA
  int seq;         // sequence that holds `begin`
  int seq_first;   // that sequence's first place
};

// Shape of one sequence: `units` units of `tiles` places each.
struct SeqTiles {
  int units, tiles;
};

// Warp-collective.  shape(s) gives sequence s's SeqTiles; runs have at least
// min_run places (short work then leaves CTAs without any).
template <class Shape>
__device__ __forceinline__ Run find_run(int n_seqs, int cta, int n_ctas, int min_run,
                                        Shape shape) {
  const int lane = threadIdx.x & 31;
  int sum = 0, kept = 0;  // kept: the lane's last sequence's places
  for (int s = lane; s < n_seqs; s += 32) {
    const SeqTiles t = shape(s);
    kept = t.units * t.tiles;
    sum += kept;
  }
  sum = __reduce_add_sync(0xffffffffu, sum);
  Run r;
  r.per = max((int)(((unsigned)sum + n_ctas - 1) / (unsigned)n_ctas), min_run);
  r.seq = 0;
  r.seq_first = 0;
  const long long begin = (long long)cta * r.per;
  r.begin = (int)min(begin, (long long)sum);
  r.end = (int)min(begin + r.per, (long long)sum);
  if (r.begin >= sum) return r;
  int before = 0;
  for (int base = 0; base < n_seqs; base += 32) {
    int mine = kept;  // (one sequence per lane: nothing to read again)
    if (n_seqs > 32) {
      mine = 0;
      if (base + lane < n_seqs) {
        const SeqTiles t = shape(base + lane);
        mine = t.units * t.tiles;
      }
    }
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, before + incl > r.begin);
    if (past != 0) {
      const int l = __ffs(past) - 1;
      r.seq = base + l;
      r.seq_first = before + __shfl_sync(0xffffffffu, incl - mine, l);
      return r;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
  return r;
}

}  // namespace tilesplit
}  // namespace nvattn
