// pair_schedule.h - which CTA pair computes which part of the products of a
// launch (pair_gemm.cuh): shared by the kernels, their launchers and a CPU
// test.
//
// A launch has one or two products; a tile of product i is a sum of k[i] K
// blocks, cut into split[i] even parts ("units"; 1: whole tiles). Product 0's
// units are the longer ones and go to the pairs in turn, unit u to pair
// u % pairs. Where that leaves `extra` pairs with one more of them, the other
// pairs begin product 1 with `early` rounds among themselves, and the rest of
// it goes round all pairs, first to those that then have less behind them.
// Pairs that work at the same time so have neighbouring units, which read the
// same rows of an operand in the same order: one read from memory serves them
// all. (An even cut of the K blocks over the pairs, which also keeps all of
// them busy, lets every pair read at a place of its own: with tiles of 256 x 256
// the two products of a 65536 x 1024 x 4096 layer took 995 us that way and 830
// us in turns; tiles of 512 x 256, in turns, take 740.)
//
// Units of a cut tile leave partial sums, one slot per unit, which a second
// kernel adds in the order of the sum.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define TNOPS_HD __host__ __device__ __forceinline__
#else
#define TNOPS_HD inline
#endif

namespace tnops {

struct PairSchedule {
  int tiles[2];  // of each product (0: no such product)
  int k[2];      // K blocks of a tile
  int split[2];  // parts of a tile
  int pairs;
  int extra, early;  // pairs with one more unit of product 0; early rounds
  int lateFirst;     // the late rounds of product 1 begin with this pair

  TNOPS_HD int units(int i) const { return tiles[i] * split[i]; }
  TNOPS_HD int others() const { return pairs - extra; }
  // First slot of product i.
  TNOPS_HD int slotBase(int i) const { return i == 1 && split[0] > 1 ? units(0) : 0; }
  TNOPS_HD int slots() const {
    return (split[0] > 1 ? units(0) : 0) + (split[1] > 1 ? units(1) : 0);
  }
};

// K blocks [kb0, kb1) of `tile` of product `which`; slot -1 for a whole tile.
struct PairWork {
  int which, tile, kb0, kb1, slot;
};

// Part s of a tile's sum starts at K block k s / split.
TNOPS_HD PairWork pairUnit(const PairSchedule& s, int which, int unit) {
  const int part = unit / s.tiles[which], n = s.split[which], k = s.k[which];
  PairWork w;
  w.which = which;
  w.tile = unit - part * s.tiles[which];
  w.kb0 = (int)((int64_t)k * part / n);
  w.kb1 = (int)((int64_t)k * (part + 1) / n);
  w.slot = n > 1 ? s.slotBase(which) + unit : -1;
  return w;
}

// Walks a pair's units in order.
struct PairWalk {
  int first;          // next unit of product 0
  int early, earlyEnd;
  int late;           // next unit of product 1 in the late rounds

  TNOPS_HD void init(const PairSchedule& s, int pair) {
    first = pair;
    early = pair >= s.extra ? pair - s.extra : 0;
    earlyEnd = pair >= s.extra ? s.others() * s.early : 0;
    const int turn = pair - s.lateFirst;
    late = s.others() * s.early + (turn < 0 ? turn + s.pairs : turn);
  }
  TNOPS_HD bool next(const PairSchedule& s, PairWork* w) {
    if (first < s.units(0)) {
      *w = pairUnit(s, 0, first);
      first += s.pairs;
      return true;
    }
    if (early < earlyEnd) {
      *w = pairUnit(s, 1, early);
      early += s.others();
      return true;
    }
    if (late < s.units(1)) {
      *w = pairUnit(s, 1, late);
      late += s.pairs;
      return true;
    }
    return false;
  }
};

// The schedule for given splits, and the K blocks of its busiest pair.
inline int planRounds(PairSchedule* s) {
  const int len0 = (s->k[0] + s->split[0] - 1) / s->split[0];
  const int len1 = (s->k[1] + s->split[1] - 1) / s->split[1];
  s->extra = s->units(0) % s->pairs;
  s->early = 0;
  s->lateFirst = 0;
  if (s->extra > 0 && s->units(1) > 0) {
    const int most = s->units(1) / s->others();
    s->early = (len0 + len1 / 2) / len1;
    if (s->early > most) s->early = most;
    if (s->early * len1 < len0) s->lateFirst = s->extra;
  }
  // The late rounds give most to the first pair of their turn; the busiest
  // pair is the first in turn among those with an extra unit or among the
  // others.
  const int rounds0 = s->units(0) / s->pairs;
  const int late = s->units(1) - s->others() * s->early;
  auto lateOf = [&](int turn) { return turn < late ? (late - turn + s->pairs - 1) / s->pairs : 0; };
  const int turnExtra = s->lateFirst == 0 ? 0 : s->others();
  const int turnOther = s->lateFirst == 0 ? s->extra : 0;
  const int other = s->early * len1 + lateOf(turnOther) * len1;
  const int extra = s->extra > 0 ? len0 + lateOf(turnExtra) * len1 : 0;
  return rounds0 * len0 + (extra > other ? extra : other);
}

// Plans the launch: sums stay whole, or with `cut` the longer product's are
// split in 2 to kMaxSplit where the busiest pair gains more than the partial
// sums cost. A K block of a 512 x 256 tile takes about 0.55 us; partial sums
// cost one more launch (about 4 us) and about 0.26 us per slot (512 KiB written
// and read).
constexpr int kMaxSplit = 8;
constexpr int kSplitSlots = 148;
inline void planPairs(PairSchedule* s, bool cut) {
  s->split[0] = s->split[1] = 1;
  int best = planRounds(s);
  if (!cut) return;
  PairSchedule t = *s;
  for (int n = 2; n <= kMaxSplit && t.tiles[0] * n <= kSplitSlots; ++n) {
    if (t.k[0] < 8 * n) break;  // at least 8 K blocks a unit
    t.split[0] = n;
    if ((t.k[0] + n - 1) / n < t.k[1] && t.tiles[1] > 0) break;  // product 0's stay the longer
    const int cost = planRounds(&t) + 7 + t.slots() / 2;
    if (cost < best) {
      best = cost;
      *s = t;
    }
  }
}

}  // namespace tnops
