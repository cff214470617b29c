// pair_schedule.h - which CTA pair computes which part of the products of a
// launch (pair_gemm.cuh): shared by the kernels, their launchers and a CPU
// test.
//
// The tiles of the launch's one or two products lie one product after the
// other; a tile of product i is a sum of k[i] blocks. Whole tiles go to the
// pairs in turn (tile t to pair t % pairs): neighbouring pairs then read the
// same rows of an operand at the same time. When the last round of that would
// leave pairs idle for long, the tiles after the last full rounds (the "rest")
// are laid out as one line of K blocks and cut evenly: pair p takes blocks
// [U p / pairs, U (p + 1) / pairs). A pair's share of a cut tile goes to one of
// its two slots of partial sums (the first part of its range to slot 0, a
// later one to slot 1: a range can cut a tile only at its two ends), and a
// second kernel adds the parts of each cut tile in pair order.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define TNOPS_HD __host__ __device__ __forceinline__
#else
#define TNOPS_HD inline
#endif

namespace tnops {

struct PairSchedule {
  int tiles[2];  // of each product
  int k[2];      // K blocks of a tile
  int whole[2];  // tiles that are not part of the rest (the first ones)
  int pairs;

  TNOPS_HD int restTiles(int i) const { return tiles[i] - whole[i]; }
  TNOPS_HD int64_t restBlocks() const {
    return (int64_t)restTiles(0) * k[0] + (int64_t)restTiles(1) * k[1];
  }
  TNOPS_HD int64_t restStart(int p) const { return restBlocks() * p / pairs; }
};

// A part of a tile: K blocks [kb0, kb1) of `tile` of product `which`; slot -1
// for a whole tile.
struct PairWork {
  int which, tile, kb0, kb1, slot;
};

// The rest's tile that holds block u of the line, and the line's first block
// of that tile.
TNOPS_HD void restTileAt(const PairSchedule& s, int64_t u, int* which, int* tile, int64_t* first) {
  const int64_t line0 = (int64_t)s.restTiles(0) * s.k[0];
  *which = u >= line0;
  const int64_t v = *which ? u - line0 : u;
  const int k = s.k[*which];
  const int64_t t = v / k;
  *tile = s.whole[*which] + (int)t;
  *first = (*which ? line0 : 0) + t * k;
}

// Walks a pair's parts in order.
struct PairWalk {
  int t;          // next whole tile, counted over both products
  int64_t u, end; // next block of the rest, and the end of this pair's range
  bool started;   // some of the rest was handed out already

  TNOPS_HD void init(const PairSchedule& s, int pair) {
    t = pair;
    u = s.restStart(pair);
    end = s.restStart(pair + 1);
    started = false;
  }
  TNOPS_HD bool next(const PairSchedule& s, PairWork* w) {
    if (t < s.whole[0] + s.whole[1]) {
      w->which = t >= s.whole[0];
      w->tile = w->which ? t - s.whole[0] : t;
      w->kb0 = 0;
      w->kb1 = s.k[w->which];
      w->slot = -1;
      t += s.pairs;
      return true;
    }
    if (u >= end) return false;
    int64_t first;
    restTileAt(s, u, &w->which, &w->tile, &first);
    const int k = s.k[w->which];
    w->kb0 = (int)(u - first);
    w->kb1 = (int)(end - first < k ? end - first : k);
    w->slot = w->kb0 == 0 && w->kb1 == k ? -1 : started ? 1 : 0;
    started = true;
    u = first + w->kb1;
    return true;
  }
};

// The cut tile that begins with pair `p`'s part: false when pair p's range does
// not end inside a tile, or its tile began with an earlier pair's part.
// `slotOf` then gives the slot of each later pair's part.
struct CutTile {
  int which, tile;
  int64_t first, end;  // the tile's blocks in the line
};
TNOPS_HD bool cutTileOf(const PairSchedule& s, int p, CutTile* c) {
  if (p + 1 >= s.pairs) return false;
  const int64_t b = s.restStart(p + 1);
  if (b <= 0 || b >= s.restBlocks() || b == s.restStart(p)) return false;
  restTileAt(s, b, &c->which, &c->tile, &c->first);
  c->end = c->first + s.k[c->which];
  if (c->first == b) return false;                // a border between tiles
  return s.restStart(p) <= c->first;
}
// Pair q's part of the cut tile: its slot, or -1 when it has none.
TNOPS_HD int cutSlot(const PairSchedule& s, const CutTile& c, int q) {
  const int64_t a = s.restStart(q), b = s.restStart(q + 1);
  if (a >= c.end || b <= c.first || a == b) return -1;
  return a >= c.first ? 0 : 1;
}

// Times of the choice below, in K blocks (a block of a 256 x 256 tile takes
// about 0.3 us): what writing and adding the cut tiles' parts costs.
constexpr int kCutCost = 32;

// Fills whole[]: everything in turn, or full rounds in turn and the rest cut,
// whichever takes fewer blocks on the busiest pair. A tile that is longer than
// a pair's even share is left to the rest entirely.
inline void planPairs(PairSchedule* s) {
  const int64_t total = (int64_t)s->tiles[0] * s->k[0] + (int64_t)s->tiles[1] * s->k[1];
  int64_t busiest = 0;  // in turn
  for (int p = 0; p < s->pairs; ++p) {
    int64_t n = 0;
    for (int i = 0, at = 0; i < 2; at += s->tiles[i], ++i) {
      // Tiles at, at + 1, ... of which pair p has those congruent to p.
      const int before = (at - p + s->pairs - 1) / s->pairs;
      const int upTo = (at + s->tiles[i] - p + s->pairs - 1) / s->pairs;
      n += (int64_t)((upTo > 0 ? upTo : 0) - (before > 0 ? before : 0)) * s->k[i];
    }
    if (n > busiest) busiest = n;
  }
  s->whole[0] = s->tiles[0];
  s->whole[1] = s->tiles[1];
  const int64_t even = (total + s->pairs - 1) / s->pairs;
  if (busiest <= even + kCutCost) return;
  int64_t left = even;
  for (int i = 0; i < 2; ++i) {
    if (s->tiles[i] == 0) continue;
    int64_t rounds = s->tiles[i] / s->pairs;
    if (rounds > left / s->k[i]) rounds = left / s->k[i];
    s->whole[i] = (int)rounds * s->pairs;
    left -= rounds * s->k[i];
  }
}

}  // namespace tnops
