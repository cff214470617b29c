// CPU test of pair_schedule.h: for many tile counts, sums and pair counts,
// every K block of every tile belongs to exactly one part, a cut tile's parts
// are exactly those that the joining kernel adds, no slot is used twice, and
// the busiest pair stays near an even share.
#include <stdio.h>
#include <stdlib.h>

#include <map>
#include <random>
#include <set>
#include <vector>

#include "pair_schedule.h"

using namespace tnops;

static void fail(const PairSchedule& s, const char* what) {
  fprintf(stderr, "FAIL %s: tiles %d %d k %d %d whole %d %d pairs %d\n", what, s.tiles[0],
          s.tiles[1], s.k[0], s.k[1], s.whole[0], s.whole[1], s.pairs);
  exit(1);
}

static void check(PairSchedule s) {
  planPairs(&s);
  for (int i = 0; i < 2; ++i)
    if (s.whole[i] < 0 || s.whole[i] > s.tiles[i]) fail(s, "whole tiles");
  std::vector<std::vector<char>> seen[2];
  for (int i = 0; i < 2; ++i) seen[i].assign(s.tiles[i], std::vector<char>(s.k[i], 0));
  std::map<std::pair<int, int>, std::set<int>> parts;  // (product, tile) -> slots
  std::set<int> used;
  int64_t busiest = 0, total = 0;
  for (int p = 0; p < s.pairs; ++p) {
    PairWalk walk;
    walk.init(s, p);
    PairWork w;
    int64_t n = 0;
    while (walk.next(s, &w)) {
      if (w.which < 0 || w.which > 1 || w.tile < 0 || w.tile >= s.tiles[w.which] || w.kb0 < 0 ||
          w.kb0 >= w.kb1 || w.kb1 > s.k[w.which])
        fail(s, "a part out of range");
      for (int k = w.kb0; k < w.kb1; ++k)
        if (seen[w.which][w.tile][k]++) fail(s, "a block twice");
      if ((w.slot < 0) != (w.kb0 == 0 && w.kb1 == s.k[w.which])) fail(s, "slot of a whole tile");
      if (w.slot >= 0) {
        if (w.slot > 1 || !used.insert(2 * p + w.slot).second) fail(s, "a slot twice");
        parts[{w.which, w.tile}].insert(2 * p + w.slot);
      }
      n += w.kb1 - w.kb0;
    }
    total += n;
    if (n > busiest) busiest = n;
  }
  for (int i = 0; i < 2; ++i)
    for (auto& t : seen[i])
      for (char c : t)
        if (!c) fail(s, "a block left out");
  for (int p = 0; p < s.pairs; ++p) {
    CutTile c;
    if (!cutTileOf(s, p, &c)) continue;
    auto it = parts.find({c.which, c.tile});
    if (it == parts.end()) fail(s, "joins a tile that is not cut, or twice");
    std::set<int> got;
    for (int q = p; q < s.pairs && s.restStart(q) < c.end; ++q)
      if (cutSlot(s, c, q) >= 0) got.insert(2 * q + cutSlot(s, c, q));
    if (got != it->second) fail(s, "joins other parts than were written");
    parts.erase(it);
  }
  if (!parts.empty()) fail(s, "a cut tile is not joined");
  const int64_t even = (total + s.pairs - 1) / s.pairs;
  if (busiest > even + kCutCost + 1) fail(s, "the busiest pair");
}

int main() {
  for (int pairs : {1, 2, 3, 66, 74})
    for (int a : {0, 1, 2, 27, 73, 74, 75, 96, 300})
      for (int b : {0, 1, 5, 74, 99})
        for (int ka : {1, 2, 12, 36, 393})
          for (int kb : {1, 7, 128})
            if (a + b > 0) check({{a, b}, {ka, kb}, {0, 0}, pairs});
  std::mt19937 rng(7);
  for (int i = 0; i < 3000; ++i) {
    auto r = [&](int n) { return (int)(rng() % n); };
    PairSchedule s{{r(400), r(400)}, {1 + r(500), 1 + r(500)}, {0, 0}, 1 + r(80)};
    if (s.tiles[0] + s.tiles[1] > 0) check(s);
  }
  printf("pair schedule ok\n");
  return 0;
}
