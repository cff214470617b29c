// CPU test of pair_schedule.h: for many tile counts, sums and pair counts,
// every K block of every tile belongs to exactly one unit, a cut tile's units
// fill its slots in the order of the sum, no slot is used twice, and the
// busiest pair has what the plan says and at most two long units more than an
// even share.
#include <stdio.h>
#include <stdlib.h>

#include <random>
#include <set>
#include <vector>

#include "pair_schedule.h"

using namespace tnops;

static void fail(const PairSchedule& s, const char* what) {
  fprintf(stderr, "FAIL %s: tiles %d %d k %d %d split %d %d pairs %d extra %d early %d late %d\n",
          what, s.tiles[0], s.tiles[1], s.k[0], s.k[1], s.split[0], s.split[1], s.pairs, s.extra,
          s.early, s.lateFirst);
  exit(1);
}

static void walk(PairSchedule s) {
  const int planned = planRounds(&s);
  std::vector<std::vector<char>> seen[2];
  for (int i = 0; i < 2; ++i) seen[i].assign(s.tiles[i], std::vector<char>(s.k[i], 0));
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
        fail(s, "a unit out of range");
      for (int k = w.kb0; k < w.kb1; ++k)
        if (seen[w.which][w.tile][k]++) fail(s, "a block twice");
      if ((w.slot < 0) != (s.split[w.which] == 1)) fail(s, "slot of a whole tile");
      if (w.slot >= 0) {
        if (w.slot >= s.slots() || !used.insert(w.slot).second) fail(s, "a slot twice");
        const int part = (w.slot - s.slotBase(w.which)) / s.tiles[w.which];
        if ((w.slot - s.slotBase(w.which)) % s.tiles[w.which] != w.tile ||
            w.kb0 != (int64_t)s.k[w.which] * part / s.split[w.which])
          fail(s, "a slot of another part");
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
  if ((int)used.size() != s.slots()) fail(s, "an empty slot");
  // Units of a split sum differ by one block, which the plan rounds up.
  if (busiest > planned) fail(s, "the plan's busiest pair");
  const int64_t even = (total + s.pairs - 1) / s.pairs;
  const int64_t len0 = (s.k[0] + s.split[0] - 1) / s.split[0];
  const int64_t len1 = s.tiles[1] ? (s.k[1] + s.split[1] - 1) / s.split[1] : 0;
  const int64_t unit = len0 > len1 ? len0 : len1;
  const int64_t rounds = s.units(0) / s.pairs + 1 + (s.units(1) + s.pairs - 1) / s.pairs + s.early;
  if (planned > even + 2 * unit + rounds) fail(s, "the busiest pair");
}

static void check(PairSchedule s) {
  for (int cut : {0, 1}) {
    PairSchedule t = s;
    planPairs(&t, cut != 0);
    if (!cut && (t.split[0] != 1 || t.split[1] != 1)) fail(t, "cut");
    if (t.split[0] > kMaxSplit || t.slots() > kSplitSlots) fail(t, "too many slots");
    walk(t);
  }
  for (int n : {2, 3, 5})  // any split
    if (s.k[0] >= n && s.k[1] >= n) {
      PairSchedule t = s;
      t.split[0] = n;
      t.split[1] = 1;
      walk(t);
      t.split[1] = n;
      walk(t);
    }
}

int main() {
  for (int pairs : {1, 2, 3, 66, 74})
    for (int a : {1, 2, 27, 73, 74, 75, 96, 300})
      for (int b : {0, 1, 5, 74, 99})
        for (int ka : {12, 36, 393})
          for (int kb : {1, 7, 12})
            check({{a, b}, {ka, kb}, {1, 1}, pairs, 0, 0, 0});
  std::mt19937 rng(7);
  for (int i = 0; i < 3000; ++i) {
    auto r = [&](int n) { return (int)(rng() % n); };
    const int ka = 1 + r(500);
    check({{1 + r(400), r(400)}, {ka, 1 + r(ka)}, {1, 1}, 1 + r(80), 0, 0, 0});
  }
  printf("pair schedule ok\n");
  return 0;
}
