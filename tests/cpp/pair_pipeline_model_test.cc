// pair_pipeline_model_test.cc - threaded CPU model of the synchronisation of
// the CTA-pair products of the training operators, with the kernels' loops and
// parity formulas:
//
//   pair_gemm.cuh   tiles of two halves with one accumulator each, some with
//                   rows in the first half only, sums from one K block to
//                   many, an epilogue that is slower or faster than the sums;
//   panel_gemm.cuh  two accumulators in turn, a panel of A that stays while a
//                   pair goes along n and is loaded again where its range
//                   passes into the next panel, a ring of single operand slots.
//
// An mbarrier has the PTX semantics that the kernels rely on: a phase
// completes when its arrivals and bytes are in, try_wait.parity(p) succeeds
// while the last completed phase has parity p, so that a waiter that misses a
// whole phase waits for good. TMA and MMA units are threads that run their
// queues in order after random delays, a commit arrives once the MMAs before
// it are done.
//
// Checks: the MMA reads what was loaded for it, the epilogue the sums of its
// own tile, every part is stored once, and nobody waits past a bound.
#include <stdio.h>

#include <atomic>
#include <chrono>
#include <condition_variable>
#include <deque>
#include <functional>
#include <mutex>
#include <random>
#include <thread>
#include <vector>

namespace {

struct Barrier {
  std::mutex mu;
  int count = 1, pending = 1;
  long tx = 0;
  unsigned phases = 0;
  void init(int c) { count = pending = c; }
  void update(int arrivals, long bytes) {
    std::lock_guard<std::mutex> l(mu);
    pending -= arrivals;
    tx += bytes;
    if (pending == 0 && tx == 0) {
      ++phases;
      pending = count;
    }
  }
  void arrive() { update(1, 0); }
  void expect(long bytes) { update(1, bytes); }
  void complete(long bytes) { update(0, -bytes); }
  bool passed(unsigned parity) {
    std::lock_guard<std::mutex> l(mu);
    return (phases & 1u) != parity;
  }
};

std::atomic<bool> gStuck{false};

bool wait(Barrier& b, unsigned parity) {
  const auto t0 = std::chrono::steady_clock::now();
  while (!b.passed(parity)) {
    if (gStuck.load()) return false;
    if (std::chrono::steady_clock::now() - t0 > std::chrono::seconds(10)) {
      gStuck = true;
      return false;
    }
    std::this_thread::yield();
  }
  return true;
}

struct Jitter {
  std::mt19937 g;
  explicit Jitter(int seed) : g((unsigned)seed) {}
  void operator()(int maxUs) {
    const int us = maxUs ? (int)(g() % (unsigned)(maxUs + 1)) : 0;
    if (us) std::this_thread::sleep_for(std::chrono::microseconds(us));
  }
};

struct Unit {
  std::mutex mu;
  std::condition_variable cv;
  std::deque<std::function<void()>> q;
  bool stop = false;
  std::thread th;
  Unit(int seed, int maxUs) {
    th = std::thread([this, seed, maxUs] {
      Jitter jitter(seed);
      for (;;) {
        std::function<void()> job;
        {
          std::unique_lock<std::mutex> l(mu);
          cv.wait(l, [this] { return stop || !q.empty(); });
          if (q.empty()) return;
          job = std::move(q.front());
          q.pop_front();
        }
        jitter(maxUs);
        job();
      }
    });
  }
  void push(std::function<void()> f) {
    {
      std::lock_guard<std::mutex> l(mu);
      q.push_back(std::move(f));
    }
    cv.notify_one();
  }
  ~Unit() {
    {
      std::lock_guard<std::mutex> l(mu);
      stop = true;
    }
    cv.notify_one();
    th.join();
  }
};

constexpr int kWarps = 8;

struct Work {
  int kBlocks, halves;
};

// pair_gemm.cuh for one pair. epiUs: delay of an epilogue warp's stores.
bool runPair(const std::vector<Work>& work, int seed, int mmaUs, int epiUs) {
  constexpr int kStages = 4;
  constexpr long kBytes = 16384;
  Barrier full[kStages], empty[2][kStages], accFull[2][2], accEmpty[2];
  for (int h = 0; h < 2; ++h) accEmpty[h].init(2 * kWarps);
  std::atomic<long> stage[2][kStages], acc[2], blocks[2];
  for (auto& c : stage)
    for (auto& x : c) x = -1;
  for (int h = 0; h < 2; ++h) acc[h] = blocks[h] = -1;
  std::atomic<bool> bad{false};
  std::atomic<int> stored{0};
  {
    Unit tma0(seed + 1, 20), tma1(seed + 2, 20), tensor(seed + 3, mmaUs);
    Unit* tma[2] = {&tma0, &tma1};
    std::vector<std::thread> threads;
    for (int r = 0; r < 2; ++r)
      threads.emplace_back([&, r] {
        unsigned g = 0;
        for (size_t t = 0; t < work.size(); ++t)
          for (int kb = 0; kb < work[t].kBlocks; ++kb, ++g) {
            const unsigned s = g % kStages;
            if (!wait(empty[r][s], ((g / kStages) & 1u) ^ 1u)) return;
            const long loads = work[t].halves + 1;
            if (r == 0) full[s].expect(2 * loads * kBytes);
            const long tag = (long)t * 1000 + kb;
            tma[r]->push([&, r, s, tag, loads] {
              stage[r][s] = tag;
              full[s].complete(loads * kBytes);
            });
          }
      });
    threads.emplace_back([&] {
      unsigned g = 0;
      for (size_t t = 0; t < work.size(); ++t) {
        const unsigned fresh = (t & 1u) ^ 1u;
        for (int kb = 0; kb < work[t].kBlocks; ++kb, ++g) {
          const unsigned s = g % kStages;
          if (!wait(full[s], (g / kStages) & 1u)) return;
          for (int h = 0; h < 2; ++h) {
            if (kb == 0 && !wait(accEmpty[h], fresh)) return;
            if (h >= work[t].halves) continue;
            const long tag = (long)t * 1000 + kb;
            tensor.push([&, s, h, t, kb, tag] {
              if (stage[0][s] != tag || stage[1][s] != tag) bad = true;
              if (kb == 0) {
                acc[h] = (long)t;
                blocks[h] = 1;
              } else if (acc[h] != (long)t) {
                bad = true;
              } else {
                blocks[h].fetch_add(1);
              }
            });
          }
          tensor.push([&, s] {
            empty[0][s].arrive();
            empty[1][s].arrive();
          });
        }
        tensor.push([&] {
          for (int h = 0; h < 2; ++h)
            for (int r = 0; r < 2; ++r) accFull[r][h].arrive();
        });
      }
    });
    for (int r = 0; r < 2; ++r)
      for (int w = 0; w < kWarps; ++w)
        threads.emplace_back([&, r, w] {
          Jitter jitter(seed * 31 + r * 17 + w);
          for (size_t t = 0; t < work.size(); ++t)
            for (int h = 0; h < 2; ++h) {
              if (!wait(accFull[r][h], t & 1u)) return;
              if (h < work[t].halves && (acc[h] != (long)t || blocks[h] != work[t].kBlocks))
                bad = true;
              accEmpty[h].arrive();
              jitter(epiUs);
              ++stored;
            }
        });
    for (auto& t : threads) t.join();
  }
  return !gStuck && !bad && stored == (int)work.size() * 2 * 2 * kWarps;
}

// panel_gemm.cuh for one pair: tiles [first, end) of panels of tilesN.
bool runPanel(int first, int end, int tilesN, int kBlocks, int resident, int slots, int seed,
              int epiUs) {
  constexpr long kBytes = 16384;
  std::vector<Barrier> full(slots), empty0(slots), empty1(slots);
  Barrier panelFull, panelEmpty[2], accFull[2][2], accEmpty[2];
  for (int b = 0; b < 2; ++b) accEmpty[b].init(2 * kWarps);
  std::vector<std::atomic<long>> ring(2 * slots), panel(2 * (resident + 1));
  for (auto& x : ring) x = -1;
  for (auto& x : panel) x = -1;
  std::atomic<long> acc[2], blocks[2];
  for (int b = 0; b < 2; ++b) acc[b] = blocks[b] = -1;
  std::atomic<bool> bad{false};
  std::atomic<int> stored{0};
  auto tagOf = [&](bool isA, int t, int kb) {
    return (isA ? 1000000000L + (long)(t / tilesN) * 1000 : (long)t * 1000) + kb;
  };
  {
    Unit tma0(seed + 1, 10), tma1(seed + 2, 10), tensor(seed + 3, 10);
    Unit* tma[2] = {&tma0, &tma1};
    std::vector<std::thread> threads;
    for (int r = 0; r < 2; ++r)
      threads.emplace_back([&, r] {
        unsigned g = 0, panels = 0;
        auto& empty = r ? empty1 : empty0;
        auto stream = [&](long tag) {
          const unsigned s = g % slots;
          if (!wait(empty[s], ((g / slots) & 1u) ^ 1u)) return false;
          if (r == 0) full[s].expect(2 * kBytes);
          tma[r]->push([&, r, s, tag] {
            ring[r * slots + s] = tag;
            full[s].complete(kBytes);
          });
          ++g;
          return true;
        };
        for (int t = first; t < end; ++t) {
          if (t == first || t % tilesN == 0) {
            if (!wait(panelEmpty[r], (panels & 1u) ^ 1u)) return;
            if (r == 0) panelFull.expect(2 * kBytes * resident);
            for (int kb = 0; kb < resident; ++kb) {
              const long tag = tagOf(true, t, kb);
              tma[r]->push([&, r, kb, tag] {
                panel[r * resident + kb] = tag;
                panelFull.complete(kBytes);
              });
            }
            ++panels;
          }
          for (int kb = 0; kb < kBlocks; ++kb) {
            if (kb >= resident && !stream(tagOf(true, t, kb))) return;
            if (!stream(tagOf(false, t, kb))) return;
          }
        }
      });
    threads.emplace_back([&] {
      unsigned g = 0, panels = 0;
      for (int t = first, local = 0; t < end; ++t, ++local) {
        const unsigned b = local & 1u, use = local >> 1;
        if (t == first || t % tilesN == 0) {
          if (!wait(panelFull, panels & 1u)) return;
          ++panels;
        }
        if (!wait(accEmpty[b], (use & 1u) ^ 1u)) return;
        for (int kb = 0; kb < kBlocks; ++kb) {
          int sa = -1;
          if (kb >= resident) {
            sa = (int)(g % slots);
            if (!wait(full[sa], (g / slots) & 1u)) return;
            ++g;
          }
          const int sb = (int)(g % slots);
          if (!wait(full[sb], (g / slots) & 1u)) return;
          ++g;
          const long tagA = tagOf(true, t, kb), tagB = tagOf(false, t, kb);
          tensor.push([&, sa, sb, b, t, kb, tagA, tagB] {
            for (int r = 0; r < 2; ++r)
              if ((sa >= 0 ? ring[r * slots + sa] : panel[r * resident + kb]) != tagA ||
                  ring[r * slots + sb] != tagB)
                bad = true;
            if (kb == 0) {
              acc[b] = t;
              blocks[b] = 1;
            } else if (acc[b] != t) {
              bad = true;
            } else {
              blocks[b].fetch_add(1);
            }
          });
          tensor.push([&, sa, sb] {
            for (auto* e : {&empty0, &empty1}) {
              if (sa >= 0) (*e)[sa].arrive();
              (*e)[sb].arrive();
            }
          });
        }
        const bool leaves = t + 1 == end || (t + 1) % tilesN == 0;
        tensor.push([&, b, leaves] {
          for (int r = 0; r < 2; ++r) {
            accFull[r][b].arrive();
            if (leaves) panelEmpty[r].arrive();
          }
        });
      }
    });
    for (int r = 0; r < 2; ++r)
      for (int w = 0; w < kWarps; ++w)
        threads.emplace_back([&, r, w] {
          Jitter jitter(seed * 29 + r * 13 + w);
          for (int t = first, local = 0; t < end; ++t, ++local) {
            const unsigned b = local & 1u, use = local >> 1;
            if (!wait(accFull[r][b], use & 1u)) return;
            if (acc[b] != t || blocks[b] != kBlocks) bad = true;
            accEmpty[b].arrive();
            jitter(epiUs);
            ++stored;
          }
        });
    for (auto& t : threads) t.join();
  }
  return !gStuck && !bad && stored == (end - first) * 2 * kWarps;
}

}  // namespace

int main() {
  int failed = 0;
  auto report = [&](const char* what, bool ok) {
    printf("%-60s %s\n", what, ok ? "ok" : "FAILED");
    failed += !ok;
  };
  // Short sums behind a slow epilogue: the tensor unit is done with the next
  // tile while the stores of this one still run.
  report("pair: one-half tiles, slow epilogue",
         runPair({{3, 2}, {1, 1}, {1, 1}, {1, 2}, {1, 1}, {2, 1}, {1, 2}, {1, 1}}, 1, 0, 3000));
  for (int seed = 0; seed < 6; ++seed) {
    std::mt19937 g((unsigned)seed);
    std::vector<Work> work;
    for (int i = 0; i < 12; ++i) work.push_back({1 + (int)(g() % 9), 1 + (int)(g() % 2)});
    report("pair: mixed tiles, slow epilogue", !gStuck && runPair(work, seed, 5, 400));
    report("pair: mixed tiles, slow tensor unit", !gStuck && runPair(work, seed, 60, 5));
  }
  for (int seed = 0; seed < 4; ++seed) {
    report("panel: several panels, part resident",
           !gStuck && runPanel(5, 23, 7, 12, 8, 6, seed, 50));
    report("panel: all resident, one tile a panel",
           !gStuck && runPanel(0, 9, 1, 4, 4, 10, seed, 200));
    report("panel: one K block", !gStuck && runPanel(2, 20, 6, 1, 1, 13, seed, 100));
  }
  printf("pair pipelines: %s\n", failed ? "FAIL" : "PASS");
  return failed ? 1 : 0;
}
