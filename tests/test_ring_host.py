"""The steps of a ring of tiles (csrc/ring.cuh) on the host, over barriers made of
threads: what a producer and its consumers do when a tile does not come."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = r"""
#include <atomic>
#include <chrono>
#include <cstdio>
#include <cstdlib>
#include <thread>
#include <vector>
#include "ring.cuh"

constexpr int kStages = 4, kConsumers = 4;
using Clock = std::chrono::steady_clock;

// a barrier that completes its phase at the n-th arrival, as an mbarrier does
struct Bar {
  std::atomic<int> arrivals{0};
  int n = 1;
  void arrive() { ++arrivals; }
  bool done(int parity) const { return (arrivals.load() / n & 1) != parity; }
};
Bar full[kStages], empty_[kStages];
std::atomic<int> aborted{0}, code{0}, in_flight{0}, reports{0};

bool wait(Bar& b, int parity, bool heed) {
  const auto t0 = Clock::now();
  while (!b.done(parity)) {
    if (heed && aborted) return false;
    if (Clock::now() - t0 > std::chrono::milliseconds(100)) return false;
    std::this_thread::yield();
  }
  return true;
}
void give_up() {
  aborted = 1;
  int none = 0;
  code.compare_exchange_strong(none, 6);
  ++reports;
}

int main(int argc, char** argv) {
  const int tiles = std::atoi(argv[1]), lost = std::atoi(argv[2]), slow = std::atoi(argv[3]);
  for (int s = 0; s < kStages; ++s) empty_[s].n = kConsumers;
  std::atomic<int> left_with{-1}, holds[kStages];
  for (auto& h : holds) h = -1;
  std::vector<std::thread> copies;
  std::thread producer([&] {
    int t = 0;
    nd::ring_produce<kStages>(
        [&] { return t < tiles; }, [&](int s, int par) { return wait(empty_[s], par, true); },
        [&](int s) {
          const int tile = t++;
          if (tile == lost) return;       // never comes
          ++in_flight;
          copies.emplace_back([&, s, tile] {
            std::this_thread::sleep_for(std::chrono::milliseconds(slow));
            holds[s] = tile;
            --in_flight;                  // written
            full[s].arrive();
          });
        },
        give_up, [&](int s, int par) { wait(full[s], par, false); });
    left_with = in_flight.load();
  });
  std::vector<int> good(kConsumers, 0), wrong(kConsumers, 0), bad(kConsumers, 0);
  std::vector<std::thread> consumers;
  for (int c = 0; c < kConsumers; ++c)
    consumers.emplace_back([&, c] {
      bool ok = true;
      for (int it = 0; it < tiles; ++it) {
        if (!nd::ring_take<kStages>(ok, it, [&](int s, int par) { return wait(full[s], par, true); }, give_up)) {
          ++bad[c];
          continue;
        }
        ++good[c];
        wrong[c] += holds[it % kStages] != it;
        empty_[it % kStages].arrive();
      }
    });
  const auto t0 = Clock::now();
  for (auto& t : consumers) t.join();
  producer.join();
  const double s = std::chrono::duration<double>(Clock::now() - t0).count();
  for (auto& t : copies) t.join();
  std::printf("%d %d %.3f", code.load(), left_with.load(), s);
  for (int c = 0; c < kConsumers; ++c) std::printf(" %d %d %d", good[c], bad[c], wrong[c]);
  std::printf("\n");
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    cxx = os.environ.get("CXX") or shutil.which("g++")
    if not cxx:
        pytest.skip("no C++ compiler")
    d = tmp_path_factory.mktemp("ring")
    (d / "ring.cpp").write_text(SOURCE)
    subprocess.run([cxx, "-O1", "-std=c++17", "-pthread", "-I", os.path.join(ROOT, "neurodsl_b200", "csrc"),
                    str(d / "ring.cpp"), "-o", str(d / "ring")], check=True)

    def run(tiles, lost=-1, slow=1):
        got = subprocess.run([str(d / "ring"), str(tiles), str(lost), str(slow)], check=True, capture_output=True,
                             text=True, timeout=60).stdout.split()
        code, left, seconds, rest = int(got[0]), int(got[1]), float(got[2]), [int(x) for x in got[3:]]
        return code, left, seconds, [tuple(rest[i:i + 3]) for i in range(0, len(rest), 3)]
    return run


@pytest.mark.parametrize("tiles", [0, 1, 3, 4, 5, 8, 23])
def test_every_tile_comes(program, tiles):
    code, left, _, consumers = program(tiles)
    assert code == 0 and left == 0
    assert consumers == [(tiles, 0, 0)] * 4


@pytest.mark.parametrize("tiles, lost", [(1, 0), (4, 3), (5, 0), (9, 4), (20, 8), (20, 19)])
@pytest.mark.parametrize("slow", [0, 5, 30])
def test_a_tile_that_does_not_come(program, tiles, lost, slow):
    """Reported, whether the producer still runs or has sent everything off; no
    consumer counts a tile from there on; the producer leaves nothing in flight; all
    of it ends within a few limits."""
    code, left, seconds, consumers = program(tiles, lost, slow)
    assert code == 6
    assert left == 0
    assert seconds < 5
    for good, bad, wrong in consumers:
        assert good <= lost and bad == tiles - good and wrong == 0
