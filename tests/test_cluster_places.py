"""How many blocks a cluster gets (csrc/clusters.h): sizes that the device has no place for are never chosen, for a launch of one fails."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qserve_b200", "csrc")
PROGRAM = r"""
#include <cstdio>
#include <initializer_list>
#include "clusters.h"
using namespace qs::paged;
static_assert(places_of(true, 7, 148, 16) == 7 && places_of(true, 148, 148, 1) == 148, "what the device says");
static_assert(places_of(true, 0, 148, 16) == 0 && places_of(true, 0, 148, 2) == 0 && places_of(true, 0, 148, 1) == 148, "none, but single blocks always run");
static_assert(places_of(false, 0, 148, 16) == 0 && places_of(false, 0, 148, 9) == 0 && places_of(false, 0, 148, 8) == 18 && places_of(false, 0, 4, 8) == 1, "it says nothing");
int main() {
  for (int most : {1, 2, 3, 4, 7, 8, 12, 16})      // the largest cluster that there is a place for
    for (int sms : {20, 74, 132, 148}) {
      auto places = [&](int n) { return places_of(true, n <= most ? sms / n : 0, sms, n); };
      for (long long clusters = 1; clusters <= 400; ++clusters) {
        const int all = most_blocks_at_once(places, 16, clusters);
        if (all < 1 || all > most || (all > 1 && places(all) < clusters)) return std::printf("%d of %d: %d for %lld\n", most, sms, all, clusters), 1;
        if (all < 16 && all < most && places(all + 1) >= clusters) return std::printf("%d of %d: %d for %lld, though one more would run\n", most, sms, all, clusters), 1;
        for (int halves : {1, 2, 16, 63, 250, 4000, 1 << 25}) {
          const int n = fastest_blocks(places, 16, 4, clusters, halves);
          if (n < 1 || n > most) return std::printf("%d of %d: %d for %lld of %d\n", most, sms, n, clusters, halves), 1;
        }
      }
    }
  // sizes between that have none
  auto holes = [](int n) { return n == 16 || n == 8 || n == 3 ? 0 : 148 / n; };
  for (long long clusters = 1; clusters <= 400; ++clusters) {
    const int all = most_blocks_at_once(holes, 16, clusters), n = fastest_blocks(holes, 16, 4, clusters, 500);
    if (holes(all) == 0 || holes(n) == 0) return std::printf("%d, %d for %lld\n", all, n, clusters), 1;
  }
  if (most_blocks_at_once([](int) { return 0; }, 16, 0) != 1) return 1;
  return 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")
def test_sizes_without_a_place(tmp_path):
    src, out = tmp_path / "places.cpp", tmp_path / "places"
    src.write_text(PROGRAM)
    built = subprocess.run(["g++", "-std=c++17", "-O1", "-I", CSRC, str(src), "-o", str(out)], capture_output=True, text=True)
    assert built.returncode == 0, built.stderr
    run = subprocess.run([str(out)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0, run.stdout
