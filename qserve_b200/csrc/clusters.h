// qserve_b200 -- how many blocks a cluster gets, by the places that the device has for clusters of each size.  Host only, without CUDA.
#pragma once
#include <cmath>

namespace qs {
namespace paged {

// Clusters of so many blocks that run at once: what the device says, which may be none (groups of fewer multiprocessors, a part of the device) for all but single blocks.
// Where it says nothing, as many as its multiprocessors hold, of the sizes that every device launches.
constexpr int places_of(bool said, int places, int sms, int blocks) {
  if (said && (places > 0 || blocks > 1)) return places > 0 ? places : 0;
  if (blocks > 8) return 0;
  return sms / blocks > 0 ? sms / blocks : 1;
}

// Blocks of each of `clusters` clusters: the most, up to `most`, of which all find places at once; one where no size has so many.
template <typename Places>
int most_blocks_at_once(Places places, int most, long long clusters) {
  int blocks = most;
  while (blocks > 1 && (places(blocks) <= 0 || places(blocks) < clusters)) --blocks;
  return blocks;
}

// Blocks of a cluster whose `warps` warps each share out the half pages of a sequence and kv head: rounds of as many clusters as run at once (two blocks on a
// multiprocessor); 5 us ahead of and behind a warp's half pages, which come one after the other, slower where two blocks share a multiprocessor; a cluster's join.  Of 63
// sizes (1 to 64 sequences of 500 to 16000 positions, 4 rows, INT4, 32 heads over 8) the choice is within 4.5 % of the best.  (us, of one, two, four, eight, sixteen
// blocks: one sequence of 500 8.3, 8.2, 7.0, 6.7, 7.6; 10 of 2000 28.9, 20.3, 21.5, 26.6, 45, but of three 16.2; one of 16000 135, 72, 40, 26, 20; 64 of 2000 63, 74,
// 93, 146.)  Sizes without a place are none.
template <typename Places>
int fastest_blocks(Places places, int most, int warps, long long clusters, int halves) {
  int chosen = 1;
  float best = 3.0e38f;
  for (int n = 1; n <= most && (n == 1 || warps * (n - 1) < halves); ++n) {
    const int held = places(n), turns = ((halves + n - 1) / n + warps - 1) / warps;
    if (held <= 0) continue;
    const float rounds = std::fmax(1.f, clusters / static_cast<float>(held));
    const float shared = std::fmin(1.f, std::fmax(0.f, 2.f * clusters / held - 1.f));  // multiprocessors with two blocks
    const float time = 0.5f * (std::ceil(rounds) + rounds) * (5.f + (n > 1 ? 0.5f + 0.1f * n : 0.f) + turns * (1.05f + 0.2f * std::sqrt(shared)));
    if (time >= best) continue;
    best = time;
    chosen = n;
  }
  return chosen;
}

}  // namespace paged
}  // namespace qs
