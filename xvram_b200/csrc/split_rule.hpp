// split_rule.hpp -- how many CTAs of a cluster share a tile's K in the few-rows tensor-core
// kernel (feed_split.cuh), and the table of cluster capacities the rule reads.  Host code
// without CUDA, so that a test can run it with failing queries.
#pragma once

#include <algorithm>
#include <atomic>

namespace xvram::feed {

// How many clusters of 2, 4 or 8 CTAs of ONE kernel a device runs at once, asked once per device and
// size.  A query that fails is not kept: the next call asks again.
class CapacityTable {
public:
  // CTAs of clusters of `size`, 0 when none fits.  query(&clusters) returns 0 or an error, which is
  // returned.
  template <class Query>
  int ctas(int device, int size, long long* out, const Query& query) {
    *out = 0;
    if (device < 0 || device >= 64)
      return 0;
    std::atomic<int>& slot = known_[device][size == 2 ? 0 : size == 4 ? 1 : 2];
    int clusters = slot.load(std::memory_order_relaxed) - 1;
    if (clusters < 0) {
      if (const int e = query(&clusters))
        return e;
      clusters = std::max(clusters, 0);
      slot.store(clusters + 1, std::memory_order_relaxed); // 0: not asked yet
    }
    *out = static_cast<long long>(clusters) * size;
    return 0;
  }

private:
  std::atomic<int> known_[64][3] = {};
};

struct Split {
  int splits = 0; // 0: no size fits
  double us = 0;
};

// The cluster size with the least estimated time, and that time in us: a stage takes 0.75 when all SMs
// read from HBM and at least 0.45 (one SM's rate); a wave of CTAs 2.5 to start, joining 1.  Clusters
// fit an SM count that the hardware's grouping of SMs limits.  What a CTA holds of a stage for
// its whole K range (held_bytes; 0 for nothing) has to fit into held_most, whatever the time.
// capacity(size, &ctas) returns 0 or an error, which is returned.
template <class Capacity>
int cheapest_split(long long tiles, int k_tiles, long long sms, int held_bytes, int held_most,
                   const Capacity& capacity, Split* best) {
  *best = Split{};
  for (int s = 1; s <= 8 && s <= k_tiles; s *= 2) {
    const long long ctas = tiles * s, stages = (k_tiles + s - 1) / s;
    long long cap = sms;
    if (s > 1)
      if (const int e = capacity(s, &cap))
        return e;
    if (cap < s || stages * held_bytes > held_most)
      continue;
    const double stage_us =
        std::max(0.45, 0.75 * static_cast<double>(std::min(ctas, cap)) / static_cast<double>(sms));
    const double t =
        static_cast<double>((ctas + cap - 1) / cap) * (2.5 + stage_us * static_cast<double>(stages)) +
        (s > 1 ? 1.0 : 0.0);
    if (best->splits == 0 || t < best->us)
      *best = {s, t};
  }
  return 0;
}

} // namespace xvram::feed
