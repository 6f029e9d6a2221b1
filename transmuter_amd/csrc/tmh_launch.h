// How work is cut into launches: whole numbers only, on the host (whose tests go over it).
#pragma once

#include <algorithm>
#include <cstdint>

namespace tmh {

// The most things of `pieces` pieces each that one launch takes, whose workgroups of `threads` threads take `per` pieces
// each: HIP takes fewer than 2^32 threads in a dimension of a grid. (Things of one piece fill whole workgroups.)
constexpr int64_t most_a_launch(int threads, int64_t per, int64_t pieces) {
  return ((int64_t{1} << 32) - 1) / threads * per / pieces;
}

// Calls launch(first, count) for runs of up to `most` of `all` things.
template <typename Launch>
void in_launches(int64_t all, int64_t most, Launch launch) {
  for (int64_t first = 0; first < all; first += most) launch(first, std::min(most, all - first));
}

}  // namespace tmh
