// What one launch holds (host arithmetic, no HIP header: a test compiles it by itself).
#pragma once

namespace lbm {

// HIP takes fewer than 2^32 threads along a grid's dimension: the most workgroups of this many threads.  Kernels whose work may need more
// stride over the rest, or are launched again for it.
constexpr long long grid_most(int threads) { return ((1ll << 32) - 1) / threads; }
// workgroups of a launch that strides over `want` workgroups' work
constexpr unsigned grid_of(long long want, int threads) { return (unsigned)(want < grid_most(threads) ? want : grid_most(threads)); }

}  // namespace lbm
