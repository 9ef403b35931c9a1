// The workspace of the attention on 8-bit pages: a status word, arrival counters (zero between launches), partial sums.
#pragma once

#include "common.cuh"

namespace leankv {
namespace bytes {

constexpr int kTimedOut = 1, kBadPage = 2, kTooMany = 4;            // status bits
constexpr int kStatusWords = 64;
constexpr int kCounters = 2048;
constexpr size_t kPartialsAt = 4 * ((size_t)kStatusWords + kCounters);

// Few query tokens: a partial result of up to 16 rows for each part of a triple.
constexpr int kMaxParts = kCounters;
__host__ __device__ constexpr size_t partial_floats(int dim, int rows) { return (size_t)rows * (dim + 2); }
constexpr size_t kWorkspaceBytes = kPartialsAt + 4 * (size_t)kMaxParts * partial_floats(128, 16);

}  // namespace bytes
}  // namespace leankv
