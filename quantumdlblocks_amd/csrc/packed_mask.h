// The mask of packed attention: query position i sees key j where
// lower <= i - j < upper.  Apart from the kernels, so that a host compiler takes it.
#pragma once

#include <cstdint>

namespace qdl {

// Without causality or a window the bounds lie 2^30 away on that side.
constexpr int kPackedFar = 1 << 30;
constexpr int packed_lower(bool causal) { return causal ? 0 : -kPackedFar; }
constexpr int packed_upper(int64_t window) { return window > 0 && window < kPackedFar ? (int)window : kPackedFar; }

// upper - lower, up to 2^31: the bound of (uint32_t)(i - j - lower).
constexpr uint32_t packed_span(int lower, int upper) { return (uint32_t)upper - (uint32_t)lower; }

}  // namespace qdl
