// portions.h -- a long call as several launches (rows of a cache in 4 bits, rows of logits, pairs of pages).  Plain C++, so that totals no machine holds can be tried on the CPU.
#pragma once
#include <stdint.h>

#include <algorithm>

namespace nb {

// f(start, count) for [0, total) in portions of at most `most`, until one does not return success (0).  A start counted in 32 bits would pass 2^32 at the end of a total
// near that and begin again, for ever
template <typename F>
auto in_portions(uint64_t total, uint32_t most, F f) -> decltype(f(0u, 0u)) {
    using R = decltype(f(0u, 0u));
    for (uint64_t at = 0; at < total; at += most) {
        const R r = f((uint32_t)at, (uint32_t)std::min<uint64_t>(most, total - at));
        if (r != R{}) return r;
    }
    return R{};
}

}  // namespace nb
