// Division by numbers that are fixed for a launch.
#pragma once

#include "common.hpp"

namespace axhip {

// n / d for n < 2^31 by one multiplication (d fixed for a launch): with m = ceil(2^(32 + s) / d), 2^s >= d, the error n / 2^(32 + s) stays
// below 1 / d.  m - 2^32 is what is kept; (hi + n) / 2^s without an overflow since n < 2^31.
struct Divisor {
    uint32_t d = 1, m = 1, s = 0;
    Divisor() = default;
    explicit Divisor(uint32_t div) : d(div), m(0), s(0) {
        while ((uint64_t(1) << s) < d) ++s;
        m = static_cast<uint32_t>(((uint64_t(1) << 32) * ((uint64_t(1) << s) - d)) / d + 1);
    }
    __device__ __forceinline__ uint32_t of(uint32_t n) const { return (__umulhi(n, m) + n) >> s; }
};

} // namespace axhip
