// Index arithmetic of the paged cache, the same on the host and in the kernels (it includes no HIP
// header, so a host compiler alone can check it).
#pragma once

#include <stdint.h>

#if defined(__HIP__) || defined(__HIPCC__)
#define Q3T_BOTH __host__ __device__ inline __attribute__((always_inline))
#else
#define Q3T_BOTH inline
#endif

namespace q3t {

// Division of 0 <= n < 2^31 by a divisor in [1, 2^31) as a multiplication, an addition and a
// shift: with 2^(l-1) < d <= 2^l and m = floor(2^32 (2^l - d) / d) + 1, floor(n / d) is
// (floor(m n / 2^32) + n) >> l (the sum stays below 2^32 since floor(m n / 2^32) <= n < 2^31).
struct Divisor {
    uint32_t d, m, l;
};
inline Divisor divisor(uint32_t d) {
    uint32_t l = 0;
    while (((uint64_t)1 << l) < d) ++l;
    return {d, (uint32_t)(((((uint64_t)1 << l) - d) << 32) / d + 1), l};
}
Q3T_BOTH uint32_t divide(uint32_t n, const Divisor &v) {
    return ((uint32_t)(((uint64_t)v.m * n) >> 32) + n) >> v.l;
}

}  // namespace q3t
