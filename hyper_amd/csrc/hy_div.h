// The token of a pair: p / k for every 0 <= p < 2^31 and 1 <= k <= 64, as a 32 x 32 -> 64 bit product and a shift.  The constants
// depend on k alone and are made on the host, once a launch.
#pragma once
#include <cstdint>

namespace hy {

// mul = ceil(2^(32 + shift) / k) with 2^shift < k <= 2^(shift + 1), so that mul < 2^32 and the product fits 64 bits; mul 0: k = 1.
// mul k exceeds 2^(32 + shift) by e < k <= 2^(shift + 1), and p e < 2^31 2^(shift + 1): p mul / 2^(32 + shift) lies above p / k by
// less than 1 / k and its floor is the quotient.
struct Divisor { uint32_t mul, shift; };

inline Divisor divisor(uint32_t k) {
    if (k <= 1) return Divisor{0, 0};
    uint32_t s = 0;
    while ((2u << s) < k) ++s;
    return Divisor{(uint32_t) (((1ull << (32 + s)) + k - 1) / k), s};
}
__host__ __device__ inline int div_k(int p, const Divisor &d) { return d.mul ? (int) ((uint32_t) (((uint64_t) (uint32_t) p * d.mul) >> 32) >> d.shift) : p; }

} // namespace hy
