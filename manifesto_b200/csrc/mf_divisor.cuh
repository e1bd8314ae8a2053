// mf_divisor.cuh -- division by a number that only the host knows: a high
// multiplication, an addition and a shift instead of some twenty instructions.
#pragma once

#include <cstdint>

namespace mf {

// x / d = (mulhi(x, mul) + x) >> shift for x below 2^31, with 2^shift >= d the
// smallest such power and mul = floor(2^32 (2^shift - d) / d) + 1: mul + 2^32
// is 2^(32 + shift) / d rounded up, off by less than 2^shift / 2^(32 + shift)
// of a quotient per unit of x.
struct Divisor {
    uint32_t d, mul, shift;
};

inline Divisor divisor(int32_t d) {
    Divisor v{static_cast<uint32_t>(d), 0, 0};
    while ((1ull << v.shift) < v.d) ++v.shift;
    v.mul = static_cast<uint32_t>((((1ull << v.shift) - v.d) << 32) / v.d + 1);
    return v;
}

__device__ __forceinline__ uint32_t operator/(uint32_t x, const Divisor& v) { return (__umulhi(x, v.mul) + x) >> v.shift; }

}  // namespace mf
