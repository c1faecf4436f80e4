// Where min-p ends: the smallest value whose probability is at least min_p times
// the largest's.  (top - x) oct <= -log2(min_p) in fp64, decided for values that
// are floats: near a guess by division, else by bisection over the floats' order,
// which ends after 32 steps wherever the guess lies (around 0 the floats are so
// dense that a rounding of the guess may be a billion of them).
#pragma once
#include <cfloat>
#include <cmath>
#include <cstdint>
#include <cstring>

namespace hq4 {

// Bits that order as the floats do, and back.
__host__ __device__ __forceinline__ uint32_t order_bits(float x) {
    uint32_t b;
    memcpy(&b, &x, 4);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__host__ __device__ __forceinline__ float order_value(uint32_t k) {
    const uint32_t b = k & 0x80000000u ? k ^ 0x80000000u : ~k;
    float x;
    memcpy(&x, &b, 4);
    return x;
}

// The least of the order bits lowest .. last that stays, where `last` does and
// with each that stays all above it do; `guess` is one of them, best at it or
// next to it.
template <class Stays>
__host__ __device__ __forceinline__ uint32_t first_that_stays(uint32_t lowest, uint32_t guess, uint32_t last, Stays stays) {
    uint32_t out = lowest - 1, in = last;  // out does not stay (or is none of them), in does
    const uint32_t below = guess - lowest > 1 ? guess - 2 : out, above = last - guess > 2 ? guess + 2 : last;
    if (below != out) (stays(below) ? in : out) = below;
    if (above < in) (stays(above) ? in : out) = above;
    while (in - out > 1) {
        const uint32_t mid = out + ((in - out) >> 1);
        (stays(mid) ? in : out) = mid;
    }
    return in;
}

// The smallest value that min_p keeps (above -inf; at most the maximum).  oct:
// octaves for a unit of x; 0 at an infinite temperature, where all finite
// entries are equally likely.
__host__ __device__ __forceinline__ float min_p_end(float min_p, float top, double oct) {
    if (!(oct > 0.0)) return -FLT_MAX;
    const double most = -log2((double)fminf(min_p, 1.0f));
    const float guess = (float)fmax((double)top - most / oct, -(double)FLT_MAX);
    return order_value(first_that_stays(order_bits(-FLT_MAX), order_bits(fminf(guess, top)), order_bits(top), [&](uint32_t k) {
               return ((double)top - (double)order_value(k)) * oct <= most;
           })) + 0.0f;
}

}  // namespace hq4
