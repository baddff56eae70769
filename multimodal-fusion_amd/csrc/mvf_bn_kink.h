// The kink of LeakyReLU behind BatchNorm, in terms of the normalised value kept in 8 bits.
//
// The backward has to know on which side of the activation's kink a value lay, and 8 bits next to
// the kink do not tell.  With u = zhat * gamma + beta the kink is at t = -beta / gamma; a code that
// would read back on the wrong side of t is moved to the nearest one on the right side (at most one
// step, and only values within half a step of t).  Past 127 steps there is no next code: where a
// value of at least 127 steps meets a t of 127 to 128 steps, its group takes the next step
// (BnKink::most).  BnKink: the test as a compare of zhat * sign with t * sign; gamma == 0 leaves
// u = beta for every row.
#pragma once

#include "mvf_rows8.h"

namespace mvf {

struct BnKink {
    float sign, at;
    __device__ __forceinline__ void load(float gamma, float beta)
    {
        if (gamma == 0.0f) {
            sign = 0.0f;
            at = beta > 0.0f ? -1.0f : 1.0f;
        } else {
            sign = gamma < 0.0f ? -1.0f : 1.0f;
            at = __fdiv_rn(-beta, gamma) * sign;
        }
    }
    __device__ __forceinline__ bool on(float zq) const { return zq * sign > at; }
    // Bits of the smallest value that needs the group's next step for t's sake; bits of infinity: none does.
    // (127 / 64 = 0x7e0000 of a mantissa; no group's largest value is below the normal numbers.)
    __device__ __forceinline__ unsigned last() const
    {
        const unsigned b = __float_as_uint(at) & 0x7fffffffu;
        return sign != 0.0f && (b & 0x007fffffu) >= 0x007e0000u && b >= 0x00800000u ? b & 0xfffe0000u : 0x7f800000u;
    }
    // max(m, r8_magnitude of a normalised value), past the range of the value's own step where it meets t there
    static __device__ __forceinline__ unsigned most(unsigned m, float zf, unsigned last)
    {
        const unsigned b = r8_magnitude(zf);
        return max(max(m, b), b >= last ? last | 0x0001ffffu : 0u);
    }
    // code (not yet clamped) moved to its side; steps of 2^(e - R8_BIAS)
    __device__ __forceinline__ float side(float q, bool on, int e) const
    {
        if (sign == 0.0f) return q;
        const float f = floorf(ldexpf(at, R8_BIAS - e));
        const float c = q * sign;
        return (on ? fmaxf(c, f + 1.0f) : fminf(c, f)) * sign;
    }
};

}  // namespace mvf
