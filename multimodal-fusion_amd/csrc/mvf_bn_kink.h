// The kink of LeakyReLU behind BatchNorm, in terms of the normalised value kept in 8 bits.
//
// The backward has to know on which side of the activation's kink a value lay, and 8 bits next to
// the kink do not tell.  With u = zhat * gamma + beta the kink is at t = -beta / gamma; a code that
// would read back on the wrong side of t is moved to the nearest one on the right side (at most one
// step, and only values within half a step of t).  BnKink: the test as a compare of zhat * sign
// with t * sign; gamma == 0 leaves u = beta for every row.
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
