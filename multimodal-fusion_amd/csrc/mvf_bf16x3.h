// float32 values as exact sums of bf16 parts for the bf16 matrix cores (v_mfma_f32_32x32x16_bf16), and
// the fold of per-workgroup partial results, shared by the weight-gradient kernels.
#pragma once

#include "mvf_common.h"

namespace mvf {

typedef float xty_acc __attribute__((ext_vector_type(16)));
typedef __bf16 xty_bf8 __attribute__((ext_vector_type(8)));
typedef unsigned xty_u4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ xty_acc xty_mfma16(xty_u4 a, xty_u4 b, xty_acc c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(xty_bf8, a), __builtin_bit_cast(xty_bf8, b), c, 0, 0, 0);
}

__device__ __forceinline__ xty_acc xty_zero()
{
    return xty_acc{0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
}

// high halves of two floats as two bf16 (the first in the low half)
__device__ __forceinline__ unsigned xty_hi2(float a, float b)
{
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}

// 8 float32 as bf16 parts: v = p[0] + p[1] + p[2] exactly for PARTS == 3, p[0] alone for values that
// one bf16 holds
template <int PARTS> struct XtyParts {
    xty_u4 p[PARTS];
    __device__ __forceinline__ void cut(const float (&v)[8])
    {
        float r[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) r[j] = v[j];
#pragma unroll
        for (int k = 0; k < PARTS; ++k) {
#pragma unroll
            for (int h = 0; h < 4; ++h) p[k][h] = xty_hi2(r[2 * h], r[2 * h + 1]);
            if (k + 1 < PARTS)
#pragma unroll
                for (int j = 0; j < 8; ++j) r[j] -= __uint_as_float(__float_as_uint(r[j]) & 0xffff0000u);
        }
    }
};

// c and 16 rows' part of the sums, the smallest parts first
__device__ __forceinline__ xty_acc xty_product(const XtyParts<3> &x, xty_u4 y, xty_acc c)
{
    return xty_mfma16(x.p[0], y, xty_mfma16(x.p[1], y, xty_mfma16(x.p[2], y, c)));
}

// Behind every addition of a product: the sums are formed here.  The product's registers are free for the next
// one, and no branch comes between the two (hipcc counts the waits that a matrix instruction's result needs along
// one side of a branch only: without this, rows of 32 -> 32 columns without bias gave wrong sums).
__device__ __forceinline__ void xty_done(xty_acc &sum)
{
    asm volatile("" : "+v"(sum));
    __builtin_amdgcn_sched_barrier(0);
}

// The matrix cores add bf16 products to float32 sums by cutting off what does not fit, towards minus
// infinity.  Sums of one sign kept in one accumulator over all rows come out 4e-6 of themselves short at 8 M
// rows, and more than in proportion beyond; sums of zero-mean terms are moved together, by 2e-6 of their
// typical size at 2 M.  So every 16 (or 32) rows are a product of their own, from zero, which the vector unit adds
// to the wave's float32 sums, to the nearest (Linear of 2 M x 64 -> 64, forward and backward, 505 -> 510 us; error
// of zero-mean sums 3e-7 -> 1.6e-7, of one sign that of their last rounding).  What a product still cuts off
// downwards cancels between the waves: odd ones sum the negated products (one operand's sign turned, by a factor
// or in its two bf16) and are subtracted where waves are joined, in float64 from the workgroup on.
__device__ __forceinline__ float xty_turned(int wave) { return wave & 1 ? -1.0f : 1.0f; }
__device__ __forceinline__ unsigned xty_flip(int wave) { return wave & 1 ? 0x80008000u : 0u; }

// Adds up the partial results of nwg workgroups: partial [nwg][NA * NB * 1024] accumulators of NA x NB
// blocks of 32 x 32 sums as v_mfma_f32_32x32x16_bf16 leaves them (vx / vy: an operand of two blocks holds
// columns 2 n and 2 n + 1 in lane n), out [A][ldo], and with partial_sums [nwg][64] the sums [A].
void xty8_fold(const float *partial, const float *partial_sums, int nwg, int NA, int NB, int vx, int vy, int A, int B,
               float *out, int ldo, float *sums, hipStream_t st);

}  // namespace mvf
