// Rows kept in 8 bits: device helpers shared by the kernels that write and read them.
//
// A row is cut into groups of 32 neighbouring columns (the last one may be shorter).  A group has
// one exponent byte e, the smallest with amax <= 127.5 * 2^(e - 133) for its largest finite
// magnitude amax, and every value one signed byte q = rint(v * 2^(133 - e)), ties to even, clamped
// to [-127, 127].  A value that is not finite has the code -128 and reads back as NaN.  The value
// read back, q * 2^(e - 133), has 7 significant bits and is exact in float32, bfloat16 and float16;
// it is off by at most half a step, 2^(e - 134) <= amax / 127.5.  Powers of two as steps make the
// codes a function of the values alone: the scaling is exact, there is one rounding.
#pragma once

#include "mvf_common.h"

namespace mvf {

constexpr int R8_GROUP = 32;
constexpr int R8_BIAS = 133;
constexpr int R8_E_MAX = 254;           // 127 * 2^121 is still finite in float32
constexpr int R8_E_MAX_F16 = 142;       // 127 * 2^9 in float16
constexpr int R8_NAN = -128;

static inline int r8_groups(int C) { return (C + R8_GROUP - 1) / R8_GROUP; }

// magnitude bits of v, 0 for a value that is not finite (magnitudes order like their bits)
__device__ __forceinline__ unsigned r8_magnitude(float v)
{
    const unsigned b = __float_as_uint(v) & 0x7fffffffu;
    return b < 0x7f800000u ? b : 0u;
}

// Exponent byte of a group from the bits of its largest magnitude: the exponent field, plus one
// when the mantissa is above that of 127.5 (1.9921875; denormals have no implicit one).
__device__ __forceinline__ int r8_exponent(unsigned amax, int most)
{
    const unsigned e = (amax + (amax < 0x00800000u ? 0x00007fffu : 0x0000ffffu)) >> 23;
    return min((int)e, most);
}

// largest value of the 8 neighbouring lanes, in all of them
__device__ __forceinline__ unsigned r8_max8(unsigned v)
{
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0xb1, 0xf, 0xf, true));     // lane ^ 1
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x4e, 0xf, 0xf, true));     // lane ^ 2
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, true));    // 7 - lane
    return v;
}

// largest value of the 4 neighbouring lanes, in all of them
__device__ __forceinline__ unsigned r8_max4(unsigned v)
{
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0xb1, 0xf, 0xf, true));
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x4e, 0xf, 0xf, true));
    return v;
}

__device__ __forceinline__ int r8_encode(float v, int e)
{
    float q = rintf(ldexpf(v, R8_BIAS - e));
    q = fminf(fmaxf(q, -127.0f), 127.0f);
    return (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u ? R8_NAN : (int)q;
}

__device__ __forceinline__ float r8_decode(int q, int e)
{
    const float v = ldexpf((float)q, e - R8_BIAS);
    return q == R8_NAN ? __uint_as_float(0x7fc00000u) : v;
}

// four codes in one word, the first column in the low byte
__device__ __forceinline__ unsigned r8_pack4(const int (&q)[4])
{
    return (unsigned)(q[0] & 255) | (unsigned)(q[1] & 255) << 8 | (unsigned)(q[2] & 255) << 16 | (unsigned)q[3] << 24;
}

__device__ __forceinline__ int r8_byte(unsigned w, int j) { return (int)(w << (24 - 8 * j)) >> 24; }

// ---- row types ------------------------------------------------------------------------------
enum { R8_F32 = 0, R8_BF16 = 1, R8_F16 = 2 };

struct RowF32 {
    typedef float T;
    static constexpr int E_MAX = R8_E_MAX;
    static __device__ __forceinline__ float get(T v) { return v; }
    static __device__ __forceinline__ T put(float v) { return v; }
};
struct RowBF16 {
    typedef unsigned short T;
    static constexpr int E_MAX = R8_E_MAX;
    static __device__ __forceinline__ float get(T v) { return __uint_as_float((unsigned)v << 16); }
    static __device__ __forceinline__ T put(float v) { return __builtin_bit_cast(unsigned short, (__bf16)v); }
    static __device__ __forceinline__ unsigned put2(float a, float b)
    {
        typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
        const bf2 t = {(__bf16)a, (__bf16)b};
        return __builtin_bit_cast(unsigned, t);
    }
};
struct RowF16 {
    typedef unsigned short T;
    static constexpr int E_MAX = R8_E_MAX_F16;
    static __device__ __forceinline__ float get(T v) { return (float)__builtin_bit_cast(_Float16, v); }
    static __device__ __forceinline__ T put(float v) { return __builtin_bit_cast(unsigned short, (_Float16)v); }
    static __device__ __forceinline__ unsigned put2(float a, float b) { return (unsigned)put(a) | (unsigned)put(b) << 16; }
};

// Wide accesses at the alignment of one element: rows of a width that is no multiple of the vector
// start anywhere, and the hardware reads and writes global memory at any address.
typedef unsigned r8_u4 __attribute__((ext_vector_type(4)));
typedef unsigned r8_u2 __attribute__((ext_vector_type(2)));
struct __attribute__((packed, aligned(4))) R8Words4 { unsigned w[4]; };
struct __attribute__((packed, aligned(2))) R8Half4 { unsigned w[2]; };
struct __attribute__((packed, aligned(2))) R8Half8 { unsigned w[4]; };
struct __attribute__((packed, aligned(2))) R8Half2 { unsigned w; };
struct __attribute__((packed, aligned(1))) R8Bytes2 { unsigned short w; };
struct __attribute__((packed, aligned(1))) R8Bytes4 { unsigned w; };
struct __attribute__((packed, aligned(1))) R8Bytes8 { unsigned w[2]; };

typedef float r8_f4 __attribute__((ext_vector_type(4)));

// 16 bytes of a result that is larger than the caches or is read again much later: a streaming store.
// It leaves the caches to what is still being read: a BatchNorm step of 2 M x 64 rows 758 -> 699 us,
// residual rows of 500000 x 64 287 -> 275 us; a reader right behind it loses and gains within 3 % at 16
// to 256 MB and gains 6 % at 4 MB.
template <class V> __device__ __forceinline__ void r8_stream(V *p, V v) { __builtin_nontemporal_store(v, p); }

// Four adjacent columns at col < C of a row of C columns (elements past C read as 0 and are not
// written).  VEC: C % 4 == 0 and the base is aligned to four elements; then col + 3 < C too.
template <class R, bool VEC>
__device__ __forceinline__ void row_load4(const typename R::T *row, int col, int C, float (&v)[4])
{
    if constexpr (VEC) {
        if constexpr (sizeof(typename R::T) == 4) {
            const float4 t = *reinterpret_cast<const float4 *>(row + col);
            v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
        } else {
            const uint2 t = *reinterpret_cast<const uint2 *>(row + col);
            v[0] = R::get((unsigned short)t.x); v[1] = R::get((unsigned short)(t.x >> 16));
            v[2] = R::get((unsigned short)t.y); v[3] = R::get((unsigned short)(t.y >> 16));
        }
    } else if (col + 4 <= C) {
        if constexpr (sizeof(typename R::T) == 4) {
            const R8Words4 t = *reinterpret_cast<const R8Words4 *>(row + col);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = __uint_as_float(t.w[j]);
        } else {
            const R8Half4 t = *reinterpret_cast<const R8Half4 *>(row + col);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = R::get((unsigned short)(t.w[j / 2] >> (16 * (j & 1))));
        }
    } else {                            // the last C % 4 columns (C is the same everywhere)
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = 0.0f;
        if (C & 2) {
            if constexpr (sizeof(typename R::T) == 4) {
                const R8Half4 t = *reinterpret_cast<const R8Half4 *>(row + col);
                v[0] = __uint_as_float(t.w[0]);
                v[1] = __uint_as_float(t.w[1]);
            } else {
                const unsigned t = reinterpret_cast<const R8Half2 *>(row + col)->w;
                v[0] = R::get((unsigned short)t);
                v[1] = R::get((unsigned short)(t >> 16));
            }
            if (C & 1) v[2] = R::get(row[col + 2]);
        } else {
            v[0] = R::get(row[col]);
        }
    }
}

template <class R, bool VEC>
__device__ __forceinline__ void row_store4(typename R::T *row, int col, int C, const float (&v)[4])
{
    if constexpr (VEC) {
        if constexpr (sizeof(typename R::T) == 4) {
            const r8_f4 t = {v[0], v[1], v[2], v[3]};
            r8_stream(reinterpret_cast<r8_f4 *>(row + col), t);
        } else {
            uint2 t;
            t.x = (unsigned)R::put(v[0]) | (unsigned)R::put(v[1]) << 16;
            t.y = (unsigned)R::put(v[2]) | (unsigned)R::put(v[3]) << 16;
            *reinterpret_cast<uint2 *>(row + col) = t;
        }
    } else if (col + 4 <= C) {
        if constexpr (sizeof(typename R::T) == 4) {
            R8Words4 t;
#pragma unroll
            for (int j = 0; j < 4; ++j) t.w[j] = __float_as_uint(v[j]);
            *reinterpret_cast<R8Words4 *>(row + col) = t;
        } else {
            R8Half4 t;
#pragma unroll
            for (int j = 0; j < 2; ++j) t.w[j] = (unsigned)R::put(v[2 * j]) | (unsigned)R::put(v[2 * j + 1]) << 16;
            *reinterpret_cast<R8Half4 *>(row + col) = t;
        }
    } else {
        if (C & 2) {
            if constexpr (sizeof(typename R::T) == 4) {
                const R8Half4 t = {{__float_as_uint(v[0]), __float_as_uint(v[1])}};
                *reinterpret_cast<R8Half4 *>(row + col) = t;
            } else {
                reinterpret_cast<R8Half2 *>(row + col)->w = (unsigned)R::put(v[0]) | (unsigned)R::put(v[1]) << 16;
            }
            if (C & 1) row[col + 2] = R::put(v[2]);
        } else {
            row[col] = R::put(v[0]);
        }
    }
}

template <bool VEC>
__device__ __forceinline__ unsigned codes_load4(const int8_t *row, int col, int C)
{
    if constexpr (VEC) {
        return *reinterpret_cast<const unsigned *>(row + col);
    } else if (col + 4 <= C) {
        return reinterpret_cast<const R8Bytes4 *>(row + col)->w;
    } else {
        if (col >= C) return 0u;
        if (!(C & 2)) return (uint8_t)row[col];
        const unsigned w = reinterpret_cast<const R8Bytes2 *>(row + col)->w;
        return C & 1 ? w | (unsigned)(uint8_t)row[col + 2] << 16 : w;
    }
}

template <bool VEC>
__device__ __forceinline__ void codes_store4(int8_t *row, int col, int C, unsigned w)
{
    if constexpr (VEC) {
        *reinterpret_cast<unsigned *>(row + col) = w;
    } else if (col + 4 <= C) {
        reinterpret_cast<R8Bytes4 *>(row + col)->w = w;
    } else if (col < C) {
        if (C & 2) {
            reinterpret_cast<R8Bytes2 *>(row + col)->w = (unsigned short)w;
            if (C & 1) row[col + 2] = (int8_t)(w >> 16);
        } else {
            row[col] = (int8_t)w;
        }
    }
}

// ---- walk over rows by slots of four columns ---------------------------------------------------
// A thread owns one slot (four columns) of its chunk of at most R8_THREADS slots (blockIdx.y) and
// steps down the rows of its block.  PAD: rows are padded to whole groups, 8 slots each, so that 8
// neighbouring lanes hold one group of one row (a slot past the last column is idle but takes part
// in the group's exchanges); otherwise a row has ceil(C / 4) slots.
constexpr int R8_THREADS = 256;

struct R8Walk {
    int col;            // first column of the slot
    bool in;            // the slot has a row to walk
    i64 r0, rend;
    int rstep;
};

template <bool PAD> __device__ __forceinline__ R8Walk r8_walk_at(i64 b0, i64 rend, int C)
{
    const int slots = PAD ? (C + R8_GROUP - 1) / R8_GROUP * 8 : (C + 3) / 4;
    const int chunk0 = blockIdx.y * R8_THREADS;
    const int cw = min(R8_THREADS, slots - chunk0);
    const int rpp = R8_THREADS / cw;
    const int t = threadIdx.x;
    R8Walk w;
    w.rstep = rpp;
    w.rend = rend;
    w.in = t < rpp * cw;
    w.col = (chunk0 + t % cw) * 4;
    w.r0 = w.in ? b0 + t / cw : w.rend;
    return w;
}

template <bool PAD> __device__ __forceinline__ R8Walk r8_walk(i64 rows, int C, i64 rows_per_block)
{
    const i64 b0 = (i64)blockIdx.x * rows_per_block;
    return r8_walk_at<PAD>(b0, min(rows, b0 + rows_per_block), C);
}

struct R8Grid {
    dim3 grid;
    i64 rows_per_block;
    int nblk;
};

// passes: least row passes per block; most: block limit
static inline R8Grid r8_grid(i64 rows, int C, bool pad, int passes, int most)
{
    const int slots = pad ? r8_groups(C) * 8 : (C + 3) / 4;
    const int cw = slots < R8_THREADS ? slots : R8_THREADS;
    const int rpp = R8_THREADS / cw;
    const int chunks = (slots + R8_THREADS - 1) / R8_THREADS;
    i64 nblk = (rows + (i64)rpp * passes - 1) / ((i64)rpp * passes);
    if (nblk > most) nblk = most;
    if (nblk < 1) nblk = 1;
    i64 rpb = (rows + nblk - 1) / nblk;
    rpb = (rpb + rpp - 1) / rpp * rpp;
    nblk = rpb > 0 ? (rows + rpb - 1) / rpb : 1;
    if (nblk < 1) nblk = 1;
    R8Grid g;
    g.grid = dim3((unsigned)nblk, (unsigned)chunks);
    g.rows_per_block = rpb;
    g.nblk = (int)nblk;
    return g;
}

}  // namespace mvf
