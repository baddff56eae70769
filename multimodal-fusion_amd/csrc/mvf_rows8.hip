// Rows in 8 bits (layout: mvf_rows8.h): what a training step keeps of a layer's input for its
// backward pass, a quarter (float32) or half (16-bit types) of the bytes.
//
// Both directions are one pass bound by HBM: s + 1 bytes per value (s = 4 or 2) and one exponent
// byte per 32.  Packing gives 8 neighbouring lanes one group of one row, four columns each: the
// largest magnitude is three lane exchanges, no LDS and no second look at the row.  Packing and
// unpacking 2 M x 64 float32 together 246 us, 1.28 GB at 5.2 TB/s; what stays below that rate are rows
// narrower than a group, whose lanes are mostly idle (4 M x 1 float16: 67 us for 28 MB).
#include "mvf_rows8.h"

namespace mvf {

constexpr int R8_ROWS = 4;              // rows in flight per thread
constexpr int R8_MAX_BLOCKS = 4096;

template <class R, bool VEC>
__global__ __launch_bounds__(R8_THREADS) void pack_rows8_kernel(
    const typename R::T *__restrict__ x, i64 rows, int C, i64 rows_per_block,
    int8_t *__restrict__ codes, uint8_t *__restrict__ exps)
{
    const R8Walk w = r8_walk<true>(rows, C, rows_per_block);
    const int G = (C + R8_GROUP - 1) / R8_GROUP;
    const bool live = w.col < C;
    const bool lead = (threadIdx.x & 7) == 0;
    auto one = [&](i64 r, const float (&v)[4]) {
        const unsigned m = r8_max8(max(max(r8_magnitude(v[0]), r8_magnitude(v[1])), max(r8_magnitude(v[2]), r8_magnitude(v[3]))));
        const int e = r8_exponent(m, R::E_MAX);
        const int q[4] = {r8_encode(v[0], e), r8_encode(v[1], e), r8_encode(v[2], e), r8_encode(v[3], e)};
        if (live) codes_store4<VEC>(codes + r * C, w.col, C, r8_pack4(q));
        if (lead) exps[r * G + w.col / R8_GROUP] = (uint8_t)e;
    };
    i64 r = w.r0;
    for (; r + (R8_ROWS - 1) * (i64)w.rstep < w.rend; r += R8_ROWS * (i64)w.rstep) {
        float v[R8_ROWS][4];
#pragma unroll
        for (int u = 0; u < R8_ROWS; ++u) {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[u][j] = 0.0f;
            if (live) row_load4<R, VEC>(x + (r + (i64)u * w.rstep) * C, w.col, C, v[u]);
        }
#pragma unroll
        for (int u = 0; u < R8_ROWS; ++u) one(r + (i64)u * w.rstep, v[u]);
    }
    for (; r < w.rend; r += w.rstep) {
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (live) row_load4<R, VEC>(x + r * C, w.col, C, v);
        one(r, v);
    }
}

template <class R, bool VEC>
__global__ __launch_bounds__(R8_THREADS) void unpack_rows8_kernel(
    const int8_t *__restrict__ codes, const uint8_t *__restrict__ exps, i64 rows, int C, i64 rows_per_block,
    typename R::T *__restrict__ y)
{
    const R8Walk w = r8_walk<false>(rows, C, rows_per_block);
    const int G = (C + R8_GROUP - 1) / R8_GROUP, g = w.col / R8_GROUP;
    auto one = [&](i64 r, unsigned q, int e) {
        const float v[4] = {r8_decode(r8_byte(q, 0), e), r8_decode(r8_byte(q, 1), e),
                            r8_decode(r8_byte(q, 2), e), r8_decode(r8_byte(q, 3), e)};
        row_store4<R, VEC>(y + r * C, w.col, C, v);
    };
    i64 r = w.r0;
    for (; r + (R8_ROWS - 1) * (i64)w.rstep < w.rend; r += R8_ROWS * (i64)w.rstep) {
        unsigned q[R8_ROWS];
        int e[R8_ROWS];
#pragma unroll
        for (int u = 0; u < R8_ROWS; ++u) {
            const i64 ru = r + (i64)u * w.rstep;
            q[u] = codes_load4<VEC>(codes + ru * C, w.col, C);
            e[u] = exps[ru * G + g];
        }
#pragma unroll
        for (int u = 0; u < R8_ROWS; ++u) one(r + (i64)u * w.rstep, q[u], e[u]);
    }
    for (; r < w.rend; r += w.rstep) one(r, codes_load4<VEC>(codes + r * C, w.col, C), exps[r * G + g]);
}

}  // namespace mvf

using namespace mvf;

extern "C" int mvf_pack_rows8(
    const void *x, int32_t type, int64_t rows, int32_t C, int8_t *codes, uint8_t *exps, void *stream)
{
    MVF_REQUIRE(rows >= 0 && C >= 1, "pack_rows8: C must be positive, rows non-negative");
    MVF_REQUIRE(type >= R8_F32 && type <= R8_F16, "pack_rows8: unknown row type %d", (int)type);
    if (rows == 0) return MVF_OK;
    MVF_REQUIRE(x && codes && exps, "pack_rows8: null argument");
    const size_t item = type == R8_F32 ? 4 : 2;
    MVF_REQUIRE((uintptr_t)x % item == 0, "pack_rows8: x must be aligned to its element size");
    const bool vec = C % 4 == 0 && (uintptr_t)x % (4 * item) == 0 && (uintptr_t)codes % 4 == 0;
    const R8Grid g = r8_grid(rows, C, true, R8_ROWS, R8_MAX_BLOCKS);
    hipStream_t st = (hipStream_t)stream;
#define MVF_PACK(R_, V_)                                                                             \
    hipLaunchKernelGGL((pack_rows8_kernel<R_, V_>), g.grid, dim3(R8_THREADS), 0, st, (const R_::T *)x, (i64)rows, \
                       (int)C, g.rows_per_block, codes, exps)
#define MVF_PACK_V(R_) do { if (vec) MVF_PACK(R_, true); else MVF_PACK(R_, false); } while (0)
    if (type == R8_F32) MVF_PACK_V(RowF32);
    else if (type == R8_BF16) MVF_PACK_V(RowBF16);
    else MVF_PACK_V(RowF16);
#undef MVF_PACK_V
#undef MVF_PACK
    MVF_LAUNCH_CHECK();
    return MVF_OK;
}

extern "C" int mvf_unpack_rows8(
    const int8_t *codes, const uint8_t *exps, int64_t rows, int32_t C, void *y, int32_t type, void *stream)
{
    MVF_REQUIRE(rows >= 0 && C >= 1, "unpack_rows8: C must be positive, rows non-negative");
    MVF_REQUIRE(type >= R8_F32 && type <= R8_F16, "unpack_rows8: unknown row type %d", (int)type);
    if (rows == 0) return MVF_OK;
    MVF_REQUIRE(y && codes && exps, "unpack_rows8: null argument");
    const size_t item = type == R8_F32 ? 4 : 2;
    MVF_REQUIRE((uintptr_t)y % item == 0, "unpack_rows8: y must be aligned to its element size");
    const bool vec = C % 4 == 0 && (uintptr_t)y % (4 * item) == 0 && (uintptr_t)codes % 4 == 0;
    const R8Grid g = r8_grid(rows, C, false, R8_ROWS, R8_MAX_BLOCKS);
    hipStream_t st = (hipStream_t)stream;
#define MVF_UNPACK(R_, V_)                                                                           \
    hipLaunchKernelGGL((unpack_rows8_kernel<R_, V_>), g.grid, dim3(R8_THREADS), 0, st, codes, exps, (i64)rows, \
                       (int)C, g.rows_per_block, (R_::T *)y)
#define MVF_UNPACK_V(R_) do { if (vec) MVF_UNPACK(R_, true); else MVF_UNPACK(R_, false); } while (0)
    if (type == R8_F32) MVF_UNPACK_V(RowF32);
    else if (type == R8_BF16) MVF_UNPACK_V(RowBF16);
    else MVF_UNPACK_V(RowF16);
#undef MVF_UNPACK_V
#undef MVF_UNPACK
    MVF_LAUNCH_CHECK();
    return MVF_OK;
}
