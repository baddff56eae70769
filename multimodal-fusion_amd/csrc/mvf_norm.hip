// Tail of a dense layer in a differentiable forward: BatchNorm1d (batch statistics in
// train mode, running statistics otherwise) + LeakyReLU on float32 rows [rows][C], forward
// and backward (the MLP blocks of core/common_modules/base_modules.py:38-48 with the
// FastBatchNorm1d of :131-156; the Linear in front of them is a plain library GEMM).
//
// Everything here is bound by HBM: the forward reads the rows twice (column sums, then
// normalise + activate) and writes them once; the backward reads rows and gradient twice
// and writes the input gradient once.  Nothing but the input of the layer is kept for
// the backward: the normalised value and the sign of the activation are recomputed.
//
// Layout: with C a multiple of 4 a thread owns one group of 4 adjacent columns for the
// whole launch (its statistics and affine terms stay in registers) and steps down the
// rows; consecutive threads read consecutive 16 bytes.  Column sums are accumulated in
// float64 per thread, reduced per block in a fixed order and written as one partial row
// per block; a second small kernel folds the partials in a fixed order, so the
// statistics are the same on every run.
#include "mvf_bn_kink.h"
#include "mvf_norm.h"
#include "mvf_rows8.h"

namespace mvf {

constexpr int BN_THREADS = 256;
constexpr int BN_FOLD_COLS = 4;         // columns per block of the fold kernels

template <int VW> __device__ __forceinline__ void bn_load(const float *p, float (&v)[VW])
{
    if constexpr (VW == 4) {
        const float4 t = *reinterpret_cast<const float4 *>(p);
        v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
    } else {
        v[0] = *p;
    }
}

template <int VW> __device__ __forceinline__ void bn_store(float *p, const float (&v)[VW])
{
    if constexpr (VW == 4) *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
    else *p = v[0];
}

// What a thread of the row-walking kernels owns: column group `cv` of its chunk of at most
// BN_THREADS groups (blockIdx.y), rows r0 + k * rstep below `rend`.
struct BnWalk {
    int col;            // first column of the thread's group, -1: idle thread
    i64 r0, rend;
    int rstep;
};

template <int VW> __device__ __forceinline__ BnWalk bn_walk(i64 rows, int C, i64 rows_per_block, int block)
{
    const int CV = C / VW;
    const int chunk0 = blockIdx.y * BN_THREADS;
    const int cw = min(BN_THREADS, CV - chunk0);            // groups in this chunk
    const int rpp = BN_THREADS / cw;                        // rows per pass of the block
    const int t = threadIdx.x;
    BnWalk w;
    w.rstep = rpp;
    const i64 b0 = block * rows_per_block;
    w.rend = min(rows, b0 + rows_per_block);
    if (t >= rpp * cw) {
        w.col = -1;
        w.r0 = w.rend;
    } else {
        w.col = (chunk0 + t % cw) * VW;
        w.r0 = b0 + t / cw;
    }
    return w;
}

// Per-column terms a thread keeps in registers.
template <int VW> struct BnTerms {
    float mean[VW], invstd[VW], gamma[VW], beta[VW];
    __device__ __forceinline__ void load(int col, const float *save_mean, const float *save_invstd,
                                         const float *weight, const float *bias)
    {
#pragma unroll
        for (int j = 0; j < VW; ++j) {
            mean[j] = save_mean[col + j];
            invstd[j] = save_invstd[col + j];
            gamma[j] = weight ? weight[col + j] : 1.0f;
            beta[j] = bias ? bias[col + j] : 0.0f;
        }
    }
};

// Block-level fold of per-thread float64 pairs into one partial row:
// partial[block][0][C] and partial[block][1][C].
template <int VW>
__device__ __forceinline__ void bn_block_fold(const double (&s)[VW], const double (&q)[VW], int C, double *partial)
{
    __shared__ double red[BN_THREADS][2 * VW];
    const int CV = C / VW;
    const int chunk0 = blockIdx.y * BN_THREADS;
    const int cw = min(BN_THREADS, CV - chunk0);
    const int rpp = BN_THREADS / cw;
    const int t = threadIdx.x;
#pragma unroll
    for (int j = 0; j < VW; ++j) {
        red[t][j] = s[j];
        red[t][VW + j] = q[j];
    }
    __syncthreads();
    if (t < cw) {
        double a[2 * VW];
#pragma unroll
        for (int j = 0; j < 2 * VW; ++j) a[j] = red[t][j];
        for (int r = 1; r < rpp; ++r)
#pragma unroll
            for (int j = 0; j < 2 * VW; ++j) a[j] += red[r * cw + t][j];
        double *p = partial + (size_t)blockIdx.x * 2 * C;
        const int col = (chunk0 + t) * VW;
#pragma unroll
        for (int j = 0; j < VW; ++j) {
            p[col + j] = a[j];
            p[C + col + j] = a[VW + j];
        }
    }
}

// Column sums of z and z*z.
template <int VW>
__global__ __launch_bounds__(BN_THREADS) void bn_sums_kernel(
    const float *__restrict__ z, i64 rows, int C, i64 rows_per_block, double *__restrict__ partial)
{
    const BnWalk w = bn_walk<VW>(rows, C, rows_per_block, blockIdx.x);
    double s[VW], q[VW];
#pragma unroll
    for (int j = 0; j < VW; ++j) s[j] = q[j] = 0.0;
    if (w.col >= 0) {
        const float *p = z + w.col;
        i64 r = w.r0;
        // four rows in flight per thread
        for (; r + 3 * (i64)w.rstep < w.rend; r += 4 * (i64)w.rstep) {
            float v[4][VW];
#pragma unroll
            for (int u = 0; u < 4; ++u) bn_load<VW>(p + (r + (i64)u * w.rstep) * C, v[u]);
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int j = 0; j < VW; ++j) {
                    const double d = (double)v[u][j];
                    s[j] += d;
                    q[j] += d * d;
                }
        }
        for (; r < w.rend; r += w.rstep) {
            float v[VW];
            bn_load<VW>(p + r * C, v);
#pragma unroll
            for (int j = 0; j < VW; ++j) {
                const double d = (double)v[j];
                s[j] += d;
                q[j] += d * d;
            }
        }
    }
    bn_block_fold<VW>(s, q, C, partial);
}

// Column sums of g and g * zhat, with zhat = (z - mean) * invstd, u = zhat * gamma + beta and
// g = grad_y * (u > 0 ? 1 : slope) (act) or grad_y.
template <int VW>
__global__ __launch_bounds__(BN_THREADS) void bn_grad_sums_kernel(
    const float *__restrict__ gy, const float *__restrict__ z, i64 rows, int C, i64 rows_per_block,
    const float *__restrict__ save_mean, const float *__restrict__ save_invstd,
    const float *__restrict__ weight, const float *__restrict__ bias, int act, float slope,
    double *__restrict__ partial)
{
    const BnWalk w = bn_walk<VW>(rows, C, rows_per_block, blockIdx.x);
    double s[VW], q[VW];
#pragma unroll
    for (int j = 0; j < VW; ++j) s[j] = q[j] = 0.0;
    if (w.col >= 0) {
        BnTerms<VW> T;
        T.load(w.col, save_mean, save_invstd, weight, bias);
        i64 r = w.r0;
        for (; r + (i64)w.rstep < w.rend; r += 2 * (i64)w.rstep) {
            float v[2][VW], g[2][VW];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                bn_load<VW>(z + (r + (i64)u * w.rstep) * C + w.col, v[u]);
                bn_load<VW>(gy + (r + (i64)u * w.rstep) * C + w.col, g[u]);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int j = 0; j < VW; ++j) {
                    const float zh = (v[u][j] - T.mean[j]) * T.invstd[j];
                    const float act_in = zh * T.gamma[j] + T.beta[j];
                    const float gg = (act && !(act_in > 0.0f)) ? g[u][j] * slope : g[u][j];
                    s[j] += (double)gg;
                    q[j] += (double)gg * (double)zh;
                }
        }
        for (; r < w.rend; r += w.rstep) {
            float v[VW], g[VW];
            bn_load<VW>(z + r * C + w.col, v);
            bn_load<VW>(gy + r * C + w.col, g);
#pragma unroll
            for (int j = 0; j < VW; ++j) {
                const float zh = (v[j] - T.mean[j]) * T.invstd[j];
                const float act_in = zh * T.gamma[j] + T.beta[j];
                const float gg = (act && !(act_in > 0.0f)) ? g[j] * slope : g[j];
                s[j] += (double)gg;
                q[j] += (double)gg * (double)zh;
            }
        }
    }
    bn_block_fold<VW>(s, q, C, partial);
}

// Fold of the partial rows: BN_FOLD_COLS columns per block, each by BN_THREADS / BN_FOLD_COLS
// threads that take interleaved partial rows; their sums are added pairwise through LDS (a
// fixed tree).  out0 / out1: the two column sums, valid in the thread with owner set.
__device__ __forceinline__ void bn_fold(const double *partial, int nblk, int C, double &out0, double &out1, bool &owner, int &col)
{
    __shared__ double red[BN_THREADS][2];
    const int t = threadIdx.x;
    const int c = t % BN_FOLD_COLS, slice = t / BN_FOLD_COLS;
    constexpr int SLICES = BN_THREADS / BN_FOLD_COLS;
    col = blockIdx.x * BN_FOLD_COLS + c;
    double a = 0.0, b = 0.0;
    if (col < C)
        for (int k = slice; k < nblk; k += SLICES) {
            a += partial[(size_t)k * 2 * C + col];
            b += partial[(size_t)k * 2 * C + C + col];
        }
    red[t][0] = a;
    red[t][1] = b;
    __syncthreads();
    for (int half = SLICES / 2; half >= 1; half >>= 1) {
        if (slice < half) {
            red[t][0] += red[t + half * BN_FOLD_COLS][0];
            red[t][1] += red[t + half * BN_FOLD_COLS][1];
        }
        __syncthreads();
    }
    owner = slice == 0 && col < C;
    out0 = red[t][0];
    out1 = red[t][1];
}

// Batch statistics from the column sums; running statistics updated as nn.BatchNorm1d does
// (biased variance for the normalisation, unbiased for the running estimate).
__global__ __launch_bounds__(BN_THREADS) void bn_stats_kernel(
    const double *__restrict__ partial, int nblk, int C, i64 rows, float eps, float momentum,
    float *__restrict__ running_mean, float *__restrict__ running_var,
    float *__restrict__ save_mean, float *__restrict__ save_invstd, double *__restrict__ terms64,
    long long *__restrict__ num_batches)
{
    if (num_batches && blockIdx.x == 0 && threadIdx.x == 0) *num_batches += 1;
    double S, Q;
    bool owner;
    int col;
    bn_fold(partial, nblk, C, S, Q, owner, col);
    if (!owner) return;
    const double n = (double)rows;
    const double mean = S / n;
    double var = Q / n - mean * mean;
    if (var < 0.0) var = 0.0;
    save_mean[col] = (float)mean;
    const double invstd = 1.0 / sqrt(var + (double)eps);
    save_invstd[col] = (float)invstd;
    if (terms64) {
        terms64[col] = mean;
        terms64[C + col] = invstd;
    }
    if (running_mean) running_mean[col] = (float)((1.0 - (double)momentum) * (double)running_mean[col] + (double)momentum * mean);
    if (running_var) {
        const double unbiased = rows > 1 ? var * n / (n - 1.0) : var;
        running_var[col] = (float)((1.0 - (double)momentum) * (double)running_var[col] + (double)momentum * unbiased);
    }
}

// Normalisation terms from the running statistics (eval mode with a graph).
__global__ void bn_running_terms_kernel(
    const float *__restrict__ running_mean, const float *__restrict__ running_var, int C, float eps,
    float *__restrict__ save_mean, float *__restrict__ save_invstd, double *__restrict__ terms64)
{
    const int c = blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= C) return;
    save_mean[c] = running_mean[c];
    const double invstd = 1.0 / sqrt((double)running_var[c] + (double)eps);
    save_invstd[c] = (float)invstd;
    if (terms64) {
        terms64[c] = (double)running_mean[c];
        terms64[C + c] = invstd;
    }
}

// Gradients of weight and bias, and the two per-column means the input gradient needs.
__global__ __launch_bounds__(BN_THREADS) void bn_grad_terms_kernel(
    const double *__restrict__ partial, int nblk, int C, i64 rows,
    float *__restrict__ grad_weight, float *__restrict__ grad_bias, float *__restrict__ col_terms)
{
    double S, Q;
    bool owner;
    int col;
    bn_fold(partial, nblk, C, S, Q, owner, col);
    if (!owner) return;
    if (grad_bias) grad_bias[col] = (float)S;
    if (grad_weight) grad_weight[col] = (float)Q;
    col_terms[col] = (float)(S / (double)rows);
    col_terms[C + col] = (float)(Q / (double)rows);
}

// y = act((z - mean) * invstd * gamma + beta)
template <int VW>
__global__ __launch_bounds__(BN_THREADS) void bn_apply_kernel(
    const float *__restrict__ z, i64 rows, int C, i64 rows_per_block,
    const float *__restrict__ save_mean, const float *__restrict__ save_invstd,
    const float *__restrict__ weight, const float *__restrict__ bias, int act, float slope,
    float *__restrict__ y)
{
    const BnWalk w = bn_walk<VW>(rows, C, rows_per_block, blockIdx.x);
    if (w.col < 0) return;
    BnTerms<VW> T;
    T.load(w.col, save_mean, save_invstd, weight, bias);
    i64 r = w.r0;
    for (; r + 3 * (i64)w.rstep < w.rend; r += 4 * (i64)w.rstep) {
        float v[4][VW];
#pragma unroll
        for (int u = 0; u < 4; ++u) bn_load<VW>(z + (r + (i64)u * w.rstep) * C + w.col, v[u]);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
#pragma unroll
            for (int j = 0; j < VW; ++j) {
                const float a = (v[u][j] - T.mean[j]) * T.invstd[j] * T.gamma[j] + T.beta[j];
                v[u][j] = (act && !(a > 0.0f)) ? a * slope : a;
            }
            bn_store<VW>(y + (r + (i64)u * w.rstep) * C + w.col, v[u]);
        }
    }
    for (; r < w.rend; r += w.rstep) {
        float v[VW];
        bn_load<VW>(z + r * C + w.col, v);
#pragma unroll
        for (int j = 0; j < VW; ++j) {
            const float a = (v[j] - T.mean[j]) * T.invstd[j] * T.gamma[j] + T.beta[j];
            v[j] = (act && !(a > 0.0f)) ? a * slope : a;
        }
        bn_store<VW>(y + r * C + w.col, v);
    }
}

// grad_z = gamma * invstd * (g - mean(g) - zhat * mean(g * zhat))   (batch statistics)
//        = gamma * invstd * g                                        (running statistics)
template <int VW>
__global__ __launch_bounds__(BN_THREADS) void bn_grad_apply_kernel(
    const float *__restrict__ gy, const float *__restrict__ z, i64 rows, int C, i64 rows_per_block,
    const float *__restrict__ save_mean, const float *__restrict__ save_invstd,
    const float *__restrict__ weight, const float *__restrict__ bias, int act, float slope,
    const float *__restrict__ col_terms, int training, float *__restrict__ gz)
{
    const BnWalk w = bn_walk<VW>(rows, C, rows_per_block, blockIdx.x);
    if (w.col < 0) return;
    BnTerms<VW> T;
    T.load(w.col, save_mean, save_invstd, weight, bias);
    float m_g[VW], m_gz[VW], k[VW];
#pragma unroll
    for (int j = 0; j < VW; ++j) {
        m_g[j] = training ? col_terms[w.col + j] : 0.0f;
        m_gz[j] = training ? col_terms[C + w.col + j] : 0.0f;
        k[j] = T.gamma[j] * T.invstd[j];
    }
    i64 r = w.r0;
    for (; r + (i64)w.rstep < w.rend; r += 2 * (i64)w.rstep) {
        float v[2][VW], g[2][VW];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            bn_load<VW>(z + (r + (i64)u * w.rstep) * C + w.col, v[u]);
            bn_load<VW>(gy + (r + (i64)u * w.rstep) * C + w.col, g[u]);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int j = 0; j < VW; ++j) {
                const float zh = (v[u][j] - T.mean[j]) * T.invstd[j];
                const float act_in = zh * T.gamma[j] + T.beta[j];
                const float gg = (act && !(act_in > 0.0f)) ? g[u][j] * slope : g[u][j];
                v[u][j] = (gg - m_g[j] - zh * m_gz[j]) * k[j];
            }
            bn_store<VW>(gz + (r + (i64)u * w.rstep) * C + w.col, v[u]);
        }
    }
    for (; r < w.rend; r += w.rstep) {
        float v[VW], g[VW];
        bn_load<VW>(z + r * C + w.col, v);
        bn_load<VW>(gy + r * C + w.col, g);
#pragma unroll
        for (int j = 0; j < VW; ++j) {
            const float zh = (v[j] - T.mean[j]) * T.invstd[j];
            const float act_in = zh * T.gamma[j] + T.beta[j];
            const float gg = (act && !(act_in > 0.0f)) ? g[j] * slope : g[j];
            v[j] = (gg - m_g[j] - zh * m_gz[j]) * k[j];
        }
        bn_store<VW>(gz + r * C + w.col, v);
    }
}

// Launch shape of the row-walking kernels: (row blocks, column chunks), rows per block a
// multiple of the rows a block covers per pass.
struct BnGrid {
    dim3 grid;
    i64 rows_per_block;
    int nblk;
};

static BnGrid bn_grid(i64 rows, int C, int VW)
{
    const int CV = C / VW;
    const int cw = CV < BN_THREADS ? CV : BN_THREADS;
    const int rpp = BN_THREADS / cw;
    const int chunks = (CV + BN_THREADS - 1) / BN_THREADS;
    // at least eight passes per block, at most BN_MAX_BLOCKS blocks
    i64 nblk = (rows + (i64)rpp * 8 - 1) / ((i64)rpp * 8);
    if (nblk > BN_MAX_BLOCKS) nblk = BN_MAX_BLOCKS;
    if (nblk < 1) nblk = 1;
    i64 rpb = (rows + nblk - 1) / nblk;
    rpb = (rpb + rpp - 1) / rpp * rpp;
    nblk = (rows + rpb - 1) / rpb;
    if (nblk < 1) nblk = 1;
    BnGrid g;
    g.grid = dim3((unsigned)nblk, (unsigned)chunks);
    g.rows_per_block = rpb;
    g.nblk = (int)nblk;
    return g;
}

// ---- the same tail with its normalised input kept in 8 bits ---------------------------------------
// What the backward reads is the 8-bit form (mvf_rows8.h) of zhat = (z - mean) * invstd instead of z:
// a byte per value, and 9 instead of 12 bytes per value in the pass that writes grad_z.  zhat and its
// code are computed in float64 (a few of the vector unit's idle cycles in a pass bound by HBM), so
// that a code does not depend on how the statistics were rounded.  (BnKink: mvf_bn_kink.h keeps a
// code on its own side of the activation's kink.)

// The second pass over rows that a first one has just summed begins where the first ended: a block of
// the first pass walks a range of rows from front to back, all ranges at once, so what the
// memory-side cache still holds are the ends of the ranges.  The second pass takes the last quarter
// of every range first, then the third, and so on (a step of 2 M x 64 rows: 724 -> 690 us).
struct BnQuarters {
    int ranges;
    i64 rows_per_range, rows_per_block;     // (a block: a quarter of a range)
    __device__ __forceinline__ void place(i64 rows, i64 &b0, i64 &rend) const
    {
        const int q = 3 - (int)(blockIdx.x / ranges), range = (int)(blockIdx.x % ranges);
        const i64 r0 = range * rows_per_range, r1 = min(rows, r0 + rows_per_range);
        b0 = min(r1, r0 + q * rows_per_block);
        rend = min(r1, b0 + rows_per_block);
    }
};

static BnQuarters bn_quarters(const BnGrid &g, int rpp)
{
    const i64 quarter = (g.rows_per_block + 3) / 4;
    return {g.nblk, g.rows_per_block, (quarter + rpp - 1) / rpp * rpp};
}

// One slot of a row: y = act((z - mean) * invstd * gamma + beta) with the terms rounded to float32
// (bn_apply_kernel's value; y may be NULL) and the code of zhat.  Called by the 8 lanes of a group together.
template <bool VEC>
__device__ __forceinline__ void bn_apply8_row(
    const float (&v)[4], i64 r, int col, int C, int G, bool live, const double (&mean64)[4], const double (&invstd64)[4],
    const float (&gamma)[4], const float (&beta)[4], const BnKink (&kink)[4], const unsigned (&last)[4],
    int act, float slope, float *y, int8_t *codes, uint8_t *exps)
{
    double zh[4];
    unsigned m = 0;
    float zf[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        zh[j] = ((double)v[j] - mean64[j]) * invstd64[j];
        zf[j] = (float)zh[j];
        if (VEC ? live : col + j < C) m = BnKink::most(m, zf[j], last[j]);
    }
    const int e = r8_exponent(r8_max8(m), R8_E_MAX);
    int q[4];
    float o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float c = (float)rint(ldexp(zh[j], R8_BIAS - e));
        if (act) c = kink[j].side(c, zh[j] * (double)gamma[j] + (double)beta[j] > 0.0, e);
        c = fminf(fmaxf(c, -127.0f), 127.0f);
        q[j] = (__float_as_uint(zf[j]) & 0x7f800000u) == 0x7f800000u ? R8_NAN : (int)c;
        const float a = (v[j] - (float)mean64[j]) * (float)invstd64[j] * gamma[j] + beta[j];
        o[j] = (act && !(a > 0.0f)) ? a * slope : a;
    }
    if (live) {
        codes_store4<VEC>(codes + r * C, col, C, r8_pack4(q));
        if (y) row_store4<RowF32, VEC>(y + r * C, col, C, o);
    }
    if (col % R8_GROUP == 0) exps[r * G + col / R8_GROUP] = (uint8_t)e;
}

template <bool VEC>
__global__ __launch_bounds__(BN_THREADS) void bn_apply8_kernel(
    const float *__restrict__ z, i64 rows, int C, BnQuarters quarters, const double *__restrict__ terms64,
    const float *__restrict__ weight, const float *__restrict__ bias, int act, float slope,
    float *__restrict__ y, int8_t *__restrict__ codes, uint8_t *__restrict__ exps)
{
    i64 b0, rend;
    quarters.place(rows, b0, rend);
    const R8Walk w = r8_walk_at<true>(b0, rend, C);
    const int G = (C + R8_GROUP - 1) / R8_GROUP;
    const bool live = w.col < C;
    float gamma[4], beta[4];
    double mean64[4], invstd64[4];
    BnKink kink[4];
    unsigned last[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int c = min(w.col + j, C - 1);
        mean64[j] = terms64[c];
        invstd64[j] = terms64[C + c];
        gamma[j] = weight ? weight[c] : 1.0f;
        beta[j] = bias ? bias[c] : 0.0f;
        kink[j].load(gamma[j], beta[j]);
        last[j] = act ? kink[j].last() : 0x7f800000u;
    }
    auto one = [&](i64 r, const float (&v)[4]) {
        bn_apply8_row<VEC>(v, r, w.col, C, G, live, mean64, invstd64, gamma, beta, kink, last, act, slope, y, codes, exps);
    };
    i64 r = w.r0;
    for (; r + 3 * (i64)w.rstep < w.rend; r += 4 * (i64)w.rstep) {
        float v[4][4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[u][j] = 0.0f;
            if (live) row_load4<RowF32, VEC>(z + (r + (i64)u * w.rstep) * C, w.col, C, v[u]);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) one(r + (i64)u * w.rstep, v[u]);
    }
    for (; r < w.rend; r += w.rstep) {
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (live) row_load4<RowF32, VEC>(z + r * C, w.col, C, v);
        one(r, v);
    }
}

// ---- few rows: a whole direction in one launch ---------------------------------------------------
// A workgroup owns a group of 32 columns over all rows: 128 lanes of rows by 8 slots of four columns.  It
// sums its columns (float64, a fixed order: lanes by exchanges, waves through LDS), forms their terms
// and goes over the rows again, which by then lie in its caches.  On the GPU the walk of 4099 rows takes
// 60 us where the three launches it replaces take 13, about 15 ns a row: even at 1024 rows, and the host
// is 13 us a training step ahead (160 -> 147).
constexpr int BN_SMALL_THREADS = 1024, BN_SMALL_LANES = BN_SMALL_THREADS / 8;
constexpr int BN_SMALL_ROWS = 1024;

// Sums of the two values of every column over the workgroup's rows: out[0][column], out[1][column].
__device__ __forceinline__ void bn_small_fold(double (&s)[4], double (&q)[4], double (*red)[8][8], double (*out)[32])
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, slot = threadIdx.x & 7;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int d = 8; d < 64; d <<= 1) {
            s[j] += __shfl_xor(s[j], d, 64);
            q[j] += __shfl_xor(q[j], d, 64);
        }
    if (lane < 8)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            red[wave][slot][j] = s[j];
            red[wave][slot][4 + j] = q[j];
        }
    __syncthreads();
    if (threadIdx.x < 64) {
        const int c = threadIdx.x & 31, which = threadIdx.x >> 5;
        double t = 0.0;
        for (int w = 0; w < BN_SMALL_THREADS / 64; ++w) t += red[w][c / 4][4 * which + c % 4];
        out[which][c] = t;
    }
    __syncthreads();
}

template <bool VEC>
__global__ __launch_bounds__(BN_SMALL_THREADS) void bn_small8_forward_kernel(
    const float *__restrict__ z, int rows, int C, const float *__restrict__ weight, const float *__restrict__ bias,
    float *__restrict__ running_mean, float *__restrict__ running_var, int training, float momentum, float eps,
    int act, float slope, long long *__restrict__ num_batches, float *__restrict__ y, int8_t *__restrict__ codes,
    uint8_t *__restrict__ exps, float *__restrict__ save_invstd)
{
    __shared__ double red[BN_SMALL_THREADS / 64][8][8], sums[2][32];
    __shared__ double terms64[2][32];
    const int col = blockIdx.x * R8_GROUP + 4 * (threadIdx.x & 7), r0 = threadIdx.x >> 3;
    const int G = gridDim.x;
    const bool live = col < C;
    if (num_batches && blockIdx.x == 0 && threadIdx.x == 0) *num_batches += 1;
    auto load = [&](int r, float (&v)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = 0.0f;
        if (live && r < rows) row_load4<RowF32, VEC>(z + (i64)r * C, col, C, v);
    };
    if (training) {
        double s[4] = {0.0, 0.0, 0.0, 0.0}, q[4] = {0.0, 0.0, 0.0, 0.0};
        for (int r = r0; r < rows; r += 4 * BN_SMALL_LANES) {
            float v[4][4];
#pragma unroll
            for (int u = 0; u < 4; ++u) load(r + u * BN_SMALL_LANES, v[u]);
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const double d = (double)v[u][j];
                    s[j] += d;
                    q[j] += d * d;
                }
        }
        bn_small_fold(s, q, red, sums);
    }
    if (threadIdx.x < 32) {
        const int c = blockIdx.x * R8_GROUP + threadIdx.x;
        double mean = 0.0, invstd = 0.0;
        if (c < C) {
            if (training) {
                const double n = (double)rows;
                mean = sums[0][threadIdx.x] / n;
                double var = sums[1][threadIdx.x] / n - mean * mean;
                if (var < 0.0) var = 0.0;
                invstd = 1.0 / sqrt(var + (double)eps);
                if (running_mean) running_mean[c] = (float)((1.0 - (double)momentum) * (double)running_mean[c] + (double)momentum * mean);
                if (running_var) running_var[c] = (float)((1.0 - (double)momentum) * (double)running_var[c] + (double)momentum * (var * n / (n - 1.0)));
            } else {
                mean = (double)running_mean[c];
                invstd = 1.0 / sqrt((double)running_var[c] + (double)eps);
            }
            save_invstd[c] = (float)invstd;
        }
        terms64[0][threadIdx.x] = mean;
        terms64[1][threadIdx.x] = invstd;
    }
    __syncthreads();
    float gamma[4], beta[4];
    double mean64[4], invstd64[4];
    BnKink kink[4];
    unsigned last[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int c = min(col + j, C - 1);
        mean64[j] = terms64[0][4 * (threadIdx.x & 7) + j];
        invstd64[j] = terms64[1][4 * (threadIdx.x & 7) + j];
        gamma[j] = weight ? weight[c] : 1.0f;
        beta[j] = bias ? bias[c] : 0.0f;
        kink[j].load(gamma[j], beta[j]);
        last[j] = act ? kink[j].last() : 0x7f800000u;
    }
    for (int r = r0; r < rows; r += 2 * BN_SMALL_LANES) {
        float v[2][4];
#pragma unroll
        for (int u = 0; u < 2; ++u) load(r + u * BN_SMALL_LANES, v[u]);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int ru = r + u * BN_SMALL_LANES;
            if (ru >= rows) break;
            bn_apply8_row<VEC>(v[u], ru, col, C, G, live, mean64, invstd64, gamma, beta, kink, last, act, slope, y, codes, exps);
        }
    }
}

template <bool VEC>
__global__ __launch_bounds__(BN_SMALL_THREADS) void bn_small8_backward_kernel(
    const float *__restrict__ gy, const int8_t *__restrict__ codes, const uint8_t *__restrict__ exps, int rows, int C,
    const float *__restrict__ weight, const float *__restrict__ bias, const float *__restrict__ save_invstd,
    int training, int act, float slope, float *__restrict__ gz, float *__restrict__ grad_weight, float *__restrict__ grad_bias)
{
    __shared__ double red[BN_SMALL_THREADS / 64][8][8], sums[2][32];
    const int col = blockIdx.x * R8_GROUP + 4 * (threadIdx.x & 7), r0 = threadIdx.x >> 3, G = gridDim.x;
    const bool live = col < C;
    BnKink kink[4];
    float k[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int c = min(col + j, C - 1);
        const float gamma = weight ? weight[c] : 1.0f;
        kink[j].load(gamma, bias ? bias[c] : 0.0f);
        k[j] = gamma * save_invstd[c];
    }
    auto load = [&](int r, float (&g)[4], unsigned &q, int &e) {
#pragma unroll
        for (int j = 0; j < 4; ++j) g[j] = 0.0f;
        q = 0u;
        e = 0;
        if (live && r < rows) {
            row_load4<RowF32, VEC>(gy + (i64)r * C, col, C, g);
            q = codes_load4<VEC>(codes + (i64)r * C, col, C);
            e = exps[(i64)r * G + blockIdx.x];
        }
    };
    auto gate = [&](float (&g)[4], unsigned q, int e, float (&zh)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            zh[j] = r8_decode(r8_byte(q, j), e);
            if (act && !kink[j].on(zh[j])) g[j] *= slope;
        }
    };
    double s[4] = {0.0, 0.0, 0.0, 0.0}, t[4] = {0.0, 0.0, 0.0, 0.0};
    for (int r = r0; r < rows; r += 2 * BN_SMALL_LANES) {
        float g[2][4], zh[4];
        unsigned q[2];
        int e[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) load(r + u * BN_SMALL_LANES, g[u], q[u], e[u]);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            gate(g[u], q[u], e[u], zh);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[j] += (double)g[u][j];
                t[j] += (double)g[u][j] * (double)zh[j];
            }
        }
    }
    bn_small_fold(s, t, red, sums);
    if (threadIdx.x < 32 && (int)(blockIdx.x * R8_GROUP + threadIdx.x) < C) {
        const int c = blockIdx.x * R8_GROUP + threadIdx.x;
        if (grad_bias) grad_bias[c] = (float)sums[0][threadIdx.x];
        if (grad_weight) grad_weight[c] = (float)sums[1][threadIdx.x];
    }
    if (!gz || !live) return;
    float m_g[4], m_gz[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        m_g[j] = (float)(sums[0][4 * (threadIdx.x & 7) + j] / (double)rows);
        m_gz[j] = (float)(sums[1][4 * (threadIdx.x & 7) + j] / (double)rows);
    }
    for (int r = r0; r < rows; r += 2 * BN_SMALL_LANES) {
        float g[2][4], zh[4];
        unsigned q[2];
        int e[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) load(r + u * BN_SMALL_LANES, g[u], q[u], e[u]);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int ru = r + u * BN_SMALL_LANES;
            if (ru >= rows) break;
            gate(g[u], q[u], e[u], zh);
#pragma unroll
            for (int j = 0; j < 4; ++j) g[u][j] = training ? (g[u][j] - m_g[j] - zh[j] * m_gz[j]) * k[j] : g[u][j] * k[j];
            row_store4<RowF32, VEC>(gz + (i64)ru * C, col, C, g[u]);
        }
    }
}

// Column sums of g and g * zhat from the codes (bn_grad_sums_kernel's, with zhat as it is read back).
template <int VW>
__global__ __launch_bounds__(BN_THREADS) void bn_grad_sums8_kernel(
    const float *__restrict__ gy, const int8_t *__restrict__ codes, const uint8_t *__restrict__ exps,
    i64 rows, int C, i64 rows_per_block, const float *__restrict__ weight, const float *__restrict__ bias,
    int act, float slope, double *__restrict__ partial)
{
    const BnWalk w = bn_walk<VW>(rows, C, rows_per_block, blockIdx.x);
    const int G = (C + R8_GROUP - 1) / R8_GROUP;
    double s[VW], q[VW];
#pragma unroll
    for (int j = 0; j < VW; ++j) s[j] = q[j] = 0.0;
    if (w.col >= 0) {
        BnKink kink[VW];
#pragma unroll
        for (int j = 0; j < VW; ++j) kink[j].load(weight ? weight[w.col + j] : 1.0f, bias ? bias[w.col + j] : 0.0f);
        const int grp = w.col / R8_GROUP;
        auto load = [&](i64 r, float (&g)[VW], unsigned &c, int &e) {
            bn_load<VW>(gy + r * C + w.col, g);
            if constexpr (VW == 4) c = *reinterpret_cast<const unsigned *>(codes + r * C + w.col);
            else c = (unsigned)(uint8_t)codes[r * C + w.col];
            e = exps[r * G + grp];
        };
        auto add = [&](const float (&g)[VW], unsigned c, int e) {
#pragma unroll
            for (int j = 0; j < VW; ++j) {
                const float zh = r8_decode(r8_byte(c, j), e);
                const float gg = (act && !kink[j].on(zh)) ? g[j] * slope : g[j];
                s[j] += (double)gg;
                q[j] += (double)gg * (double)zh;
            }
        };
        i64 r = w.r0;
        for (; r + 3 * (i64)w.rstep < w.rend; r += 4 * (i64)w.rstep) {
            float g[4][VW];
            unsigned c[4];
            int e[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) load(r + (i64)u * w.rstep, g[u], c[u], e[u]);
#pragma unroll
            for (int u = 0; u < 4; ++u) add(g[u], c[u], e[u]);
        }
        for (; r < w.rend; r += w.rstep) {
            float g[VW];
            unsigned c;
            int e;
            load(r, g, c, e);
            add(g, c, e);
        }
    }
    bn_block_fold<VW>(s, q, C, partial);
}

// grad_z from the codes (bn_grad_apply_kernel's formula).
template <int VW>
__global__ __launch_bounds__(BN_THREADS) void bn_grad_apply8_kernel(
    const float *__restrict__ gy, const int8_t *__restrict__ codes, const uint8_t *__restrict__ exps,
    i64 rows, int C, BnQuarters quarters, const float *__restrict__ save_invstd,
    const float *__restrict__ weight, const float *__restrict__ bias, int act, float slope,
    const float *__restrict__ col_terms, int training, float *__restrict__ gz)
{
    i64 b0, rend;
    quarters.place(rows, b0, rend);
    BnWalk w = bn_walk<VW>(rend - b0, C, rend - b0, 0);
    w.r0 += b0;
    w.rend += b0;
    if (w.col < 0) return;
    const int G = (C + R8_GROUP - 1) / R8_GROUP, grp = w.col / R8_GROUP;
    float m_g[VW], m_gz[VW], k[VW];
    BnKink kink[VW];
#pragma unroll
    for (int j = 0; j < VW; ++j) {
        const float gamma = weight ? weight[w.col + j] : 1.0f;
        kink[j].load(gamma, bias ? bias[w.col + j] : 0.0f);
        m_g[j] = training ? col_terms[w.col + j] : 0.0f;
        m_gz[j] = training ? col_terms[C + w.col + j] : 0.0f;
        k[j] = gamma * save_invstd[w.col + j];
    }
    auto load = [&](i64 r, float (&g)[VW], unsigned &c, int &e) {
        bn_load<VW>(gy + r * C + w.col, g);
        if constexpr (VW == 4) c = *reinterpret_cast<const unsigned *>(codes + r * C + w.col);
        else c = (unsigned)(uint8_t)codes[r * C + w.col];
        e = exps[r * G + grp];
    };
    auto store = [&](i64 r, const float (&g)[VW], unsigned c, int e) {
        float v[VW];
#pragma unroll
        for (int j = 0; j < VW; ++j) {
            const float zh = r8_decode(r8_byte(c, j), e);
            const float gg = (act && !kink[j].on(zh)) ? g[j] * slope : g[j];
            // (running statistics: m_gz is zero, and a value that is not finite stays with its own row)
            v[j] = training ? (gg - m_g[j] - zh * m_gz[j]) * k[j] : gg * k[j];
        }
        if constexpr (VW == 4) {
            const r8_f4 t = {v[0], v[1], v[2], v[3]};
            r8_stream(reinterpret_cast<r8_f4 *>(gz + r * C + w.col), t);
        } else {
            bn_store<VW>(gz + r * C + w.col, v);
        }
    };
    i64 r = w.r0;
    for (; r + 3 * (i64)w.rstep < w.rend; r += 4 * (i64)w.rstep) {
        float g[4][VW];
        unsigned c[4];
        int e[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) load(r + (i64)u * w.rstep, g[u], c[u], e[u]);
#pragma unroll
        for (int u = 0; u < 4; ++u) store(r + (i64)u * w.rstep, g[u], c[u], e[u]);
    }
    for (; r < w.rend; r += w.rstep) {
        float g[VW];
        unsigned c;
        int e;
        load(r, g, c, e);
        store(r, g, c, e);
    }
}

static size_t bn_partial_bytes(int C) { return align_up((size_t)BN_MAX_BLOCKS * 2 * (size_t)C * sizeof(double)); }

}  // namespace mvf

using namespace mvf;

extern "C" size_t mvf_batch_norm_act_workspace_bytes(int32_t C)
{
    if (C < 1) return 0;
    return bn_partial_bytes(C) + align_up(2 * (size_t)C * sizeof(float));
}

extern "C" int mvf_batch_norm_act_forward(
    const float *z, int64_t rows, int32_t C, const float *weight, const float *bias,
    float *running_mean, float *running_var, int32_t training, float momentum, float eps,
    int32_t act, float slope, float *y, float *save_mean, float *save_invstd,
    const double *col_sums, int32_t n_col_sums, void *workspace, size_t workspace_bytes, void *stream)
{
    MVF_REQUIRE(rows >= 1 && C >= 1, "batch_norm_act_forward: rows and C must be positive");
    MVF_REQUIRE(z && y && save_mean && save_invstd, "batch_norm_act_forward: null argument");
    MVF_REQUIRE(training || (running_mean && running_var),
                "batch_norm_act_forward: running statistics are needed outside train mode");
    MVF_REQUIRE(!training || rows > 1, "batch_norm_act_forward: more than one row per channel is needed in train mode");
    MVF_REQUIRE(!training || col_sums || (workspace && workspace_bytes >= mvf_batch_norm_act_workspace_bytes(C)),
                "batch_norm_act_forward: workspace too small");
    MVF_REQUIRE(!col_sums || n_col_sums >= 1, "batch_norm_act_forward: column sums without partial rows");
    hipStream_t st = (hipStream_t)stream;
    const bool vec = C % 4 == 0 && (uintptr_t)z % 16 == 0 && (uintptr_t)y % 16 == 0;
    const BnGrid g = bn_grid(rows, C, vec ? 4 : 1);
    if (training) {
        const double *partial = col_sums;
        int nblk = n_col_sums;
        if (!col_sums) {
            double *mine = (double *)workspace;
            if (vec) hipLaunchKernelGGL(bn_sums_kernel<4>, g.grid, dim3(BN_THREADS), 0, st, z, (i64)rows, C, g.rows_per_block, mine);
            else hipLaunchKernelGGL(bn_sums_kernel<1>, g.grid, dim3(BN_THREADS), 0, st, z, (i64)rows, C, g.rows_per_block, mine);
            partial = mine;
            nblk = g.nblk;
        }
        hipLaunchKernelGGL(bn_stats_kernel, dim3(cdiv(C, BN_FOLD_COLS)), dim3(BN_THREADS), 0, st,
                           partial, nblk, C, (i64)rows, eps, momentum,
                           running_mean, running_var, save_mean, save_invstd, (double *)nullptr, (long long *)nullptr);
    } else {
        hipLaunchKernelGGL(bn_running_terms_kernel, dim3(cdiv(C, 256)), dim3(256), 0, st,
                           (const float *)running_mean, (const float *)running_var, C, eps, save_mean, save_invstd,
                           (double *)nullptr);
    }
    if (vec)
        hipLaunchKernelGGL(bn_apply_kernel<4>, g.grid, dim3(BN_THREADS), 0, st, z, (i64)rows, C, g.rows_per_block,
                           (const float *)save_mean, (const float *)save_invstd, weight, bias, act, slope, y);
    else
        hipLaunchKernelGGL(bn_apply_kernel<1>, g.grid, dim3(BN_THREADS), 0, st, z, (i64)rows, C, g.rows_per_block,
                           (const float *)save_mean, (const float *)save_invstd, weight, bias, act, slope, y);
    MVF_LAUNCH_CHECK();
    return MVF_OK;
}

extern "C" int mvf_batch_norm_act_backward(
    const float *grad_y, const float *z, int64_t rows, int32_t C, const float *weight, const float *bias,
    const float *save_mean, const float *save_invstd, int32_t training, int32_t act, float slope,
    float *grad_z, float *grad_weight, float *grad_bias,
    void *workspace, size_t workspace_bytes, void *stream)
{
    MVF_REQUIRE(rows >= 1 && C >= 1, "batch_norm_act_backward: rows and C must be positive");
    MVF_REQUIRE(grad_y && z && save_mean && save_invstd && grad_z, "batch_norm_act_backward: null argument");
    MVF_REQUIRE(workspace && workspace_bytes >= mvf_batch_norm_act_workspace_bytes(C),
                "batch_norm_act_backward: workspace too small");
    hipStream_t st = (hipStream_t)stream;
    const bool vec = C % 4 == 0 && (uintptr_t)z % 16 == 0 && (uintptr_t)grad_y % 16 == 0 && (uintptr_t)grad_z % 16 == 0;
    const BnGrid g = bn_grid(rows, C, vec ? 4 : 1);
    double *partial = (double *)workspace;
    float *col_terms = (float *)((char *)workspace + bn_partial_bytes(C));
    if (training || grad_weight || grad_bias) {
        if (vec)
            hipLaunchKernelGGL(bn_grad_sums_kernel<4>, g.grid, dim3(BN_THREADS), 0, st, grad_y, z, (i64)rows, C,
                               g.rows_per_block, save_mean, save_invstd, weight, bias, act, slope, partial);
        else
            hipLaunchKernelGGL(bn_grad_sums_kernel<1>, g.grid, dim3(BN_THREADS), 0, st, grad_y, z, (i64)rows, C,
                               g.rows_per_block, save_mean, save_invstd, weight, bias, act, slope, partial);
        hipLaunchKernelGGL(bn_grad_terms_kernel, dim3(cdiv(C, BN_FOLD_COLS)), dim3(BN_THREADS), 0, st,
                           (const double *)partial, g.nblk, C, (i64)rows, grad_weight, grad_bias, col_terms);
    }
    if (vec)
        hipLaunchKernelGGL(bn_grad_apply_kernel<4>, g.grid, dim3(BN_THREADS), 0, st, grad_y, z, (i64)rows, C,
                           g.rows_per_block, save_mean, save_invstd, weight, bias, act, slope,
                           (const float *)col_terms, training, grad_z);
    else
        hipLaunchKernelGGL(bn_grad_apply_kernel<1>, g.grid, dim3(BN_THREADS), 0, st, grad_y, z, (i64)rows, C,
                           g.rows_per_block, save_mean, save_invstd, weight, bias, act, slope,
                           (const float *)col_terms, training, grad_z);
    MVF_LAUNCH_CHECK();
    return MVF_OK;
}

extern "C" size_t mvf_batch_norm_act8_workspace_bytes(int32_t C)
{
    if (C < 1) return 0;
    return mvf_batch_norm_act_workspace_bytes(C) + align_up(2 * (size_t)C * sizeof(double));
}

namespace mvf {

Bn8Workspace bn8_workspace(void *workspace, int C)
{
    char *p = (char *)workspace;
    return {(double *)p, (float *)(p + bn_partial_bytes(C)), (double *)(p + mvf_batch_norm_act_workspace_bytes(C))};
}

void bn8_statistics(const float *z, i64 rows, int C, float *running_mean, float *running_var, int training, float momentum,
                    float eps, const double *col_sums, int n_col_sums, long long *num_batches, const Bn8Workspace &w,
                    float *save_invstd, hipStream_t st)
{
    if (!training) {
        hipLaunchKernelGGL(bn_running_terms_kernel, dim3(cdiv(C, 256)), dim3(256), 0, st, (const float *)running_mean,
                           (const float *)running_var, C, eps, w.terms, save_invstd, w.terms64);
        return;
    }
    const double *partial = col_sums;
    int nblk = n_col_sums;
    if (!col_sums) {
        const bool vec = C % 4 == 0 && (uintptr_t)z % 16 == 0;
        const BnGrid g = bn_grid(rows, C, vec ? 4 : 1);
        if (vec) hipLaunchKernelGGL(bn_sums_kernel<4>, g.grid, dim3(BN_THREADS), 0, st, z, rows, C, g.rows_per_block, w.partial);
        else hipLaunchKernelGGL(bn_sums_kernel<1>, g.grid, dim3(BN_THREADS), 0, st, z, rows, C, g.rows_per_block, w.partial);
        partial = w.partial;
        nblk = g.nblk;
    }
    hipLaunchKernelGGL(bn_stats_kernel, dim3(cdiv(C, BN_FOLD_COLS)), dim3(BN_THREADS), 0, st, partial, nblk, C, rows, eps,
                       momentum, running_mean, running_var, w.terms, save_invstd, w.terms64, num_batches);
}

void bn8_grad_terms(const Bn8Workspace &w, int nblk, int C, i64 rows, float *grad_weight, float *grad_bias, hipStream_t st)
{
    hipLaunchKernelGGL(bn_grad_terms_kernel, dim3(cdiv(C, BN_FOLD_COLS)), dim3(BN_THREADS), 0, st, (const double *)w.partial,
                       nblk, C, rows, grad_weight, grad_bias, w.terms);
}

}  // namespace mvf

extern "C" int mvf_batch_norm_act8_forward(
    const float *z, int64_t rows, int32_t C, const float *weight, const float *bias,
    float *running_mean, float *running_var, int32_t training, float momentum, float eps,
    int32_t act, float slope, int64_t *num_batches, float *y, int8_t *codes, uint8_t *exps, float *save_invstd,
    const double *col_sums, int32_t n_col_sums, void *workspace, size_t workspace_bytes, void *stream)
{
    MVF_REQUIRE(rows >= 1 && C >= 1, "batch_norm_act8_forward: rows and C must be positive");
    MVF_REQUIRE(z && codes && exps && save_invstd, "batch_norm_act8_forward: null argument");
    MVF_REQUIRE(training || (running_mean && running_var),
                "batch_norm_act8_forward: running statistics are needed outside train mode");
    MVF_REQUIRE(!training || rows > 1, "batch_norm_act8_forward: more than one row per channel is needed in train mode");
    MVF_REQUIRE(workspace && workspace_bytes >= mvf_batch_norm_act8_workspace_bytes(C),
                "batch_norm_act8_forward: workspace too small");
    MVF_REQUIRE(!col_sums || n_col_sums >= 1, "batch_norm_act8_forward: column sums without partial rows");
    hipStream_t st = (hipStream_t)stream;
    const bool vec = C % 4 == 0 && (uintptr_t)z % 16 == 0 && (uintptr_t)y % 16 == 0 && (uintptr_t)codes % 4 == 0;
    if (rows <= BN_SMALL_ROWS && !col_sums) {
#define MVF_BN_SMALL(V_)                                                                                            \
    hipLaunchKernelGGL(bn_small8_forward_kernel<V_>, dim3(r8_groups(C)), dim3(BN_SMALL_THREADS), 0, st, z, (int)rows, C, weight, \
                       bias, running_mean, running_var, training, momentum, eps, act, slope, (long long *)num_batches, y, codes, \
                       exps, save_invstd)
        if (vec) MVF_BN_SMALL(true);
        else MVF_BN_SMALL(false);
#undef MVF_BN_SMALL
        MVF_LAUNCH_CHECK();
        return MVF_OK;
    }
    const Bn8Workspace w = bn8_workspace(workspace, C);
    bn8_statistics(z, rows, C, running_mean, running_var, training, momentum, eps, col_sums, n_col_sums, (long long *)num_batches, w,
                   save_invstd, st);
    const double *terms64 = w.terms64;
    // the ranges of the pass over z that made the statistics
    const BnGrid g = bn_grid(rows, C, C % 4 == 0 && (uintptr_t)z % 16 == 0 ? 4 : 1);
    const int slots = r8_groups(C) * 8, cw = slots < BN_THREADS ? slots : BN_THREADS;
    const BnQuarters quarters = bn_quarters(g, BN_THREADS / cw);
    const dim3 grid(4 * (unsigned)g.nblk, (unsigned)((slots + BN_THREADS - 1) / BN_THREADS));
    if (vec)
        hipLaunchKernelGGL(bn_apply8_kernel<true>, grid, dim3(BN_THREADS), 0, st, z, (i64)rows, C, quarters,
                           terms64, weight, bias,
                           act, slope, y, codes, exps);
    else
        hipLaunchKernelGGL(bn_apply8_kernel<false>, grid, dim3(BN_THREADS), 0, st, z, (i64)rows, C, quarters,
                           terms64, weight, bias,
                           act, slope, y, codes, exps);
    MVF_LAUNCH_CHECK();
    return MVF_OK;
}

extern "C" int mvf_batch_norm_act8_backward(
    const float *grad_y, const int8_t *codes, const uint8_t *exps, int64_t rows, int32_t C,
    const float *weight, const float *bias, const float *save_invstd, int32_t training, int32_t act, float slope,
    float *grad_z, float *grad_weight, float *grad_bias,
    void *workspace, size_t workspace_bytes, void *stream)
{
    MVF_REQUIRE(rows >= 1 && C >= 1, "batch_norm_act8_backward: rows and C must be positive");
    MVF_REQUIRE(grad_y && codes && exps && save_invstd, "batch_norm_act8_backward: null argument");
    MVF_REQUIRE(workspace && workspace_bytes >= mvf_batch_norm_act8_workspace_bytes(C),
                "batch_norm_act8_backward: workspace too small");
    hipStream_t st = (hipStream_t)stream;
    const bool vec = C % 4 == 0 && (uintptr_t)grad_y % 16 == 0 && (uintptr_t)grad_z % 16 == 0 && (uintptr_t)codes % 4 == 0;
    if (rows <= BN_SMALL_ROWS) {
#define MVF_BN_SMALL(V_)                                                                                            \
    hipLaunchKernelGGL(bn_small8_backward_kernel<V_>, dim3(r8_groups(C)), dim3(BN_SMALL_THREADS), 0, st, grad_y, codes, exps, \
                       (int)rows, C, weight, bias, save_invstd, training, act, slope, grad_z, grad_weight, grad_bias)
        if (vec) MVF_BN_SMALL(true);
        else MVF_BN_SMALL(false);
#undef MVF_BN_SMALL
        MVF_LAUNCH_CHECK();
        return MVF_OK;
    }
    const BnGrid g = bn_grid(rows, C, vec ? 4 : 1);
    const Bn8Workspace ws8 = bn8_workspace(workspace, C);
    double *partial = ws8.partial;
    float *col_terms = ws8.terms;
    if ((training && grad_z) || grad_weight || grad_bias) {
        if (vec)
            hipLaunchKernelGGL(bn_grad_sums8_kernel<4>, g.grid, dim3(BN_THREADS), 0, st, grad_y, codes, exps, (i64)rows, C,
                               g.rows_per_block, weight, bias, act, slope, partial);
        else
            hipLaunchKernelGGL(bn_grad_sums8_kernel<1>, g.grid, dim3(BN_THREADS), 0, st, grad_y, codes, exps, (i64)rows, C,
                               g.rows_per_block, weight, bias, act, slope, partial);
        bn8_grad_terms(ws8, g.nblk, C, rows, grad_weight, grad_bias, st);
    }
    if (grad_z) {
        const int CV = C / (vec ? 4 : 1), cw = CV < BN_THREADS ? CV : BN_THREADS;
        const BnQuarters quarters = bn_quarters(g, BN_THREADS / cw);
        const dim3 grid(4 * (unsigned)g.nblk, g.grid.y);
        if (vec)
            hipLaunchKernelGGL(bn_grad_apply8_kernel<4>, grid, dim3(BN_THREADS), 0, st, grad_y, codes, exps, (i64)rows, C,
                               quarters, save_invstd, weight, bias, act, slope, (const float *)col_terms, training, grad_z);
        else
            hipLaunchKernelGGL(bn_grad_apply8_kernel<1>, grid, dim3(BN_THREADS), 0, st, grad_y, codes, exps, (i64)rows, C,
                               quarters, save_invstd, weight, bias, act, slope, (const float *)col_terms, training, grad_z);
    }
    MVF_LAUNCH_CHECK();
    return MVF_OK;
}
