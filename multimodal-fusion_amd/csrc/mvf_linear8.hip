// A Linear over many float32 rows together with what its 8-bit kept rows need (mvf_rows8.h), one pass over
// the rows each way, at most 64 columns in and out:
//
//   forward   y = v W^T (+ b) and the codes, with v = x (codes of x), or v = act(bn(z)) (codes of the
//             normalised z): the activated rows exist in LDS only.  The products and their order
//             are those of mvf_linear.hip: the same bits.
//   backward  of the Linear: grad_x = g W, grad_W = g^T xq and grad_b = sum g from one read of g;
//             of BatchNorm + LeakyReLU + Linear: a pass of reductions that leaves grad_W and the column sums
//             of BatchNorm's backward, and a pass that forms g W and writes grad_z.
//
// Bound by HBM (per row of I -> O columns: forward 4 (I + O) + I bytes, backward 4 (I + O) + I, with
// BatchNorm 4 O + I more).  Structure of mvf_linear.hip: a wave owns tiles of 32 rows, loaded in
// memory order a tile ahead, parked in its own LDS region and read back as operands.  One workgroup per
// compute unit, two or three waves per SIMD: one's vector work fills the other's matrix instructions;
// for their registers' sake W lies in LDS as well, read four operands at a time.  In memory order a
// lane has the same four columns in all its pieces (a row of 8, 16, 32 or 64 columns is 2, 4, 8 or 16
// pieces of 16 bytes), so BatchNorm's column terms stay in registers, a group of 32 columns is 8
// neighbouring lanes, and codes are stored 256 bytes at a time.  The weight gradient runs on the bf16
// matrix cores with exact parts (mvf_bf16x3.h): the tile's g column by column out of LDS, cut into three
// parts; a value read back from 8 bits is one bf16.
//
// 2 M rows of 64 -> 64 columns: a Linear forward and backward 496 to 515 us by box (4.6 TB/s; as separate launches
// of product, packing, grad_x and grad_W 671 us); behind BatchNorm 832 to 870 us.  A kernel trace, in which every
// launch is slower, splits the latter into 93 us of statistics, 370 forward, 215 for the sums' pass, 246 for grad_z
// and 23 for three folds.  Not bound by memory alone: the Linear's forward takes 286 us in the trace, 268 without its
// packing, 261 without storing y and 220 without its products.  Two waves per SIMD leave matrix and vector work, and
// the way through LDS, partly one behind the other, and the registers allow no third (wave
// priorities around the products: nothing).
#include "mvf_bf16x3.h"
#include "mvf_bn_kink.h"
#include "mvf_norm.h"
#include "mvf_rows8.h"

namespace mvf {

constexpr int L8_FWD_THREADS = 512;         // (a third wave per SIMD gained nothing)
// (two waves per SIMD where more than 32 columns on a side leave no registers for a third)
constexpr int l8_bwd_threads(int KO, int KI) { return KO <= 4 && KI <= 4 ? 768 : 512; }
constexpr int T8_THREADS = 512;
constexpr int L8_ROWS = 32;                 // rows per tile
constexpr int L8_MAX_WGS = 256;             // one per compute unit

typedef float l8_f4 __attribute__((ext_vector_type(4)));
typedef float l8_f2 __attribute__((ext_vector_type(2)));

struct L8Bn {                               // BatchNorm + LeakyReLU in front of the Linear
    const float *mean, *invstd;             // float32 [I]
    const double *terms64;                  // [2][I] mean, 1 / spread (forward)
    const float *weight, *bias;             // [I] or NULL
    const float *col_terms;                 // [2][I] column means of g and g * zq (backward)
    int act, training;
    float slope;
};

// LDS written by some lanes of a wave and read by others: the operations of a wave are executed in
// order, the compiler has to keep them so
__device__ __forceinline__ void l8_wave_sync()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// How a tile is done. WHOLE: all its rows exist (and the output's pieces fill the lanes); NEXT: another
// one follows.
template <bool W, bool N> struct L8Tile { static constexpr bool WHOLE = W, NEXT = N; };

// An LDS offset the compiler takes for new: operands read at it stay in LDS instead of being moved
// out of the tile loop into registers.
__device__ __forceinline__ unsigned l8_fresh(unsigned at)
{
    asm volatile("" : "+v"(at));
    return at;
}

// largest value of the lanes that hold a group of 32 columns (rows of fewer: of the row)
template <int IQ> __device__ __forceinline__ unsigned l8_group_max(unsigned v)
{
    if constexpr (IQ >= 8) return r8_max8(v);
    else if constexpr (IQ >= 4) return r8_max4(v);
    else return max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0xb1, 0xf, 0xf, true));
}

// ---- forward ----------------------------------------------------------------------------------
// EXACT: O = 32 NO columns out, a constant.
template <int KQ, int NO, bool TAIL, bool STATS, bool EXACT>
__global__ __launch_bounds__(L8_FWD_THREADS) void linear8_forward_kernel(
    const float *x, const float *W, const float *bias, int O_, i64 rows,
    L8Bn bn, float *y, int8_t *codes, uint8_t *exps, double *col_sums)
{
    constexpr int I = 8 * KQ, IQ = 2 * KQ, HALF = 4 * KQ, GR = I > 32 ? 2 : 1;
    const int O = EXACT ? 32 * NO : O_;
    constexpr int PITCH_I = I * 4 + 16, THREADS = L8_FWD_THREADS, WAVES = THREADS / 64;
    __shared__ __attribute__((aligned(16))) char lds[WAVES][L8_ROWS * (64 * 4 + 16)];
    __shared__ __attribute__((aligned(16))) char wlds[32 * NO * PITCH_I];
    __shared__ __attribute__((aligned(16))) float blds[32 * NO];
    // BatchNorm's terms of the columns: float64 mean and 1 / spread; the same in float32, weight, bias;
    // the kink's sign, place and last value
    __shared__ __attribute__((aligned(16))) double tlds[TAIL ? 2 * I : 1];
    __shared__ __attribute__((aligned(16))) float flds[TAIL ? 7 * I : 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 31, kh = lane >> 5;
    const int oq = O >> 2;
    const unsigned pitch_o = (unsigned)O * 4u + 16u;
    char *buf = lds[wave];

    // W as rows (zeros past O): the first operand, lane = output channel, k = the lane half's columns
    for (int i = threadIdx.x; i < 32 * NO * I; i += THREADS)
        *(float *)(wlds + i / I * PITCH_I + i % I * 4) = i / I < O ? W[i] : 0.0f;
    if (threadIdx.x < 32 * NO) blds[threadIdx.x] = bias && (int)threadIdx.x < O ? bias[threadIdx.x] : 0.0f;
    if constexpr (TAIL) {
        if (threadIdx.x < I) {
            const int c = threadIdx.x;
            const float gamma = bn.weight ? bn.weight[c] : 1.0f, beta = bn.bias ? bn.bias[c] : 0.0f;
            BnKink k;
            k.load(gamma, beta);
            tlds[c] = bn.terms64[c];
            tlds[I + c] = bn.terms64[I + c];
            flds[c] = bn.mean[c];
            flds[I + c] = bn.invstd[c];
            flds[2 * I + c] = gamma;
            flds[3 * I + c] = beta;
            flds[4 * I + c] = k.sign;
            flds[5 * I + c] = k.at;
            flds[6 * I + c] = __uint_as_float(bn.act ? k.last() : 0x7f800000u);
        }
    }
    __syncthreads();
    const unsigned w_at = (unsigned)(n * PITCH_I + kh * HALF * 4);
    unsigned out_at[4 * NO];
#pragma unroll
    for (int j = 0; j < 4 * NO; ++j) {
        const unsigned f = (unsigned)lane + 64u * j, r = f / (unsigned)oq;
        out_at[j] = r * pitch_o + (f - r * oq) * 16u;
    }
    // the lane's columns in memory order, and its row in the first piece
    const int col = 4 * (lane % IQ), row0 = lane / IQ;
    const i64 nfull = rows / L8_ROWS;       // whole tiles; the rows behind them are a tile of their own
    const int rest = (int)(rows - nfull * L8_ROWS);
    const i64 wid = (i64)blockIdx.x * WAVES + wave, nwaves = (i64)gridDim.x * WAVES;
    l8_f4 g[KQ];
    auto load_tile = [&](i64 t, int live) {
        const l8_f4 *src = (const l8_f4 *)(x + (size_t)t * L8_ROWS * I);
#pragma unroll
        for (int j = 0; j < KQ; ++j) {
            const int f = lane + 64 * j;
            g[j] = src[live == L8_ROWS || f < live * IQ ? f : live * IQ - 1];
        }
    };
    // column sums of y and y * y (STATS): lane = column, over every row of the lane half's share; float64
    // from the first addition on, because sum(y^2) / n - mean^2 cancels when a column's mean is large
    double sum1 = 0.0, sum2 = 0.0;
    const int sc = NO == 2 ? lane : n, srows = NO == 2 ? L8_ROWS : L8_ROWS / 2, sr0 = NO == 2 ? 0 : kh * srows;

    // One tile.  WHOLE: all its rows exist and O is a multiple of 32, so that every store of the main loop is
    // unconditional: a wait for the next tile's loads can then leave this tile's stores behind.
    auto tile = [&](i64 t, int live, i64 next, auto how) {
        constexpr bool WHOLE = decltype(how)::WHOLE;
        unsigned *qdst = (unsigned *)(codes + (size_t)t * L8_ROWS * I);
        uint8_t *edst = exps + (size_t)t * L8_ROWS * GR;
        float terms[7][4];          // mean, 1 / spread, gamma, beta, kink
        double terms64[2][4];
        if constexpr (TAIL) {
            const int c = (int)l8_fresh((unsigned)col);
#pragma unroll
            for (int i = 0; i < 7; ++i) {
                const l8_f4 v = *(const l8_f4 *)(flds + i * I + c);
#pragma unroll
                for (int k = 0; k < 4; ++k) terms[i][k] = v[k];
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) terms64[i][k] = tlds[i * I + c + k];
        }
#pragma unroll
        for (int j = 0; j < KQ; ++j) {
            const int r = row0 + j * (64 / IQ);
            float v[4] = {g[j][0], g[j][1], g[j][2], g[j][3]};
            int q[4], e;
            if constexpr (TAIL) {
                double zh[4];
                float zf[4];
                unsigned m = 0;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    zh[k] = ((double)v[k] - terms64[0][k]) * terms64[1][k];
                    zf[k] = (float)zh[k];
                    m = BnKink::most(m, zf[k], __float_as_uint(terms[6][k]));
                }
                e = r8_exponent(l8_group_max<IQ>(m), R8_E_MAX);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float c = (float)rint(ldexp(zh[k], R8_BIAS - e));
                    if (bn.act)
                        c = BnKink{terms[4][k], terms[5][k]}.side(c, zh[k] * (double)terms[2][k] + (double)terms[3][k] > 0.0, e);
                    c = fminf(fmaxf(c, -127.0f), 127.0f);
                    q[k] = (__float_as_uint(zf[k]) & 0x7f800000u) == 0x7f800000u ? R8_NAN : (int)c;
                    const float a = (v[k] - terms[0][k]) * terms[1][k] * terms[2][k] + terms[3][k];
                    v[k] = (bn.act && !(a > 0.0f)) ? a * bn.slope : a;
                }
            } else {
                const unsigned m = max(max(r8_magnitude(v[0]), r8_magnitude(v[1])), max(r8_magnitude(v[2]), r8_magnitude(v[3])));
                e = r8_exponent(l8_group_max<IQ>(m), R8_E_MAX);
#pragma unroll
                for (int k = 0; k < 4; ++k) q[k] = r8_encode(v[k], e);
            }
            if (WHOLE || r < live) {
                qdst[lane + 64 * j] = r8_pack4(q);
                edst[r * GR + col / R8_GROUP] = (uint8_t)e;         // (by every lane of the group)
            }
            const l8_f4 p = {v[0], v[1], v[2], v[3]};
            *(l8_f4 *)(buf + r * PITCH_I + col * 4) = p;
        }
        // (fenced: left alone, the scheduler moves the loads down to their use)
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (decltype(how)::NEXT) load_tile(next, L8_ROWS);
        __builtin_amdgcn_sched_barrier(0);
        l8_wave_sync();
        float xv[4 * KQ];
#pragma unroll
        for (int q = 0; q < KQ; ++q) {
            const l8_f4 v = *(const l8_f4 *)(buf + n * PITCH_I + kh * HALF * 4 + 16 * q);
            xv[4 * q] = v[0]; xv[4 * q + 1] = v[1]; xv[4 * q + 2] = v[2]; xv[4 * q + 3] = v[3];
        }
        xty_acc acc[NO];
#pragma unroll
        for (int o = 0; o < NO; ++o)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const l8_f4 b = *(const l8_f4 *)(blds + l8_fresh(4 * kh) + 32 * o + 8 * q);
#pragma unroll
                for (int k = 0; k < 4; ++k) acc[o][4 * q + k] = b[k];
            }
        const char *wp = wlds + l8_fresh(w_at);
#pragma unroll
        for (int q = 0; q < KQ; ++q) {
            l8_f4 w[NO];
#pragma unroll
            for (int o = 0; o < NO; ++o) w[o] = *(const l8_f4 *)(wp + 32 * o * PITCH_I + 16 * q);
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int o = 0; o < NO; ++o)
                    acc[o] = __builtin_amdgcn_mfma_f32_32x32x2f32(w[o][s], xv[4 * q + s], acc[o], 0, 0, 0);
        }
        l8_wave_sync();
#pragma unroll
        for (int o = 0; o < NO; ++o)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int ch = 32 * o + 8 * q + 4 * kh;
                if (ch < O) {
                    const l8_f4 v = {acc[o][4 * q], acc[o][4 * q + 1], acc[o][4 * q + 2], acc[o][4 * q + 3]};
                    *(l8_f4 *)(buf + (unsigned)n * pitch_o + (unsigned)ch * 4u) = v;
                }
            }
        l8_wave_sync();
        l8_f4 *dst = (l8_f4 *)(y + (size_t)t * L8_ROWS * O);
#pragma unroll
        for (int j = 0; j < 4 * NO; ++j) {
            const int f = lane + 64 * j;
            if (WHOLE || f < live * oq) r8_stream(dst + f, *(const l8_f4 *)(buf + out_at[j]));
        }
        if constexpr (STATS) {
            if (sc < O) {
#pragma unroll 8
                for (int r = 0; r < srows; ++r) {
                    const float v = *(const float *)(buf + (unsigned)(sr0 + r) * pitch_o + (unsigned)sc * 4u);
                    const double d = sr0 + r < live ? (double)v : 0.0;
                    sum1 += d;
                    sum2 += d * d;
                }
            }
        }
        l8_wave_sync();
    };
    if (wid < nfull) {
        load_tile(wid, L8_ROWS);
        // (the last tile asks for itself once more, rather than for nothing under a condition)
        // (and the first tile outside the loop: with its stores behind the loads of the second, the loop is
        // entered as it is repeated, and its waits need not allow for fewer)
        i64 t = wid;
        tile(t, L8_ROWS, t + nwaves < nfull ? t + nwaves : t, L8Tile<EXACT, true>());
        for (t += nwaves; t < nfull; t += nwaves) tile(t, L8_ROWS, t + nwaves < nfull ? t + nwaves : t, L8Tile<EXACT, true>());
    }
    if (rest > 0 && wid == nfull % nwaves) {
        load_tile(nfull, rest);
        tile(nfull, rest, 0, L8Tile<false, false>());
    }
    if constexpr (STATS) {
        if constexpr (NO == 1) {
            sum1 += __shfl_xor(sum1, 32, 64);
            sum2 += __shfl_xor(sum2, 32, 64);
        }
        // the workgroup's waves in order
        __syncthreads();
        double *red = (double *)lds[0];
        if (lane < 32 * NO && sc < O) {
            red[wave * 2 * O + sc] = sum1;
            red[wave * 2 * O + O + sc] = sum2;
        }
        __syncthreads();
        if ((int)threadIdx.x < 2 * O) {
            double t = red[threadIdx.x];
            for (int k = 1; k < WAVES; ++k) t += red[k * 2 * O + threadIdx.x];
            col_sums[(size_t)blockIdx.x * 2 * O + threadIdx.x] = t;
        }
    }
}

// ---- backward ---------------------------------------------------------------------------------
enum { L8_LINEAR = 0, L8_APPLY = 1 };

// O <= 8 KO columns of g (EXACT: 8 KO, a constant), I = 8 KI columns of the kept rows.
template <int KO, int KI, int MODE, bool EXACT>
__global__ __launch_bounds__(l8_bwd_threads(KO, KI)) void linear8_backward_kernel(
    const float *gsrc, int O_, const int8_t *codes, const uint8_t *exps,
    const float *W, i64 rows, L8Bn bn, int want_sums, float *grad,
    float *partial, float *partial_sums)
{
    constexpr int I = 8 * KI, IQ = 2 * KI, GR = I > 32 ? 2 : 1;
    constexpr int THREADS = l8_bwd_threads(KO, KI), WAVES = THREADS / 64;
    const int O = EXACT ? 8 * KO : O_;
    constexpr int NI = I > 32 ? 2 : 1, NA = KO > 4 ? 2 : 1;
    constexpr int PITCH_I = I * 4 + 16;
    constexpr int PITCH_W = KO * 8 * 4 + 16;
    constexpr bool XTY = MODE != L8_APPLY;
    constexpr int PITCH_Q = I * 2 + 16, PLANE = L8_ROWS * PITCH_Q;
    constexpr int TILE = L8_ROWS * ((KO * 8 > I ? KO * 8 : I) * 4 + 16);
    constexpr int REGION = TILE + (XTY ? PLANE : 0);
    constexpr int FOLD = XTY ? (NA * NI * 1024 + WAVES * 64) * 4 : 0;
    constexpr int LDS = WAVES * REGION > FOLD ? WAVES * REGION : FOLD;
    __shared__ __attribute__((aligned(16))) char lds[LDS];
    __shared__ __attribute__((aligned(16))) char wlds[32 * NI * PITCH_W];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 31, kh = lane >> 5;
    const int half = O >> 1, oq = O >> 2;
    const unsigned pitch_o = (unsigned)O * 4u + 16u;
    char *buf = lds + wave * REGION, *plane = buf + TILE;

    // W transposed (zeros past I, and past O): the product's first operand, lane = column of the kept
    // rows, k = the lane half's columns of g
    for (int i = threadIdx.x; i < 32 * NI * KO * 8; i += THREADS) {
        const int c = i % (32 * NI), o = i / (32 * NI);
        *(float *)(wlds + c * PITCH_W + o * 4) = c < I && o < O ? W[(size_t)o * I + c] : 0.0f;
    }
    __syncthreads();
    const unsigned w_at = (unsigned)(n * PITCH_W + kh * half * 4);
    unsigned in_at[KO];
#pragma unroll
    for (int j = 0; j < KO; ++j) {
        const unsigned f = (unsigned)lane + 64u * j, r = f / (unsigned)oq;
        in_at[j] = r * pitch_o + (f - r * oq) * 16u;
    }
    // the lane's kept columns in memory order, and its row in the first piece
    const int col = 4 * (lane % IQ), row0 = lane / IQ;
    float scale[4], m_g[4], m_gz[4];
    BnKink kink[4];
    if constexpr (MODE == L8_APPLY) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float gamma = bn.weight ? bn.weight[col + k] : 1.0f;
            kink[k].load(gamma, bn.bias ? bn.bias[col + k] : 0.0f);
            if (!bn.act) kink[k].sign = 0.0f, kink[k].at = -1.0f;       // (every number is on)
            scale[k] = gamma * bn.invstd[col + k];
            m_g[k] = bn.training ? bn.col_terms[col + k] : 0.0f;
            m_gz[k] = bn.training ? bn.col_terms[I + col + k] : 0.0f;
        }
    }
    // columns of g for the weight gradient (past O: column 0, never stored)
    const int gc = NA == 2 ? (2 * n < O ? 2 * n : 0) : (n < O ? n : 0);
    const int qc = NI == 2 ? 2 * n : (n < I ? n : 0);
    // odd waves sum -g^T y (mvf_bf16x3.h)
    [[maybe_unused]] const float turned = xty_turned(wave);
    [[maybe_unused]] const unsigned flip = xty_flip(wave);
    xty_acc run[XTY ? NA : 1][XTY ? NI : 1];
    float sums[NA];
    if constexpr (XTY) {
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            sums[i] = 0.0f;
#pragma unroll
            for (int b = 0; b < NI; ++b)
#pragma unroll
                for (int e = 0; e < 16; ++e) run[i][b][e] = 0.0f;
        }
    }
    const i64 nfull = rows / L8_ROWS;
    const int rest = (int)(rows - nfull * L8_ROWS);
    const i64 wid = (i64)blockIdx.x * WAVES + wave, nwaves = (i64)gridDim.x * WAVES;
    l8_f4 g[KO];
    unsigned qw[KI];
    int ew;
    auto load_tile = [&](i64 t, int live) {
        const l8_f4 *src = (const l8_f4 *)(gsrc + (size_t)t * L8_ROWS * O);
#pragma unroll
        for (int j = 0; j < KO; ++j) {
            const int f = lane + 64 * j;
            g[j] = src[(EXACT && live == L8_ROWS) || f < live * oq ? f : live * oq - 1];
        }
        const unsigned *qsrc = (const unsigned *)(codes + (size_t)t * L8_ROWS * I);
#pragma unroll
        for (int j = 0; j < KI; ++j) {
            const int f = lane + 64 * j;
            qw[j] = qsrc[live == L8_ROWS || f < live * IQ ? f : live * IQ - 1];
        }
        ew = exps[(size_t)t * L8_ROWS * GR + (lane < live * GR ? lane : live * GR - 1)];
    };
    // One tile; WHOLE: all its rows exist (see the forward).
    auto tile = [&](i64 t, int live, i64 next, auto how) {
        constexpr bool WHOLE = decltype(how)::WHOLE;
        // g as rows; rows past the end are zeros
#pragma unroll
        for (int j = 0; j < KO; ++j) {
            const int f = lane + 64 * j;
            const l8_f4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
            if (EXACT || f < L8_ROWS * oq) *(l8_f4 *)(buf + in_at[j]) = WHOLE || f < live * oq ? g[j] : zero;
        }
        // the kept rows as they read back, one bf16 each, for the weight gradient
        unsigned q[KI];
        int e[KI];
#pragma unroll
        for (int j = 0; j < KI; ++j) {
            // (rows past the end as zeros here too: a code of NaN would survive the zeros of g)
            q[j] = WHOLE || row0 + j * (64 / IQ) < live ? qw[j] : 0u;
            e[j] = __shfl(ew, (row0 + j * (64 / IQ)) * GR + col / R8_GROUP, 64);
            if constexpr (XTY) {
                float v[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = r8_decode(r8_byte(q[j], k), e[j]);
                const r8_u2 d = {xty_hi2(v[0], v[1]), xty_hi2(v[2], v[3])};
                *(r8_u2 *)(plane + (row0 + j * (64 / IQ)) * PITCH_Q + col * 2) = d;
            }
        }
        l8_wave_sync();
        // g^T y: lane = column, 8 rows of 16
        if constexpr (XTY) {
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                XtyParts<3> gp[NA];
                unsigned d[8];
                float c[NA][8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const char *at = buf + (unsigned)(16 * st + 8 * kh + k) * pitch_o + (unsigned)gc * 4u;
                    if constexpr (NA == 2) {
                        const l8_f2 v = *(const l8_f2 *)at;
                        c[0][k] = v[0];
                        c[1][k] = v[1];
                    } else {
                        c[0][k] = *(const float *)at;
                    }
                    const char *qt = plane + (16 * st + 8 * kh + k) * PITCH_Q + qc * 2;
                    d[k] = NI == 2 ? *(const unsigned *)qt : (unsigned)*(const unsigned short *)qt;
                }
#pragma unroll
                for (int i = 0; i < NA; ++i) {
                    gp[i].cut(c[i]);
                    if (want_sums)
                        sums[i] += ((c[i][0] + c[i][1]) + (c[i][2] + c[i][3])) + ((c[i][4] + c[i][5]) + (c[i][6] + c[i][7]));
                }
#pragma unroll
                for (int b = 0; b < NI; ++b) {
                    xty_u4 yp;
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        yp[k] = __builtin_amdgcn_perm(d[2 * k + 1], d[2 * k], b == 0 ? 0x05040100u : 0x07060302u) ^ flip;
#pragma unroll
                    for (int i = 0; i < NA; ++i) {
                        run[i][b] += xty_product(gp[i], yp, xty_zero());
                        xty_done(run[i][b]);
                    }
                }
            }
        }
        // the next tile asked for here, where the weight gradient's operands have left their registers; the
        // product hides its way
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (decltype(how)::NEXT) load_tile(next, L8_ROWS);
        __builtin_amdgcn_sched_barrier(0);
        // g W: lane = row
        xty_acc acc[NI];
#pragma unroll
        for (int b = 0; b < NI; ++b)
#pragma unroll
            for (int k = 0; k < 16; ++k) acc[b][k] = 0.0f;
        {
            const char *wp = wlds + l8_fresh(w_at), *gp = buf + (unsigned)n * pitch_o + (unsigned)(kh * half) * 4u;
#pragma unroll
            for (int p = 0; p < KO; ++p) {
                l8_f4 v = {0.0f, 0.0f, 0.0f, 0.0f}, w[NI];
                if (EXACT || 4 * p < half) v = *(const l8_f4 *)(gp + 16 * p);
#pragma unroll
                for (int b = 0; b < NI; ++b) {
                    w[b] = *(const l8_f4 *)(wp + 32 * b * PITCH_W + 16 * p);
                    if (!EXACT && 4 * p >= half) w[b] = v;
                }
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int b = 0; b < NI; ++b)
                        acc[b] = __builtin_amdgcn_mfma_f32_32x32x2f32(w[b][k], v[k], acc[b], 0, 0, 0);
            }
        }
        l8_wave_sync();
        // g W as rows, then in memory order
#pragma unroll
        for (int b = 0; b < NI; ++b)
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                const int ch = 32 * b + 8 * p + 4 * kh;
                if (ch < I) {
                    const l8_f4 v = {acc[b][4 * p], acc[b][4 * p + 1], acc[b][4 * p + 2], acc[b][4 * p + 3]};
                    *(l8_f4 *)(buf + n * PITCH_I + ch * 4) = v;
                }
            }
        l8_wave_sync();
        l8_f4 *dst = (l8_f4 *)(grad + (size_t)t * L8_ROWS * I);
#pragma unroll
        for (int j = 0; j < KI; ++j) {
            const int r = row0 + j * (64 / IQ);
            l8_f4 v = *(const l8_f4 *)(buf + r * PITCH_I + col * 4);
            if constexpr (MODE == L8_APPLY) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float zq = r8_decode(r8_byte(q[j], k), e[j]);
                    const float gg = kink[k].on(zq) ? v[k] : v[k] * bn.slope;
                    v[k] = bn.training ? (gg - m_g[k] - zq * m_gz[k]) * scale[k] : gg * scale[k];
                }
            }
            if (WHOLE || r < live) r8_stream(dst + lane + 64 * j, v);
        }
        l8_wave_sync();
    };
    // grad_z's pass goes from the last tile to the first: the memory-side cache still holds the end of what the
    // sums' pass has read (2 M rows of 64 columns: 240 -> 235 us)
    auto at = [&](i64 t) { return MODE == L8_APPLY ? nfull - 1 - t : t; };
    if (wid < nfull) {
        load_tile(at(wid), L8_ROWS);
        i64 t = wid;
        tile(at(t), L8_ROWS, at(t + nwaves < nfull ? t + nwaves : t), L8Tile<true, true>());
        for (t += nwaves; t < nfull; t += nwaves) tile(at(t), L8_ROWS, at(t + nwaves < nfull ? t + nwaves : t), L8Tile<true, true>());
    }
    if (rest > 0 && wid == nfull % nwaves) {
        load_tile(nfull, rest);
        tile(nfull, rest, 0, L8Tile<false, false>());
    }

    if constexpr (XTY) {
        __syncthreads();
        float *fold = (float *)lds, *fold_sums = fold + NA * NI * 1024;
        for (int turn = 0; turn < WAVES; ++turn) {
            if (wave == turn) {
#pragma unroll
                for (int i = 0; i < NA; ++i)
#pragma unroll
                    for (int b = 0; b < NI; ++b)
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            const int at = ((i * NI + b) * 16 + k) * 64 + lane;
                            fold[at] = turn == 0 ? run[i][b][k] : __fmaf_rn(turned, run[i][b][k], fold[at]);
                        }
            }
            __syncthreads();
        }
        float *p = partial + (size_t)blockIdx.x * (NA * NI * 1024);
        for (int at = threadIdx.x; at < NA * NI * 1024; at += THREADS) p[at] = fold[at];
        if (want_sums) {
#pragma unroll
            for (int i = 0; i < NA; ++i) {
                const float s = sums[i] + __shfl_xor(sums[i], 32, 64);
                if (kh == 0) fold_sums[wave * 64 + (NA == 2 ? 2 * n + i : n)] = s;
            }
            __syncthreads();
            if (threadIdx.x < 32 * NA) {
                float s = 0.0f;
#pragma unroll
                for (int k = 0; k < WAVES; ++k) s += fold_sums[k * 64 + threadIdx.x];
                partial_sums[(size_t)blockIdx.x * 64 + threadIdx.x] = s;
            }
        }
    }
}

// The sums' pass behind BatchNorm + LeakyReLU, a reduction over the rows alone.  With on = 1 above the kink
// and 0 below, zq the rows read back and s the slope, what the activation passes on of a gradient is
// t = s + (1 - s) on of it, and the Linear's input is t (gamma zq + beta).  So with
//   P = g^T (t zq) = s g^T zq + (1 - s) g^T (on zq),      Q = g^T t = s sum g + (1 - s) g^T on
// grad_W = gamma P + beta Q, and BatchNorm's column sums, of t (g W) and t (g W) zq, are the columns of
// W . Q and W . P: neither g W nor the activated rows are formed.  zq, on zq and on are exact in one bf16, so
// the three products are nine of the bf16 matrix cores', exact but for the additions; a tile of 32 rows is one
// product from zero (mvf_bf16x3.h), added to the wave's sums by the vector unit.  2 M rows of 64 -> 64 columns
// take 215 us in the kernel trace (added per 16 rows: 225; with the sums kept in the matrix cores' accumulators,
// and their errors: 196 to 203, 161 of them without the products, 128 for the bytes).  Past 32 columns of g two
// waves share a tile, 32 columns each: three sums of 64 x 64 would leave room for one wave per SIMD (four waves a
// tile, of 32 x 32 sums, in accumulators: 227 to 253 us).
template <int KO, int KI, bool EXACT>
__global__ __launch_bounds__(T8_THREADS) void tail8_sums_kernel(
    const float *gsrc, int O_, const int8_t *codes, const uint8_t *exps, i64 rows, L8Bn bn, float *partial, float *partial_sums)
{
    constexpr int I = 8 * KI, IQ = 2 * KI, GR = I > 32 ? 2 : 1;
    constexpr int WAVES = T8_THREADS / 64;
    constexpr int NA = KO > 4 ? 2 : 1, NI = I > 32 ? 2 : 1, UNITS = WAVES / NA;
    constexpr int GP = NA == 2 ? 4 : KO;                    // pieces of g a lane loads
    constexpr int PITCH_G = 32 * GP + 16, TILE = L8_ROWS * PITCH_G;
    constexpr int PITCH_Q = I * 2 + 16, REGION = TILE + L8_ROWS * PITCH_Q;
    constexpr int SLOTS = NA * NI * 1024;                   // sums of one product
    constexpr int FOLD = (3 * SLOTS + WAVES * 32) * 4;
    __shared__ __attribute__((aligned(16))) char lds[WAVES * REGION > FOLD ? WAVES * REGION : FOLD];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 31, kh = lane >> 5;
    const int unit = wave / NA, h = wave % NA;              // (the waves of a tile, the wave's half of g)
    const int O = EXACT ? 8 * KO : O_;
    const int width = NA == 1 ? O : h == 0 || EXACT ? 32 : O - 32, gq = width >> 2;
    char *buf = lds + wave * REGION, *plane = buf + TILE;
    const int gc = n < width ? n : 0;                       // (past the width: column 0, left out of the fold)
    const int qc = NI == 2 ? 2 * n : (n < I ? n : 0);
    // the columns' kinks for rows with the sign of gamma taken in: on where sign zq > at
    unsigned signs = 0u;
    float at[NI];
#pragma unroll
    for (int b = 0; b < NI; ++b) {
        const float gamma = bn.weight ? bn.weight[qc + b] : 1.0f, beta = bn.bias ? bn.bias[qc + b] : 0.0f;
        BnKink kink;
        kink.load(gamma, beta);
        if (gamma < 0.0f) signs |= b == 0 ? 0x8000u : 0x80000000u;
        at[b] = !bn.act ? -__builtin_inff() : gamma != 0.0f ? kink.at : beta > 0.0f ? -__builtin_inff() : __builtin_inff();
    }
    // where the lane's pieces of g come from and go to
    unsigned from[GP], to[GP];
#pragma unroll
    for (int j = 0; j < GP; ++j) {
        const unsigned f = min((unsigned)lane + 64u * j, (unsigned)(L8_ROWS * gq - 1)), r = f / (unsigned)gq;
        from[j] = (r * (unsigned)O + 32u * h + (f - r * gq) * 4u) * 4u;
        to[j] = r * PITCH_G + (f - r * gq) * 16u;
    }
    const int col = 4 * (lane % IQ), row0 = lane / IQ;      // the lane's codes in memory order
    xty_acc all[NI], above[NI], on[NI];                     // of sign zq, on sign zq, on
    float sums = 0.0f;
#pragma unroll
    for (int b = 0; b < NI; ++b)
#pragma unroll
        for (int k = 0; k < 16; ++k) all[b][k] = above[b][k] = on[b][k] = 0.0f;

    const i64 nfull = rows / L8_ROWS;
    const int rest = (int)(rows - nfull * L8_ROWS);
    const i64 uid = (i64)blockIdx.x * UNITS + unit, nunits = (i64)gridDim.x * UNITS;
    const float turned = xty_turned((int)uid);              // odd units sum -g^T (...) (mvf_bf16x3.h)
    l8_f4 g[GP];
    unsigned qw[KI];
    int ew;
    auto load_tile = [&](i64 t, int live) {
        const char *src = (const char *)(gsrc + (size_t)t * L8_ROWS * O);
        const unsigned last = ((unsigned)(live - 1) * O + 32u * h) * 4u;
#pragma unroll
        for (int j = 0; j < GP; ++j)
            g[j] = *(const l8_f4 *)(src + (live == L8_ROWS || lane + 64 * j < live * gq ? from[j] : last));
        const unsigned *qsrc = (const unsigned *)(codes + (size_t)t * L8_ROWS * I);
#pragma unroll
        for (int j = 0; j < KI; ++j) {
            const int f = lane + 64 * j;
            qw[j] = qsrc[live == L8_ROWS || f < live * IQ ? f : live * IQ - 1];
        }
        ew = exps[(size_t)t * L8_ROWS * GR + (lane < live * GR ? lane : live * GR - 1)];
    };
    auto tile = [&](int live, i64 next, auto how) {
        constexpr bool WHOLE = decltype(how)::WHOLE;
#pragma unroll
        for (int j = 0; j < GP; ++j) {
            const int f = lane + 64 * j;
            const l8_f4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
            if (EXACT || f < L8_ROWS * gq) *(l8_f4 *)(buf + to[j]) = WHOLE || f < live * gq ? g[j] * turned : zero;
        }
        // the kept rows as they read back, one bf16 each; codes of NaN are looked for in all of them at once
        int e[KI];
        float least = 0.0f;
#pragma unroll
        for (int j = 0; j < KI; ++j) {
            // (rows past the end as zeros here too: a code of NaN would survive the zeros of g)
            if (!WHOLE && row0 + j * (64 / IQ) >= live) qw[j] = 0u;
            e[j] = __shfl(ew, (row0 + j * (64 / IQ)) * GR + col / R8_GROUP, 64);
            const float step = ldexpf(1.0f, e[j] - R8_BIAS);
            float c[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) c[k] = (float)r8_byte(qw[j], k);
            least = fminf(fminf(least, c[0]), c[1]);
            least = fminf(fminf(least, c[2]), c[3]);
            const r8_u2 d = {xty_hi2(c[0] * step, c[1] * step), xty_hi2(c[2] * step, c[3] * step)};
            *(r8_u2 *)(plane + (row0 + j * (64 / IQ)) * PITCH_Q + col * 2) = d;
        }
        if (__any(least == (float)R8_NAN)) {
#pragma unroll
            for (int j = 0; j < KI; ++j) {
                float v[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = r8_decode(r8_byte(qw[j], k), e[j]);
                const r8_u2 d = {xty_hi2(v[0], v[1]), xty_hi2(v[2], v[3])};
                *(r8_u2 *)(plane + (row0 + j * (64 / IQ)) * PITCH_Q + col * 2) = d;
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (decltype(how)::NEXT) load_tile(next, L8_ROWS);
        __builtin_amdgcn_sched_barrier(0);
        l8_wave_sync();
        // lane = column, 8 rows of 16, twice
        XtyParts<3> gp[2];
        unsigned d[2][8];
#pragma unroll
        for (int st = 0; st < 2; ++st) {
            float c[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int r = 16 * st + 8 * kh + k;
                c[k] = *(const float *)(buf + r * PITCH_G + gc * 4);
                const char *qt = plane + r * PITCH_Q + qc * 2;
                d[st][k] = (NI == 2 ? *(const unsigned *)qt : (unsigned)*(const unsigned short *)qt) ^ signs;
            }
            sums += ((c[0] + c[1]) + (c[2] + c[3])) + ((c[4] + c[5]) + (c[6] + c[7]));
            gp[st].cut(c);
        }
#pragma unroll
        for (int b = 0; b < NI; ++b) {
            xty_u4 zp[2], up[2];
#pragma unroll
            for (int st = 0; st < 2; ++st)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const unsigned lo = d[st][2 * k], hi = d[st][2 * k + 1];
                    zp[st][k] = __builtin_amdgcn_perm(hi, lo, b == 0 ? 0x05040100u : 0x07060302u);
                    unsigned u = __uint_as_float(b == 0 ? lo << 16 : lo & 0xffff0000u) > at[b] ? 0xffffu : 0u;
                    up[st][k] = __uint_as_float(b == 0 ? hi << 16 : hi & 0xffff0000u) > at[b] ? u | 0xffff0000u : u;
                }
            auto add = [&](xty_acc &sum, xty_u4 y0, xty_u4 y1) {
                sum += xty_product(gp[1], y1, xty_product(gp[0], y0, xty_zero()));
                xty_done(sum);
            };
            add(all[b], zp[0], zp[1]);
            add(above[b], zp[0] & up[0], zp[1] & up[1]);
            add(on[b], up[0] & 0x3f803f80u, up[1] & 0x3f803f80u);       // (1.0 twice)
        }
        l8_wave_sync();
    };
    if (uid < nfull) {
        load_tile(uid, L8_ROWS);
        for (i64 t = uid; t < nfull; t += nunits) tile(L8_ROWS, t + nunits < nfull ? t + nunits : t, L8Tile<true, true>());
    }
    if (rest > 0 && uid == nfull % nunits) {
        load_tile(nfull, rest);
        tile(rest, 0, L8Tile<false, false>());
    }

    // the units joined in their order
    __syncthreads();
    float *fold = (float *)lds, *fold_sums = fold + 3 * SLOTS;
    for (int turn = 0; turn < UNITS; ++turn) {
        if (unit == turn) {
#pragma unroll
            for (int b = 0; b < NI; ++b)
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    const int slot = ((h * NI + b) * 16 + k) * 64 + lane;
                    fold[slot] = __fmaf_rn(turned, all[b][k], turn == 0 ? 0.0f : fold[slot]);
                    fold[SLOTS + slot] = __fmaf_rn(turned, above[b][k], turn == 0 ? 0.0f : fold[SLOTS + slot]);
                    fold[2 * SLOTS + slot] = __fmaf_rn(turned, on[b][k], turn == 0 ? 0.0f : fold[2 * SLOTS + slot]);
                }
        }
        __syncthreads();
    }
    float *p = partial + (size_t)blockIdx.x * (3 * SLOTS);
    for (int slot = threadIdx.x; slot < 3 * SLOTS; slot += T8_THREADS) p[slot] = fold[slot];
    const float s = turned * (sums + __shfl_xor(sums, 32, 64));
    if (kh == 0) fold_sums[wave * 32 + n] = s;
    __syncthreads();
    if (threadIdx.x < 32 * NA) {
        float t = 0.0f;
#pragma unroll
        for (int k = 0; k < UNITS; ++k) t += fold_sums[(k * NA + threadIdx.x / 32) * 32 + threadIdx.x % 32];
        partial_sums[(size_t)blockIdx.x * 64 + threadIdx.x] = t;
    }
}

// Its workgroups added up in float64: grad_W, grad_b (blocks of their own) and, per 32 columns of g by
// accumulator and lane half, the part of BatchNorm's column sums that its rows of W give: partial_bn
// [32 NA][2][I].
constexpr int T8_FOLD_SLOTS = 16, T8_FOLD_SLICES = 32;
__global__ __launch_bounds__(T8_FOLD_SLOTS * T8_FOLD_SLICES) void tail8_fold_kernel(
    const float *__restrict__ partial, const float *__restrict__ partial_sums, int nwg, int NA, int NI, int O, int I,
    const float *__restrict__ W, L8Bn bn, float *__restrict__ grad_weight, float *__restrict__ grad_bias,
    double *__restrict__ partial_bn)
{
    __shared__ double red[T8_FOLD_SLICES][4][T8_FOLD_SLOTS];
    const int slot = threadIdx.x % T8_FOLD_SLOTS, slice = threadIdx.x / T8_FOLD_SLOTS;
    const int slots = NA * NI * 1024, at = blockIdx.x * T8_FOLD_SLOTS + slot;
    const bool of_bias = at >= slots;                       // (whole blocks)
    const int lane = at & 63, e = (at >> 6) & 15, blk = at >> 10;
    const int o = of_bias ? at - slots : blk / NI * 32 + (e & 3) + 8 * (e >> 2) + 4 * (lane >> 5);
    const int c = NI == 2 ? 2 * (lane & 31) + blk % 2 : lane & 31;
    const int per = (nwg + T8_FOLD_SLICES - 1) / T8_FOLD_SLICES, k1 = min(nwg, (slice + 1) * per);
    double s[4] = {0.0, 0.0, 0.0, 0.0};                     // of zq, on zq, on, g alone
    if (of_bias) {
        for (int k = slice * per; k < k1; ++k) s[3] += (double)partial_sums[(size_t)k * 64 + o];
    } else {
#pragma unroll 4
        for (int k = slice * per; k < k1; ++k) {
#pragma unroll
            for (int i = 0; i < 3; ++i) s[i] += (double)partial[((size_t)k * 3 + i) * slots + at];
            s[3] += (double)partial_sums[(size_t)k * 64 + o];
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) red[slice][i][slot] = s[i];
    __syncthreads();
    if (slice != 0) return;
    for (int k = 1; k < T8_FOLD_SLICES; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] += red[k][i][slot];
    if (of_bias) {
        if (o < O) grad_bias[o] = (float)s[3];
        return;
    }
    if (c >= I) return;
    double P = 0.0, Q = 0.0, w = 0.0;
    if (o < O) {
        const double slope = (double)bn.slope;
        P = slope * s[0] + (1.0 - slope) * s[1];            // (with the sign of gamma in it)
        if (bn.weight && bn.weight[c] < 0.0f) P = -P;
        Q = slope * s[3] + (1.0 - slope) * s[2];
        w = (double)W[(size_t)o * I + c];
        grad_weight[(size_t)o * I + c] =
            (float)((bn.weight ? (double)bn.weight[c] : 1.0) * P + (bn.bias ? (double)bn.bias[c] : 0.0) * Q);
    }
    double *out = partial_bn + (size_t)((blk / NI * 16 + e) * 2 + (lane >> 5)) * 2 * I;
    out[c] = o < O ? w * Q : 0.0;
    out[I + c] = o < O ? w * P : 0.0;
}

static int l8_workgroups(i64 rows, int threads)
{
    int dev = 0, cus = 256;
    if (hipGetDevice(&dev) != hipSuccess ||
        hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus < 1) cus = 256;
    const i64 ntiles = (rows + L8_ROWS - 1) / L8_ROWS;
    const int waves = threads / 64;
    i64 n = (ntiles + waves - 1) / waves;
    if (n > cus) n = cus;
    if (n > L8_MAX_WGS) n = L8_MAX_WGS;
    return (int)n;
}

template <bool TAIL>
static void l8_forward(const float *x, int I, const float *W, const float *bias, int O, i64 rows, const L8Bn &bn, float *y,
                       int8_t *codes, uint8_t *exps, double *col_sums, int nwg, hipStream_t st)
{
    const int no = O > 32 ? 2 : 1;
#define MVF_L8F(KQ_, NO_, ST_)                                                                                     \
    do {                                                                                                           \
        if (O == 32 * NO_)                                                                                         \
            hipLaunchKernelGGL((linear8_forward_kernel<KQ_, NO_, TAIL, ST_, true>), dim3((unsigned)nwg), dim3(L8_FWD_THREADS), 0, \
                               st, x, W, bias, O, rows, bn, y, codes, exps, col_sums);                             \
        else                                                                                                       \
            hipLaunchKernelGGL((linear8_forward_kernel<KQ_, NO_, TAIL, ST_, false>), dim3((unsigned)nwg), dim3(L8_FWD_THREADS), 0, \
                               st, x, W, bias, O, rows, bn, y, codes, exps, col_sums);                             \
    } while (0)
#define MVF_L8F_NO(KQ_)                                                                                            \
    case 8 * KQ_:                                                                                                  \
        if (col_sums) { if (no == 1) MVF_L8F(KQ_, 1, true); else MVF_L8F(KQ_, 2, true); }                          \
        else { if (no == 1) MVF_L8F(KQ_, 1, false); else MVF_L8F(KQ_, 2, false); }                                 \
        break
    switch (I) {
    MVF_L8F_NO(1); MVF_L8F_NO(2); MVF_L8F_NO(4); default: MVF_L8F_NO(8);
    }
#undef MVF_L8F_NO
#undef MVF_L8F
}

// (the workgroups launched: the partial results there are)
template <int MODE>
static int l8_backward(const float *g, int O, const int8_t *codes, const uint8_t *exps, const float *W, int I, i64 rows,
                        const L8Bn &bn, int want_sums, float *grad, float *partial, float *partial_sums, hipStream_t st)
{
    int nwg = 0;
#define MVF_L8B(KO_, KI_)                                                                                          \
    do {                                                                                                           \
        constexpr int threads = l8_bwd_threads(KO_, KI_);                                                          \
        nwg = l8_workgroups(rows, threads);                                                                        \
        if (O == 8 * KO_)                                                                                          \
            hipLaunchKernelGGL((linear8_backward_kernel<KO_, KI_, MODE, true>), dim3((unsigned)nwg), dim3(threads), 0, st, \
                               g, O, codes, exps, W, rows, bn, want_sums, grad, partial, partial_sums); \
        else                                                                                                       \
            hipLaunchKernelGGL((linear8_backward_kernel<KO_, KI_, MODE, false>), dim3((unsigned)nwg), dim3(threads), 0, st, \
                               g, O, codes, exps, W, rows, bn, want_sums, grad, partial, partial_sums); \
    } while (0)
#define MVF_L8B_KI(KO_)                                                                                            \
    do {                                                                                                           \
        switch (I) {                                                                                               \
        case 8: MVF_L8B(KO_, 1); break;                                                                            \
        case 16: MVF_L8B(KO_, 2); break;                                                                           \
        case 32: MVF_L8B(KO_, 4); break;                                                                           \
        default: MVF_L8B(KO_, 8); break;                                                                           \
        }                                                                                                          \
    } while (0)
    if (O <= 8) MVF_L8B_KI(1);
    else if (O <= 16) MVF_L8B_KI(2);
    else if (O <= 32) MVF_L8B_KI(4);
    else MVF_L8B_KI(8);
#undef MVF_L8B_KI
#undef MVF_L8B
    return nwg;
}

// fold of linear8_backward_kernel's weight-gradient partials
static void l8_fold(const float *partial, const float *partial_sums, int nwg, int I, int O, float *grad_weight, float *grad_bias, hipStream_t st)
{
    const int NA = O > 32 ? 2 : 1, NB = I > 32 ? 2 : 1;
    xty8_fold(partial, partial_sums, nwg, NA, NB, NA == 2, NB == 2, O, I, grad_weight, I, grad_bias, st);
}

// The sums' pass and its fold; the rows of partial_bn that hold BatchNorm's sums afterwards.
static int l8_tail_sums(const float *g, int O, const int8_t *codes, const uint8_t *exps, const float *W, int I, i64 rows,
                        const L8Bn &bn, float *grad_weight, float *grad_bias, float *partial, float *partial_sums,
                        double *partial_bn, hipStream_t st)
{
    const int NA = O > 32 ? 2 : 1, NI = I > 32 ? 2 : 1, nwg = l8_workgroups(rows, T8_THREADS / NA);
#define MVF_T8(KO_, KI_)                                                                                           \
    do {                                                                                                           \
        if (O == 8 * KO_)                                                                                          \
            hipLaunchKernelGGL((tail8_sums_kernel<KO_, KI_, true>), dim3((unsigned)nwg), dim3(T8_THREADS), 0, st, g, O, codes, \
                               exps, rows, bn, partial, partial_sums);                                             \
        else                                                                                                       \
            hipLaunchKernelGGL((tail8_sums_kernel<KO_, KI_, false>), dim3((unsigned)nwg), dim3(T8_THREADS), 0, st, g, O, codes, \
                               exps, rows, bn, partial, partial_sums);                                             \
    } while (0)
#define MVF_T8_KI(KO_)                                                                                             \
    do {                                                                                                           \
        switch (I) {                                                                                               \
        case 8: MVF_T8(KO_, 1); break;                                                                             \
        case 16: MVF_T8(KO_, 2); break;                                                                            \
        case 32: MVF_T8(KO_, 4); break;                                                                            \
        default: MVF_T8(KO_, 8); break;                                                                            \
        }                                                                                                          \
    } while (0)
    if (O <= 8) MVF_T8_KI(1);
    else if (O <= 16) MVF_T8_KI(2);
    else if (O <= 32) MVF_T8_KI(4);
    else MVF_T8_KI(8);
#undef MVF_T8_KI
#undef MVF_T8
    const int blocks = NA * NI * 1024 / T8_FOLD_SLOTS + (grad_bias ? 64 / T8_FOLD_SLOTS : 0);
    hipLaunchKernelGGL(tail8_fold_kernel, dim3(blocks), dim3(T8_FOLD_SLOTS * T8_FOLD_SLICES), 0, st, (const float *)partial,
                       (const float *)partial_sums, nwg, NA, NI, O, I, W, bn, grad_weight, grad_bias, partial_bn);
    return 32 * NA;
}

static bool l8_aligned(const void *p, size_t to) { return (uintptr_t)p % to == 0; }

}  // namespace mvf

using namespace mvf;

extern "C" int mvf_linear_rows8_supported(int32_t I, int32_t O)
{
    return (I == 8 || I == 16 || I == 32 || I == 64) && O >= 8 && O <= 64 && O % 8 == 0;
}

extern "C" int mvf_linear_rows8_forward(
    const float *x, int32_t I, const float *weight, const float *bias, int32_t O, int64_t rows, float *y,
    int8_t *codes, uint8_t *exps, double *col_sums, size_t col_sums_bytes, int32_t *n_col_sums, void *stream)
{
    MVF_REQUIRE(mvf_linear_rows8_supported(I, O), "linear_rows8_forward: %d -> %d columns are not supported", I, O);
    MVF_REQUIRE(rows >= 1, "linear_rows8_forward: rows must be positive");
    MVF_REQUIRE(x && weight && y && codes && exps, "linear_rows8_forward: null argument");
    MVF_REQUIRE(l8_aligned(x, 16) && l8_aligned(y, 16) && l8_aligned(codes, 4), "linear_rows8_forward: x, y or codes not aligned");
    MVF_REQUIRE(!col_sums || (n_col_sums && col_sums_bytes >= mvf_linear_rows_sums_bytes(O)),
                "linear_rows8_forward: too small buffer for the column sums");
    const int nwg = l8_workgroups(rows, L8_FWD_THREADS);
    if (n_col_sums) *n_col_sums = col_sums ? nwg : 0;
    l8_forward<false>(x, I, weight, bias, O, rows, L8Bn{}, y, codes, exps, col_sums, nwg, (hipStream_t)stream);
    MVF_LAUNCH_CHECK();
    return MVF_OK;
}

extern "C" int mvf_linear_rows8_backward(
    const float *grad_y, const int8_t *codes, const uint8_t *exps, const float *weight, int32_t I, int32_t O, int64_t rows,
    float *grad_x, float *grad_weight, float *grad_bias, void *workspace, size_t workspace_bytes, void *stream)
{
    MVF_REQUIRE(mvf_linear_rows8_supported(I, O), "linear_rows8_backward: %d -> %d columns are not supported", I, O);
    MVF_REQUIRE(rows >= 1, "linear_rows8_backward: rows must be positive");
    MVF_REQUIRE(grad_y && codes && exps && weight && grad_x && grad_weight, "linear_rows8_backward: null argument");
    MVF_REQUIRE(l8_aligned(grad_y, 16) && l8_aligned(grad_x, 16) && l8_aligned(codes, 4),
                "linear_rows8_backward: grad_y, grad_x or codes not aligned");
    MVF_REQUIRE(workspace && workspace_bytes >= mvf_xty8_workspace_bytes(), "linear_rows8_backward: workspace too small");
    hipStream_t st = (hipStream_t)stream;
    float *partial = (float *)workspace, *partial_sums = (float *)((char *)workspace + mvf_xty_workspace_bytes());
    const int nwg = l8_backward<L8_LINEAR>(grad_y, O, codes, exps, weight, I, rows, L8Bn{}, grad_bias != nullptr, grad_x, partial,
                                           partial_sums, st);
    l8_fold(partial, partial_sums, nwg, I, O, grad_weight, grad_bias, st);
    MVF_LAUNCH_CHECK();
    return MVF_OK;
}

extern "C" size_t mvf_batch_norm_act_linear8_workspace_bytes(int32_t I)
{
    return I < 1 ? 0 : mvf_batch_norm_act8_workspace_bytes(I) + mvf_xty8_workspace_bytes();
}

extern "C" int mvf_batch_norm_act_linear8_forward(
    const float *z, int64_t rows, int32_t I, const float *bn_weight, const float *bn_bias,
    float *running_mean, float *running_var, int32_t training, float momentum, float eps, int32_t act, float slope,
    int64_t *num_batches, const float *weight, const float *bias, int32_t O, float *y, int8_t *codes, uint8_t *exps, float *save_invstd,
    const double *col_sums, int32_t n_col_sums, double *y_sums, size_t y_sums_bytes, int32_t *n_y_sums,
    void *workspace, size_t workspace_bytes, void *stream)
{
    MVF_REQUIRE(mvf_linear_rows8_supported(I, O), "batch_norm_act_linear8_forward: %d -> %d columns are not supported", I, O);
    MVF_REQUIRE(rows >= 1 && (!training || rows > 1), "batch_norm_act_linear8_forward: too few rows");
    MVF_REQUIRE(z && weight && y && codes && exps && save_invstd, "batch_norm_act_linear8_forward: null argument");
    MVF_REQUIRE(training || (running_mean && running_var),
                "batch_norm_act_linear8_forward: running statistics are needed outside train mode");
    MVF_REQUIRE(l8_aligned(z, 16) && l8_aligned(y, 16) && l8_aligned(codes, 4), "batch_norm_act_linear8_forward: z, y or codes not aligned");
    MVF_REQUIRE(!col_sums || n_col_sums >= 1, "batch_norm_act_linear8_forward: column sums without partial rows");
    MVF_REQUIRE(!y_sums || (n_y_sums && y_sums_bytes >= mvf_linear_rows_sums_bytes(O)),
                "batch_norm_act_linear8_forward: too small buffer for the column sums");
    MVF_REQUIRE(workspace && workspace_bytes >= mvf_batch_norm_act_linear8_workspace_bytes(I),
                "batch_norm_act_linear8_forward: workspace too small");
    hipStream_t st = (hipStream_t)stream;
    const Bn8Workspace w = bn8_workspace(workspace, I);
    bn8_statistics(z, rows, I, running_mean, running_var, training, momentum, eps, col_sums, n_col_sums, (long long *)num_batches, w,
                   save_invstd, st);
    const L8Bn bn = {w.terms, save_invstd, w.terms64, bn_weight, bn_bias, nullptr, act, training, slope};
    const int nwg = l8_workgroups(rows, L8_FWD_THREADS);
    if (n_y_sums) *n_y_sums = y_sums ? nwg : 0;
    l8_forward<true>(z, I, weight, bias, O, rows, bn, y, codes, exps, y_sums, nwg, st);
    MVF_LAUNCH_CHECK();
    return MVF_OK;
}

extern "C" int mvf_batch_norm_act_linear8_backward(
    const float *grad_y, const int8_t *codes, const uint8_t *exps, int64_t rows, int32_t I, const float *bn_weight,
    const float *bn_bias, const float *save_invstd, int32_t training, int32_t act, float slope, const float *weight, int32_t O,
    float *grad_z, float *grad_bn_weight, float *grad_bn_bias, float *grad_weight, float *grad_bias,
    void *workspace, size_t workspace_bytes, void *stream)
{
    MVF_REQUIRE(mvf_linear_rows8_supported(I, O), "batch_norm_act_linear8_backward: %d -> %d columns are not supported", I, O);
    MVF_REQUIRE(rows >= 1, "batch_norm_act_linear8_backward: rows must be positive");
    MVF_REQUIRE(grad_y && codes && exps && save_invstd && weight && grad_weight, "batch_norm_act_linear8_backward: null argument");
    MVF_REQUIRE(l8_aligned(grad_y, 16) && l8_aligned(grad_z, 16) && l8_aligned(codes, 4),
                "batch_norm_act_linear8_backward: grad_y, grad_z or codes not aligned");
    MVF_REQUIRE(workspace && workspace_bytes >= mvf_batch_norm_act_linear8_workspace_bytes(I),
                "batch_norm_act_linear8_backward: workspace too small");
    hipStream_t st = (hipStream_t)stream;
    const Bn8Workspace w = bn8_workspace(workspace, I);
    char *xty = (char *)workspace + mvf_batch_norm_act8_workspace_bytes(I);
    float *partial = (float *)xty, *partial_sums = (float *)(xty + mvf_xty_workspace_bytes());
    const L8Bn bn = {nullptr, save_invstd, nullptr, bn_weight, bn_bias, w.terms, act, training, act ? slope : 1.0f};
    const int nblk = l8_tail_sums(grad_y, O, codes, exps, weight, I, rows, bn, grad_weight, grad_bias, partial, partial_sums,
                                  w.partial, st);
    bn8_grad_terms(w, nblk, I, rows, grad_bn_weight, grad_bn_bias, st);
    if (grad_z)
        l8_backward<L8_APPLY>(grad_y, O, codes, exps, weight, I, rows, bn, 0, grad_z, nullptr, nullptr, st);
    MVF_LAUNCH_CHECK();
    return MVF_OK;
}
