// A gated residual block between two norms, on rows [rows][C] of float32, bfloat16 or float16:
//
//   out = x + scale * gate * N(f; post)        h = N(out; pre)
//
// N is an RMS norm, n * w with n = v / sqrt(mean(v^2) + eps), or a layer norm, n * w + b with
// n = (v - mean v) / sqrt(var v + eps); gate is one value per row and group of C / G neighbouring
// channels, scale one per channel, and a row that is not `seen` adds nothing (f is not read there).
// All arithmetic is float32; out and h are rounded once (h comes from the unrounded out).
//
// Bound by HBM: forward 2 reads and 2 writes of a row, backward the same with the gradients and what
// was kept of x and f (as they are, or in 8 bits: mvf_rows8.h).  A team of lanes owns a row, so
// that a row is read once and stays in registers while its statistics are formed (mean first, then
// the squared differences: no cancellation): 8 to 64 lanes for up to 1024 channels (sums by lane
// exchanges only), a whole workgroup up to 4096.  A lane keeps its channels for the whole launch and
// holds their weights in registers.
//
// Backward, with n, o the normalised f and out, d the whole gradient of out and mean over channels:
//   d  = d_out + r_out * (dh w_pre - o mean(dh w_pre o) - [layer] mean(dh w_pre))     = d_x
//   df = r_f * (e - n mean(e n) - [layer] mean(e)),  e = d gate scale w_post
//   d_gate = sum over the group of d scale (n w + b)
//   column sums over the rows: A = d gate n, B = d gate, P = dh o, Q = dh give
//   d_scale = w A + b B, d_w_post = scale A, d_b_post = scale B, d_w_pre = P, d_b_pre = Q.
// The column sums are float32 per lane over its rows, folded per workgroup and then over the
// workgroups in float64, in a fixed order: the same bits on every run.
#include "mvf_rows8.h"

namespace mvf {

constexpr int RN_THREADS = 256;
constexpr int RN_MAX_C = 4096;
constexpr int RN_MAX_BLOCKS_BWD = 1024;
constexpr int RN_MAX_BLOCKS_FWD = 4096;
enum { RN_NONE = 0, RN_RMS = 1, RN_LAYER = 2 };

struct ResidualArgs {
    const void *x, *f;              // rows; f may be NULL
    const int8_t *qx, *qf;          // backward: codes instead of x, f
    const uint8_t *ex, *ef;
    const float *gate;              // [rows][G] or NULL
    const uint8_t *seen;            // [rows] or NULL
    const float *scale, *w_post, *b_post, *w_pre, *b_pre;   // [C] or NULL
    float *stats;                   // [4][rows]: 1 / spread and mean of f, of out (or NULL)
    int G, post, pre;
    float eps_post, eps_pre;
    i64 rows;
    int C;
};

// lane exchange inside rows of 16 lanes
template <int CTRL> __device__ __forceinline__ float rn_dpp(float v)
{
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}

// Sums over a team of TPR lanes, in all of them, a fixed tree.  lds: TPR > 64 only, two buffers of
// RN_LDS floats used in turn, so that one barrier per call is enough (whoever writes a buffer again
// has passed the barrier of the call between, behind every read of the buffer's last use).
constexpr int RN_LDS = 2 * (RN_THREADS / 64);
template <int TPR, int N>
__device__ __forceinline__ void team_sum(float (&v)[N], float *lds, int &turn)
{
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] += rn_dpp<0xb1>(v[i]);         // lane ^ 1
        v[i] += rn_dpp<0x4e>(v[i]);         // lane ^ 2
        v[i] += rn_dpp<0x141>(v[i]);        // mirrored inside 8
        if constexpr (TPR >= 16) v[i] += rn_dpp<0x140>(v[i]);       // mirrored inside 16
        if constexpr (TPR >= 32) v[i] += __shfl_xor(v[i], 16, 64);
        if constexpr (TPR >= 64) v[i] += __shfl_xor(v[i], 32, 64);
    }
    if constexpr (TPR > 64) {
        constexpr int W = TPR / 64;
        static_assert(N * W <= RN_LDS, "buffer");
        float *p = lds + turn * RN_LDS;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) p[i * W + threadIdx.x / 64] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float s = p[i * W];
#pragma unroll
            for (int k = 1; k < W; ++k) s += p[i * W + k];
            v[i] = s;
        }
        turn ^= 1;
    }
}

// What a lane knows of its channels.
template <int TPR, int NV, bool VEC> struct RnChannels {
    int col[NV];                    // first of four
    int grp[NV][VEC ? 1 : 4];       // gate group (VEC: groups are multiples of four channels)
    __device__ __forceinline__ void init(int C, int G)
    {
        const int gw = G > 0 ? C / G : C;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            col[j] = 4 * (j * TPR + (int)(threadIdx.x % TPR));
#pragma unroll
            for (int k = 0; k < (VEC ? 1 : 4); ++k) grp[j][k] = min(col[j] + k, C - 1) / gw;
        }
    }
    __device__ __forceinline__ bool has(int j, int k, int C) const { return VEC ? col[j] < C : col[j] + k < C; }
};

template <int NV> __device__ __forceinline__ void rn_vector(const float *p, const int (&col)[NV], int C, float none, float (&v)[NV][4])
{
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) v[j][k] = col[j] + k < C ? (p ? p[col[j] + k] : none) : 0.0f;
}

template <class R, int NV, bool VEC>
__device__ __forceinline__ void rn_load(const void *base, i64 row, const int (&col)[NV], int C, float (&v)[NV][4])
{
    const typename R::T *p = (const typename R::T *)base + row * C;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[j][k] = 0.0f;
        if (col[j] < C) row_load4<R, VEC>(p, col[j], C, v[j]);
    }
}

template <class R, int NV, bool VEC>
__device__ __forceinline__ void rn_store(void *base, i64 row, const int (&col)[NV], int C, const float (&v)[NV][4])
{
    typename R::T *p = (typename R::T *)base + row * C;
#pragma unroll
    for (int j = 0; j < NV; ++j)
        if (col[j] < C) row_store4<R, VEC>(p, col[j], C, v[j]);
}

template <int NV, bool VEC>
__device__ __forceinline__ void rn_decode(const int8_t *codes, const uint8_t *exps, i64 row, const int (&col)[NV], int C, float (&v)[NV][4])
{
    const int GR = (C + R8_GROUP - 1) / R8_GROUP;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[j][k] = 0.0f;
        if (col[j] < C) {
            const unsigned q = codes_load4<VEC>(codes + row * C, col[j], C);
            const int e = exps[row * GR + col[j] / R8_GROUP];
#pragma unroll
            for (int k = 0; k < 4; ++k) v[j][k] = r8_decode(r8_byte(q, k), e);
        }
    }
}

template <class R, int NV, bool VEC>
__device__ __forceinline__ void rn_encode(int8_t *codes, uint8_t *exps, i64 row, const int (&col)[NV], int C, const float (&v)[NV][4])
{
    const int GR = (C + R8_GROUP - 1) / R8_GROUP;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const unsigned m = max(max(r8_magnitude(v[j][0]), r8_magnitude(v[j][1])), max(r8_magnitude(v[j][2]), r8_magnitude(v[j][3])));
        const int e = r8_exponent(r8_max8(m), R::E_MAX);
        if (col[j] < C) {
            const int q[4] = {r8_encode(v[j][0], e), r8_encode(v[j][1], e), r8_encode(v[j][2], e), r8_encode(v[j][3], e)};
            codes_store4<VEC>(codes + row * C, col[j], C, r8_pack4(q));
            if ((threadIdx.x & 7) == 0) exps[row * GR + col[j] / R8_GROUP] = (uint8_t)e;
        }
    }
}

// gate of the lane's channels, 0 on a row that is not seen (1 without a gate)
template <int TPR, int NV, bool VEC>
__device__ __forceinline__ void rn_gate(const ResidualArgs &a, i64 row, const RnChannels<TPR, NV, VEC> &ch, float (&g)[NV][4])
{
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if constexpr (VEC) {
                if (k > 0) { g[j][k] = g[j][0]; continue; }
            }
            g[j][k] = a.gate ? a.gate[row * a.G + ch.grp[j][VEC ? 0 : k]] : 1.0f;
        }
}

// 1 / spread and mean (0 for an RMS norm) of a team's row
template <int TPR, int NV, bool VEC>
__device__ __forceinline__ void rn_stats(const float (&v)[NV][4], const RnChannels<TPR, NV, VEC> &ch, int C, int kind, float eps,
                                         float *lds, int &turn, float &r, float &mu)
{
    mu = 0.0f;
    if (kind == RN_LAYER) {
        float s[1] = {0.0f};
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int k = 0; k < 4; ++k) s[0] += v[j][k];            // (channels past C hold zeros)
        team_sum<TPR, 1>(s, lds, turn);
        mu = s[0] / (float)C;
    }
    float s[1] = {0.0f};
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float d = ch.has(j, k, C) ? v[j][k] - mu : 0.0f;
            s[0] = __fmaf_rn(d, d, s[0]);
        }
    team_sum<TPR, 1>(s, lds, turn);
    r = 1.0f / sqrtf(s[0] / (float)C + eps);
}

template <class R, int TPR, int NV, bool VEC>
__global__ __launch_bounds__(RN_THREADS) void residual_forward_kernel(
    const ResidualArgs a, void *__restrict__ out, void *__restrict__ h,
    int8_t *__restrict__ qx, uint8_t *__restrict__ ex, int8_t *__restrict__ qf, uint8_t *__restrict__ ef)
{
    __shared__ float lds[2 * RN_LDS];
    int turn = 0;
    const int C = a.C;
    RnChannels<TPR, NV, VEC> ch;
    ch.init(C, a.G);
    float scale[NV][4], w_post[NV][4], b_post[NV][4], w_pre[NV][4], b_pre[NV][4];
    rn_vector<NV>(a.scale, ch.col, C, 1.0f, scale);
    rn_vector<NV>(a.w_post, ch.col, C, 1.0f, w_post);
    rn_vector<NV>(a.b_post, ch.col, C, 0.0f, b_post);
    rn_vector<NV>(a.w_pre, ch.col, C, 1.0f, w_pre);
    rn_vector<NV>(a.b_pre, ch.col, C, 0.0f, b_pre);
    constexpr int TEAMS = RN_THREADS / TPR;
    for (i64 row = (i64)blockIdx.x * TEAMS + threadIdx.x / TPR; row < a.rows; row += (i64)gridDim.x * TEAMS) {
        const bool adds = a.f && (!a.seen || a.seen[row]);
        float x[NV][4], f[NV][4], g[NV][4];
        rn_load<R, NV, VEC>(a.x, row, ch.col, C, x);
        if (adds) {
            rn_load<R, NV, VEC>(a.f, row, ch.col, C, f);
            rn_gate<TPR, NV, VEC>(a, row, ch, g);
        } else {
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k) f[j][k] = g[j][k] = 0.0f;
        }
        if (qx) rn_encode<R, NV, VEC>(qx, ex, row, ch.col, C, x);
        if (qf) rn_encode<R, NV, VEC>(qf, ef, row, ch.col, C, f);
        float r = 1.0f, mu = 0.0f;
        if (adds) {                         // (the same in all lanes of a team)
            if (a.post != RN_NONE) rn_stats<TPR, NV, VEC>(f, ch, C, a.post, a.eps_post, lds, turn, r, mu);
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float v = __fmaf_rn((f[j][k] - mu) * r, w_post[j][k], b_post[j][k]);
                    x[j][k] = ch.has(j, k, C) ? __fmaf_rn(scale[j][k] * g[j][k], v, x[j][k]) : 0.0f;
                }
        }
        if (out) rn_store<R, NV, VEC>(out, row, ch.col, C, x);
        float r2 = 1.0f, mu2 = 0.0f;
        if (a.pre != RN_NONE) {
            rn_stats<TPR, NV, VEC>(x, ch, C, a.pre, a.eps_pre, lds, turn, r2, mu2);
            float y[NV][4];
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k) y[j][k] = __fmaf_rn((x[j][k] - mu2) * r2, w_pre[j][k], b_pre[j][k]);
            rn_store<R, NV, VEC>(h, row, ch.col, C, y);
        }
        if (a.stats && threadIdx.x % TPR == 0) {
            a.stats[row] = r;
            a.stats[a.rows + row] = mu;
            a.stats[2 * a.rows + row] = r2;
            a.stats[3 * a.rows + row] = mu2;
        }
    }
}

template <class R, int TPR, int NV, bool VEC>
__global__ __launch_bounds__(RN_THREADS) void residual_backward_kernel(
    const ResidualArgs a, const void *__restrict__ d_out, const void *__restrict__ d_h,
    void *__restrict__ d_x, void *__restrict__ d_f, float *__restrict__ d_gate, float *__restrict__ partial)
{
    __shared__ float lds[2 * RN_LDS];
    __shared__ float fold[RN_THREADS * 4 * NV];
    int turn = 0;
    const int C = a.C;
    RnChannels<TPR, NV, VEC> ch;
    ch.init(C, a.G);
    float scale[NV][4], w_post[NV][4], b_post[NV][4], w_pre[NV][4];
    rn_vector<NV>(a.scale, ch.col, C, 1.0f, scale);
    rn_vector<NV>(a.w_post, ch.col, C, 1.0f, w_post);
    rn_vector<NV>(a.b_post, ch.col, C, 0.0f, b_post);
    rn_vector<NV>(a.w_pre, ch.col, C, 1.0f, w_pre);
    // column sums: d gate n, d gate, dh o, dh
    float acc[4][NV][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[i][j][k] = 0.0f;
    const float inv_c = 1.0f / (float)C;
    constexpr int TEAMS = RN_THREADS / TPR;
    for (i64 row = (i64)blockIdx.x * TEAMS + threadIdx.x / TPR; row < a.rows; row += (i64)gridDim.x * TEAMS) {
        const bool adds = (a.f || a.qf) && (!a.seen || a.seen[row]);
        float d[NV][4], n[NV][4], g[NV][4];
        float rf = 1.0f;
        if (d_out) {
            rn_load<R, NV, VEC>(d_out, row, ch.col, C, d);
        } else {
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k) d[j][k] = 0.0f;
        }
        if (adds) {
            if (a.qf) rn_decode<NV, VEC>(a.qf, a.ef, row, ch.col, C, n);
            else rn_load<R, NV, VEC>(a.f, row, ch.col, C, n);
            rn_gate<TPR, NV, VEC>(a, row, ch, g);
            if (a.post != RN_NONE) {
                rf = a.stats[row];
                const float mu = a.stats[a.rows + row];
#pragma unroll
                for (int j = 0; j < NV; ++j)
#pragma unroll
                    for (int k = 0; k < 4; ++k) n[j][k] = ch.has(j, k, C) ? (n[j][k] - mu) * rf : 0.0f;
            }
        } else {
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k) n[j][k] = g[j][k] = 0.0f;
        }
        if (a.pre != RN_NONE && d_h) {
            float o[NV][4], dh[NV][4];
            if (a.qx) rn_decode<NV, VEC>(a.qx, a.ex, row, ch.col, C, o);
            else rn_load<R, NV, VEC>(a.x, row, ch.col, C, o);
            rn_load<R, NV, VEC>(d_h, row, ch.col, C, dh);
            const float r = a.stats[2 * a.rows + row], mu = a.stats[3 * a.rows + row];
            float s[2] = {0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float v = __fmaf_rn(n[j][k], w_post[j][k], b_post[j][k]);
                    const float u = adds ? __fmaf_rn(scale[j][k] * g[j][k], v, o[j][k]) : o[j][k];
                    o[j][k] = ch.has(j, k, C) ? (u - mu) * r : 0.0f;
                    acc[2][j][k] = __fmaf_rn(dh[j][k], o[j][k], acc[2][j][k]);
                    acc[3][j][k] += dh[j][k];
                    dh[j][k] *= w_pre[j][k];
                    s[0] = __fmaf_rn(dh[j][k], o[j][k], s[0]);
                    s[1] += dh[j][k];
                }
            team_sum<TPR, 2>(s, lds, turn);
            const float m0 = s[0] * inv_c, m1 = a.pre == RN_LAYER ? s[1] * inv_c : 0.0f;
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k) d[j][k] += r * ((dh[j][k] - m1) - o[j][k] * m0);
        }
        if (d_x) rn_store<R, NV, VEC>(d_x, row, ch.col, C, d);
        if (!a.f && !a.qf) continue;        // (uniform)
        float e[NV][4];
        float s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float dg = d[j][k] * g[j][k];
                acc[0][j][k] = __fmaf_rn(dg, n[j][k], acc[0][j][k]);
                acc[1][j][k] += dg;
                e[j][k] = dg * scale[j][k] * w_post[j][k];
                s[0] = __fmaf_rn(e[j][k], n[j][k], s[0]);
                s[1] += e[j][k];
            }
        if (d_f) {
            if (a.post != RN_NONE) {
                team_sum<TPR, 2>(s, lds, turn);
                const float m0 = s[0] * inv_c, m1 = a.post == RN_LAYER ? s[1] * inv_c : 0.0f;
#pragma unroll
                for (int j = 0; j < NV; ++j)
#pragma unroll
                    for (int k = 0; k < 4; ++k) e[j][k] = adds ? rf * ((e[j][k] - m1) - n[j][k] * m0) : 0.0f;
            }
            rn_store<R, NV, VEC>(d_f, row, ch.col, C, e);
        }
        if (d_gate) {
            for (int q = 0; q < a.G; ++q) {
                float t[1] = {0.0f};
#pragma unroll
                for (int j = 0; j < NV; ++j)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float v = __fmaf_rn(n[j][k], w_post[j][k], b_post[j][k]);
                        if (adds && ch.grp[j][VEC ? 0 : k] == q && ch.has(j, k, C)) t[0] = __fmaf_rn(d[j][k] * scale[j][k], v, t[0]);
                    }
                team_sum<TPR, 1>(t, lds, turn);
                if (threadIdx.x % TPR == 0) d_gate[row * a.G + q] = t[0];
            }
        }
    }
    // the workgroup's column sums: teams in order
    if (!partial) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int k = 0; k < 4; ++k) fold[(threadIdx.x / TPR * TPR * NV + j * TPR + threadIdx.x % TPR) * 4 + k] = acc[i][j][k];
        __syncthreads();
        for (int c = threadIdx.x; c < C; c += RN_THREADS) {
            float s = fold[c];
            for (int t = 1; t < TEAMS; ++t) s += fold[t * TPR * NV * 4 + c];
            partial[((size_t)blockIdx.x * 4 + i) * C + c] = s;
        }
    }
}

// Column gradients from the workgroups' sums: 16 columns and 16 slices of the workgroups a block.
__global__ __launch_bounds__(256) void residual_fold_kernel(
    const float *__restrict__ partial, int nblk, int C, const float *__restrict__ scale,
    const float *__restrict__ w_post, const float *__restrict__ b_post,
    float *__restrict__ d_scale, float *__restrict__ d_w_post, float *__restrict__ d_b_post,
    float *__restrict__ d_w_pre, float *__restrict__ d_b_pre)
{
    __shared__ double red[4][16][16];
    const int c0 = threadIdx.x % 16, slice = threadIdx.x / 16, c = blockIdx.x * 16 + c0;
    double s[4] = {0.0, 0.0, 0.0, 0.0};
    if (c < C)
        for (int b = slice; b < nblk; b += 16)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] += (double)partial[((size_t)b * 4 + i) * C + c];
#pragma unroll
    for (int i = 0; i < 4; ++i) red[i][slice][c0] = s[i];
    __syncthreads();
    if (slice != 0 || c >= C) return;
    for (int k = 1; k < 16; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] += red[i][k][c0];
    const double sc = scale ? scale[c] : 1.0, w = w_post ? w_post[c] : 1.0, b = b_post ? b_post[c] : 0.0;
    if (d_scale) d_scale[c] = (float)(w * s[0] + b * s[1]);
    if (d_w_post) d_w_post[c] = (float)(sc * s[0]);
    if (d_b_post) d_b_post[c] = (float)(sc * s[1]);
    if (d_w_pre) d_w_pre[c] = (float)s[2];
    if (d_b_pre) d_b_pre[c] = (float)s[3];
}

// Team of a row of C channels: the smallest whose lanes hold it in one piece of four channels each,
// then two and four pieces per lane, then a workgroup.
struct RnShape { int tpr, nv; };
static RnShape rn_shape(int C)
{
    if (C <= 32) return {8, 1};
    if (C <= 64) return {16, 1};
    if (C <= 128) return {32, 1};
    if (C <= 256) return {64, 1};
    if (C <= 512) return {64, 2};
    if (C <= 1024) return {64, 4};
    return {256, 4};
}

static unsigned rn_blocks(i64 rows, int tpr, int most)
{
    const int teams = RN_THREADS / tpr;
    i64 n = (rows + teams - 1) / teams;
    if (n > most) n = most;
    return (unsigned)(n < 1 ? 1 : n);
}

static bool rn_vec(const ResidualArgs &a, int type, const void *const *rows, int n)
{
    const size_t item = type == R8_F32 ? 4 : 2;
    if (a.C % 4 != 0 || (a.G > 0 && (a.C / a.G) % 4 != 0)) return false;
    for (int i = 0; i < n; ++i)
        if ((uintptr_t)rows[i] % (4 * item) != 0) return false;
    return true;
}

static int rn_check(const ResidualArgs &a, int type, const char *who)
{
    MVF_REQUIRE(type >= R8_F32 && type <= R8_F16, "%s: unknown row type %d", who, type);
    MVF_REQUIRE(a.rows >= 0 && a.C >= 1 && a.C <= RN_MAX_C, "%s: 1 to %d channels, rows non-negative", who, RN_MAX_C);
    MVF_REQUIRE(a.post >= RN_NONE && a.post <= RN_LAYER && a.pre >= RN_NONE && a.pre <= RN_LAYER, "%s: unknown norm", who);
    MVF_REQUIRE(!a.gate || (a.G >= 1 && a.C % a.G == 0), "%s: %d channels do not split into %d gate groups", who, a.C, a.G);
    return MVF_OK;
}

}  // namespace mvf

using namespace mvf;

#define MVF_RN_SHAPES(R_, V_)                                                                       \
    do {                                                                                            \
        switch (shape.tpr * 16 + shape.nv) {                                                        \
        case 8 * 16 + 1: MVF_RN_LAUNCH(R_, 8, 1, V_); break;                                        \
        case 16 * 16 + 1: MVF_RN_LAUNCH(R_, 16, 1, V_); break;                                      \
        case 32 * 16 + 1: MVF_RN_LAUNCH(R_, 32, 1, V_); break;                                      \
        case 64 * 16 + 1: MVF_RN_LAUNCH(R_, 64, 1, V_); break;                                      \
        case 64 * 16 + 2: MVF_RN_LAUNCH(R_, 64, 2, V_); break;                                      \
        case 64 * 16 + 4: MVF_RN_LAUNCH(R_, 64, 4, V_); break;                                      \
        default: MVF_RN_LAUNCH(R_, 256, 4, V_); break;                                              \
        }                                                                                           \
    } while (0)
#define MVF_RN_TYPES()                                                                              \
    do {                                                                                            \
        if (type == R8_F32) { if (vec) MVF_RN_SHAPES(RowF32, true); else MVF_RN_SHAPES(RowF32, false); }         \
        else if (type == R8_BF16) { if (vec) MVF_RN_SHAPES(RowBF16, true); else MVF_RN_SHAPES(RowBF16, false); } \
        else { if (vec) MVF_RN_SHAPES(RowF16, true); else MVF_RN_SHAPES(RowF16, false); }           \
    } while (0)

extern "C" int mvf_residual_norm_forward(
    const void *x, const void *f, int32_t type, int64_t rows, int32_t C, const float *gate, int32_t G,
    const uint8_t *seen, const float *scale, int32_t post, const float *w_post, const float *b_post, float eps_post,
    int32_t pre, const float *w_pre, const float *b_pre, float eps_pre, void *out, void *h,
    int8_t *x_codes, uint8_t *x_exps, int8_t *f_codes, uint8_t *f_exps, float *stats, void *stream)
{
    const ResidualArgs a = {x, f, nullptr, nullptr, nullptr, nullptr, gate, seen, scale, w_post, b_post, w_pre, b_pre,
                            stats, gate ? G : 0, post, pre, eps_post, eps_pre, (i64)rows, C};
    const int rc = rn_check(a, type, "residual_norm_forward");
    if (rc != MVF_OK) return rc;
    if (rows == 0) return MVF_OK;
    MVF_REQUIRE(x && (out || pre != RN_NONE) && (h || pre == RN_NONE), "residual_norm_forward: null argument");
    MVF_REQUIRE((x_codes != nullptr) == (x_exps != nullptr) && (f_codes != nullptr) == (f_exps != nullptr),
                "residual_norm_forward: codes and exponents belong together");
    const void *const ptrs[] = {x, f, out, h};
    const bool vec = rn_vec(a, type, ptrs, 4) && (uintptr_t)x_codes % 4 == 0 && (uintptr_t)f_codes % 4 == 0;
    const RnShape shape = rn_shape(C);
    const dim3 grid(rn_blocks(rows, shape.tpr, RN_MAX_BLOCKS_FWD));
    hipStream_t st = (hipStream_t)stream;
#define MVF_RN_LAUNCH(R_, TPR_, NV_, V_)                                                                          \
    hipLaunchKernelGGL((residual_forward_kernel<R_, TPR_, NV_, V_>), grid, dim3(RN_THREADS), 0, st, a, out, h, x_codes, \
                       x_exps, f_codes, f_exps)
    MVF_RN_TYPES();
#undef MVF_RN_LAUNCH
    MVF_LAUNCH_CHECK();
    return MVF_OK;
}

extern "C" size_t mvf_residual_norm_workspace_bytes(int64_t rows, int32_t C)
{
    if (rows < 1 || C < 1 || C > RN_MAX_C) return 0;
    return align_up((size_t)rn_blocks(rows, rn_shape(C).tpr, RN_MAX_BLOCKS_BWD) * 4 * (size_t)C * sizeof(float));
}

extern "C" int mvf_residual_norm_backward(
    const void *d_out, const void *d_h, const void *x, const int8_t *x_codes, const uint8_t *x_exps,
    const void *f, const int8_t *f_codes, const uint8_t *f_exps, int32_t type, int64_t rows, int32_t C,
    const float *gate, int32_t G, const uint8_t *seen, const float *scale, int32_t post, const float *w_post,
    const float *b_post, int32_t pre, const float *w_pre, const float *stats, void *d_x, void *d_f, float *d_gate,
    float *d_scale, float *d_w_post, float *d_b_post, float *d_w_pre, float *d_b_pre,
    void *workspace, size_t workspace_bytes, void *stream)
{
    const ResidualArgs a = {x, f, x_codes, f_codes, x_exps, f_exps, gate, seen, scale, w_post, b_post, w_pre, nullptr,
                            const_cast<float *>(stats), gate ? G : 0, post, pre, 0.0f, 0.0f, (i64)rows, C};
    const int rc = rn_check(a, type, "residual_norm_backward");
    if (rc != MVF_OK) return rc;
    MVF_REQUIRE((x_codes != nullptr) == (x_exps != nullptr) && (f_codes != nullptr) == (f_exps != nullptr),
                "residual_norm_backward: codes and exponents belong together");
    const bool columns = d_scale || d_w_post || d_b_post || d_w_pre || d_b_pre;
    MVF_REQUIRE(rows == 0 || d_out || d_h, "residual_norm_backward: no gradient");
    MVF_REQUIRE(rows == 0 || pre == RN_NONE || !d_h || x || x_codes, "residual_norm_backward: the pre-norm needs x");
    MVF_REQUIRE(rows == 0 || stats || (post == RN_NONE && pre == RN_NONE), "residual_norm_backward: null statistics");
    MVF_REQUIRE(!d_f || f || f_codes, "residual_norm_backward: a gradient of f without f");
    MVF_REQUIRE(!d_gate || gate, "residual_norm_backward: a gradient of the gate without a gate");
    MVF_REQUIRE(!columns || rows == 0 || (workspace && workspace_bytes >= mvf_residual_norm_workspace_bytes(rows, C)),
                "residual_norm_backward: workspace too small");
    hipStream_t st = (hipStream_t)stream;
    const RnShape shape = rn_shape(C);
    const dim3 grid(rn_blocks(rows, shape.tpr, RN_MAX_BLOCKS_BWD));
    float *partial = columns ? (float *)workspace : nullptr;
    if (rows > 0) {
        const void *const ptrs[] = {x, f, d_out, d_h, d_x, d_f};
        const bool vec = rn_vec(a, type, ptrs, 6) && (uintptr_t)x_codes % 4 == 0 && (uintptr_t)f_codes % 4 == 0;
#define MVF_RN_LAUNCH(R_, TPR_, NV_, V_)                                                                          \
    hipLaunchKernelGGL((residual_backward_kernel<R_, TPR_, NV_, V_>), grid, dim3(RN_THREADS), 0, st, a, d_out, d_h, d_x, \
                       d_f, d_gate, partial)
        MVF_RN_TYPES();
#undef MVF_RN_LAUNCH
    }
    if (columns)
        hipLaunchKernelGGL(residual_fold_kernel, dim3(cdiv(C, 16)), dim3(256), 0, st, (const float *)partial,
                           rows > 0 ? (int)grid.x : 0, (int)C, scale, w_post, b_post, d_scale, d_w_post, d_b_post, d_w_pre, d_b_pre);
    MVF_LAUNCH_CHECK();
    return MVF_OK;
}
