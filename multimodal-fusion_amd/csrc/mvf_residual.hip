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
// the squared differences: no cancellation): 4 to 64 lanes up to 1024 float32 or 1536 16-bit channels
// (sums by lane exchanges only), a whole workgroup up to 4096.  A lane keeps its channels for the
// whole launch, reads their weights from LDS, and has its next row under way while it works on one.
// 262144 x 512 bfloat16 forward 240 to 256 us by box (4.2 to 4.5 TB/s), 500000 x 64 float32 forward and backward
// 262 to 268 us (109 + 157 + 9 in the kernel trace; 4.5 TB/s); 40007 x 1000 bfloat16 322 us (111 + 208 + 8; 2.5
// TB/s): there a lane has 16 channels and the backward 64 column sums for them, with the rest more registers than
// two waves per SIMD have, and one wave waits for its memory and works in turn.
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
constexpr int RN_MAX_BLOCKS_BWD = 1024;     // (the workspace holds a partial row each)
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

// ---- teams ------------------------------------------------------------------------------------
// A workgroup: teams of TPR lanes, one row each (TPR > 64: one team).
template <int TPR> struct RnBlock {
    static constexpr int THREADS = RN_THREADS;
    static constexpr int TEAMS = THREADS / TPR;
};
// Waves per SIMD a kernel with n channels a lane is compiled for: as many as its registers allow with few
// spills (float32 backward with one piece a lane up to 10 registers, with three 14 to 24; forward of unaligned
// rows with one piece 2; the others none).  A launch fills the chip with exactly that many: a second, partly
// filled round of workgroups costs as much as a whole one (262144 x 512 bfloat16 forward 245 to 256 us with
// the 1024 workgroups that its kernel fits, 318 with 1280).  Forward and backward of 500000 x 64 float32 with 3, 4, 5
// waves for the backward: 268, 268, 445 us (spills); of 40007 x 1000 bfloat16 with 1, 2: 326, 444 us (spills).
static constexpr int rn_waves_fwd(int n) { return n <= 4 ? 6 : n <= 8 ? 4 : n <= 12 ? 3 : 2; }
static constexpr int rn_waves_bwd(int n) { return n <= 4 ? 4 : n <= 12 ? 2 : 1; }

// lane exchange inside rows of 16 lanes
template <int CTRL> __device__ __forceinline__ float rn_dpp(float v)
{
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}

// v of the lane 16 (32) away added: the two results of the swap are the two halves in every lane
__device__ __forceinline__ float rn_add16(float v)
{
    const r8_u2 t = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(t.x) + __uint_as_float(t.y);
}
__device__ __forceinline__ float rn_add32(float v)
{
    const r8_u2 t = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(t.x) + __uint_as_float(t.y);
}

// Sums over a team of TPR lanes, in all of them, a fixed tree.  lds: TPR > 64 only, two buffers of
// RN_LDS floats used in turn, so that one barrier per call is enough (whoever writes a buffer again
// has passed the barrier of the call between, behind every read of the buffer's last use).
constexpr int RN_LDS = 4 * (RN_THREADS / 64);
template <int TPR, int N>
__device__ __forceinline__ void team_sum(float (&v)[N], float *lds, int &turn)
{
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] += rn_dpp<0xb1>(v[i]);         // lane ^ 1
        v[i] += rn_dpp<0x4e>(v[i]);         // lane ^ 2
        if constexpr (TPR >= 8) v[i] += rn_dpp<0x141>(v[i]);        // mirrored inside 8
        if constexpr (TPR >= 16) v[i] += rn_dpp<0x140>(v[i]);       // mirrored inside 16
        if constexpr (TPR >= 32) v[i] = rn_add16(v[i]);
        if constexpr (TPR >= 64) v[i] = rn_add32(v[i]);
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

// ---- pieces -----------------------------------------------------------------------------------
// A lane's share of a row: NV pieces of W adjacent channels (16 bytes: 4 float32 or 8 of 16 bits),
// piece j at channel W * (j * TPR + lane of the team).  Pieces are loaded as raw words, a row ahead
// of their use.  VEC: C is a multiple of W and every row starts at a multiple of 16 bytes; otherwise
// a piece inside the row is one access at the alignment of an element, and the last, cut piece goes
// element by element.
template <class R> struct RnPiece { static constexpr int W = 16 / sizeof(typename R::T); };

template <class R, bool VEC>
__device__ __forceinline__ void piece_load(const typename R::T *row, int col, int C, unsigned (&w)[4])
{
    if (VEC && col < C) {
        const r8_u4 t = *reinterpret_cast<const r8_u4 *>(row + col);
        w[0] = t.x; w[1] = t.y; w[2] = t.z; w[3] = t.w;
        return;
    }
    constexpr int W = RnPiece<R>::W;
    if (!VEC && col + W <= C) {
        if constexpr (W == 4) {
            const R8Words4 t = *reinterpret_cast<const R8Words4 *>(row + col);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = t.w[i];
        } else {
            const R8Half8 t = *reinterpret_cast<const R8Half8 *>(row + col);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = t.w[i];
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = 0u;
    if (!VEC && col < C) {                  // the last C % W channels: 8, 4, 2 bytes (C is the same everywhere)
        if constexpr (W == 4) {
            if (C & 2) {
                const R8Half4 t = *reinterpret_cast<const R8Half4 *>(row + col);
                w[0] = t.w[0];
                w[1] = t.w[1];
                if (C & 1) w[2] = __float_as_uint(row[col + 2]);
            } else {
                w[0] = __float_as_uint(row[col]);
            }
        } else {
            if (C & 4) {
                const R8Half4 t = *reinterpret_cast<const R8Half4 *>(row + col);
                w[0] = t.w[0];
                w[1] = t.w[1];
                if (C & 2) {
                    w[2] = reinterpret_cast<const R8Half2 *>(row + col + 4)->w;
                    if (C & 1) w[3] = row[col + 6];
                } else if (C & 1) {
                    w[2] = row[col + 4];
                }
            } else if (C & 2) {
                w[0] = reinterpret_cast<const R8Half2 *>(row + col)->w;
                if (C & 1) w[1] = row[col + 2];
            } else {
                w[0] = row[col];
            }
        }
    }
}

template <class R> __device__ __forceinline__ void piece_values(const unsigned (&w)[4], float (&v)[RnPiece<R>::W])
{
#pragma unroll
    for (int k = 0; k < RnPiece<R>::W; ++k) {
        if constexpr (RnPiece<R>::W == 4) v[k] = __uint_as_float(w[k]);
        else v[k] = R::get((unsigned short)(w[k / 2] >> (16 * (k & 1))));
    }
}

template <class R, bool VEC>
__device__ __forceinline__ void piece_store(typename R::T *row, int col, int C, const float (&v)[RnPiece<R>::W])
{
    constexpr int W = RnPiece<R>::W;
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (W == 4) w[i] = __float_as_uint(v[i]);
        else w[i] = R::put2(v[2 * i], v[2 * i + 1]);
    }
    if (VEC && col < C) {
        const r8_u4 t = {w[0], w[1], w[2], w[3]};
        r8_stream(reinterpret_cast<r8_u4 *>(row + col), t);
    } else if (!VEC && col + W <= C) {
        if constexpr (W == 4) {
            const R8Words4 t = {{w[0], w[1], w[2], w[3]}};
            *reinterpret_cast<R8Words4 *>(row + col) = t;
        } else {
            const R8Half8 t = {{w[0], w[1], w[2], w[3]}};
            *reinterpret_cast<R8Half8 *>(row + col) = t;
        }
    } else if (!VEC && col < C) {
        if constexpr (W == 4) {
            if (C & 2) {
                const R8Half4 t = {{w[0], w[1]}};
                *reinterpret_cast<R8Half4 *>(row + col) = t;
                if (C & 1) row[col + 2] = v[2];
            } else {
                row[col] = v[0];
            }
        } else {
            if (C & 4) {
                const R8Half4 t = {{w[0], w[1]}};
                *reinterpret_cast<R8Half4 *>(row + col) = t;
                if (C & 2) {
                    reinterpret_cast<R8Half2 *>(row + col + 4)->w = w[2];
                    if (C & 1) row[col + 6] = (unsigned short)w[3];
                } else if (C & 1) {
                    row[col + 4] = (unsigned short)w[2];
                }
            } else if (C & 2) {
                reinterpret_cast<R8Half2 *>(row + col)->w = w[0];
                if (C & 1) row[col + 2] = (unsigned short)w[1];
            } else {
                row[col] = (unsigned short)w[0];
            }
        }
    }
}

// codes of a piece: W bytes in W / 4 words
template <int W, bool VEC>
__device__ __forceinline__ void piece_codes_load(const int8_t *row, int col, int C, unsigned (&q)[W / 4])
{
#pragma unroll
    for (int i = 0; i < W / 4; ++i) q[i] = 0u;
    if (col >= C) return;
    if constexpr (VEC && W == 8) {
        const r8_u2 t = *reinterpret_cast<const r8_u2 *>(row + col);
        q[0] = t.x;
        q[1] = t.y;
    } else if constexpr (VEC) {
        q[0] = *reinterpret_cast<const unsigned *>(row + col);
    } else {
#pragma unroll
        for (int i = 0; i < W / 4; ++i) q[i] = codes_load4<false>(row, col + 4 * i, C);
    }
}

template <int W, bool VEC>
__device__ __forceinline__ void piece_codes_store(int8_t *row, int col, int C, const unsigned (&q)[W / 4])
{
    if (col >= C) return;
    if constexpr (VEC && W == 8) {
        const r8_u2 t = {q[0], q[1]};
        *reinterpret_cast<r8_u2 *>(row + col) = t;
    } else if constexpr (VEC) {
        *reinterpret_cast<unsigned *>(row + col) = q[0];
    } else {
#pragma unroll
        for (int i = 0; i < W / 4; ++i) codes_store4<false>(row, col + 4 * i, C, q[i]);
    }
}

// ---- what a lane knows of its channels --------------------------------------------------------
template <int TPR, int NV, int W> struct RnChannels {
    int col[NV];            // first of W
    int ga[NV], gb[NV];     // gate groups of the piece's first and last channel
    int cut[NV];            // channels of the piece in front of the boundary between them
    int gw;                 // channels per group
    float inv_c;
    __device__ __forceinline__ void init(int C, int G)
    {
        inv_c = 1.0f / (float)C;
        gw = G > 1 ? C / G : 1 << 30;       // (one group or none: a single one without an end)
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            col[j] = W * (j * TPR + (int)(threadIdx.x % TPR));
            const int c0 = min(col[j], C - 1), c1 = min(col[j] + W - 1, C - 1);
            ga[j] = c0 / gw;
            gb[j] = c1 / gw;
            cut[j] = gb[j] * gw - col[j];
        }
    }
    // every piece lies in at most two groups
    __device__ __forceinline__ bool simple() const { return gw >= W; }
};

// Per-channel vectors (channels past C: 0) in LDS, as four floats of every lane's pieces side by
// side: a lane reads its own with 16-byte loads free of bank conflicts.  (In registers they would
// cost a wave or more per SIMD, and the kernels live on waves that wait for memory.)
template <int TPR, int NV, int W, int N> struct RnVectors {
    static constexpr int PIECES = TPR * NV, FLOATS = PIECES * W;
    static __device__ __forceinline__ int at(int c) { return (c % W / 4 * PIECES + c / W) * 4 + c % 4; }
    // every thread of the workgroup; a barrier follows
    static __device__ __forceinline__ void fill(float *lds, int i, const float *p, int C, float none, const float *times = nullptr)
    {
        for (int c = threadIdx.x; c < FLOATS; c += RnBlock<TPR>::THREADS)
            lds[i * FLOATS + at(c)] = c < C ? (p ? p[c] : none) * (times ? times[c] : 1.0f) : 0.0f;
    }
    static __device__ __forceinline__ void read(const float *lds, int i, int j, float (&v)[W])
    {
        const int piece = j * TPR + (int)(threadIdx.x % TPR);
#pragma unroll
        for (int h = 0; h < W / 4; ++h) {
            const float4 t = *reinterpret_cast<const float4 *>(lds + i * FLOATS + (h * PIECES + piece) * 4);
            v[4 * h] = t.x; v[4 * h + 1] = t.y; v[4 * h + 2] = t.z; v[4 * h + 3] = t.w;
        }
    }
};

// gate of the lane's channels of a row (1 without a gate): the groups of first and last channel,
// then a value per channel
template <int NV> struct RnGate { float a[NV], b[NV]; };
template <int TPR, int NV, int W>
__device__ __forceinline__ void gate_load(const ResidualArgs &a, i64 row, const RnChannels<TPR, NV, W> &ch, RnGate<NV> &g)
{
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        g.a[j] = a.gate ? a.gate[row * a.G + ch.ga[j]] : 1.0f;
        g.b[j] = a.gate ? a.gate[row * a.G + ch.gb[j]] : 1.0f;
    }
}
template <int TPR, int NV, int W>
__device__ __forceinline__ void gate_values(const ResidualArgs &a, i64 row, const RnChannels<TPR, NV, W> &ch, const RnGate<NV> &g,
                                            float (&v)[NV][W])
{
    if (ch.simple()) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int k = 0; k < W; ++k) v[j][k] = k < ch.cut[j] ? g.a[j] : g.b[j];
    } else {                // groups narrower than a piece
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            int q = ch.ga[j], rest = ch.col[j] - q * ch.gw;
#pragma unroll
            for (int k = 0; k < W; ++k) {
                v[j][k] = a.gate[row * a.G + min(q, a.G - 1)];
                if (++rest == ch.gw) { rest = 0; ++q; }
            }
        }
    }
}

// 1 / spread and mean (0 for an RMS norm) of a team's row
template <int TPR, int NV, int W>
__device__ __forceinline__ void rn_stats(const float (&v)[NV][W], const RnChannels<TPR, NV, W> &ch, int C, int kind, float eps,
                                         float *lds, int &turn, float &r, float &mu)
{
    mu = 0.0f;
    if (kind == RN_LAYER) {
        float s[1] = {0.0f};
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int k = 0; k < W; ++k) s[0] += v[j][k];            // (channels past C hold zeros)
        team_sum<TPR, 1>(s, lds, turn);
        mu = s[0] * ch.inv_c;
    }
    float s[1] = {0.0f};
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int k = 0; k < W; ++k) {
            const float d = kind == RN_LAYER ? (ch.col[j] + k < C ? v[j][k] - mu : 0.0f) : v[j][k];
            s[0] = __fmaf_rn(d, d, s[0]);
        }
    team_sum<TPR, 1>(s, lds, turn);
    // the hardware's estimate (1 ulp) and one Newton step
    const float t = __fmaf_rn(s[0], ch.inv_c, eps);
    r = __builtin_amdgcn_rsqf(t);
    const float c = __fmaf_rn(-t * r, r, 1.0f);
    if (t >= 1.17549435e-38f && t < INFINITY) r = __fmaf_rn(0.5f * r, c, r);
}

template <class R, int TPR, int NV, bool VEC, int W = RnPiece<R>::W>
__device__ __forceinline__ void rn_encode(int8_t *codes, uint8_t *exps, i64 row, const int (&col)[NV], int C, const float (&v)[NV][W])
{
    const int GR = (C + R8_GROUP - 1) / R8_GROUP;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        unsigned m = 0;
#pragma unroll
        for (int k = 0; k < W; ++k) m = max(m, r8_magnitude(v[j][k]));
        m = W == 4 && TPR >= 8 ? r8_max8(m) : r8_max4(m);         // (a row of 4 lanes is one group)
        const int e = r8_exponent(m, R::E_MAX);
        unsigned q[W / 4];
#pragma unroll
        for (int i = 0; i < W / 4; ++i) {
            const int t[4] = {r8_encode(v[j][4 * i], e), r8_encode(v[j][4 * i + 1], e), r8_encode(v[j][4 * i + 2], e),
                              r8_encode(v[j][4 * i + 3], e)};
            q[i] = r8_pack4(t);
        }
        piece_codes_store<W, VEC>(codes + row * C, col[j], C, q);
        if (col[j] < C && col[j] % R8_GROUP == 0) exps[row * GR + col[j] / R8_GROUP] = (uint8_t)e;
    }
}

// ---- forward ----------------------------------------------------------------------------------
template <class R, int TPR, int NV, bool VEC>
__global__ __launch_bounds__(RnBlock<TPR>::THREADS, rn_waves_fwd(NV * RnPiece<R>::W)) void residual_forward_kernel(
    const ResidualArgs a, void *__restrict__ out_, void *__restrict__ h_,
    int8_t *__restrict__ qx, uint8_t *__restrict__ ex, int8_t *__restrict__ qf, uint8_t *__restrict__ ef)
{
    typedef typename R::T Tv;
    constexpr int W = RnPiece<R>::W;
    constexpr int TEAMS = RnBlock<TPR>::TEAMS;
    __shared__ float lds[TPR > 64 ? 2 * RN_LDS : 1];
    int turn = 0;
    const int C = a.C;
    const Tv *xs = (const Tv *)a.x, *fs = (const Tv *)a.f;
    Tv *outs = (Tv *)out_, *hs = (Tv *)h_;
    RnChannels<TPR, NV, W> ch;
    ch.init(C, a.G);
    // scale w_post, scale b_post, w_pre, b_pre
    typedef RnVectors<TPR, NV, W, 4> V;
    __shared__ __attribute__((aligned(16))) float vec[4 * V::FLOATS];
    V::fill(vec, 0, a.w_post, C, 1.0f, a.scale);
    V::fill(vec, 1, a.b_post, C, 0.0f, a.scale);
    V::fill(vec, 2, a.w_pre, C, 1.0f);
    V::fill(vec, 3, a.b_pre, C, 0.0f);
    __syncthreads();

    // a row's words on their way: x and, where it adds something, f and its gate
    struct Ahead {
        unsigned x[NV][4], f[NV][4];
        RnGate<NV> g;
        bool adds;
    };
    const i64 stride = (i64)gridDim.x * TEAMS;
    auto seen_at = [&](i64 row) { return fs && (!a.seen || (row < a.rows && a.seen[row])); };
    auto fetch = [&](Ahead &p, i64 row, bool adds) {
        p.adds = adds;
#pragma unroll
        for (int j = 0; j < NV; ++j) piece_load<R, VEC>(xs + row * C, ch.col[j], C, p.x[j]);
        if (adds) {
#pragma unroll
            for (int j = 0; j < NV; ++j) piece_load<R, VEC>(fs + row * C, ch.col[j], C, p.f[j]);
            gate_load(a, row, ch, p.g);
        } else {
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) p.f[j][i] = 0u;
        }
    };
    i64 row = (i64)blockIdx.x * TEAMS + threadIdx.x / TPR;
    if (row >= a.rows) return;              // (a whole team; a workgroup of one team has no barrier to miss)
    Ahead p;
    fetch(p, row, seen_at(row));
    bool adds_next = seen_at(row + stride);
    for (; row < a.rows; row += stride) {
        float x[NV][W], f[NV][W], g[NV][W];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            piece_values<R>(p.x[j], x[j]);
            piece_values<R>(p.f[j], f[j]);
        }
        const bool adds = p.adds;           // (the same in all lanes of a team)
        if (adds) gate_values(a, row, ch, p.g, g);
        if (row + stride < a.rows) {
            fetch(p, row + stride, adds_next);
            adds_next = seen_at(row + 2 * stride);
        }
        if (qx) rn_encode<R, TPR, NV, VEC>(qx, ex, row, ch.col, C, x);
        if (qf) rn_encode<R, TPR, NV, VEC>(qf, ef, row, ch.col, C, f);
        float r = 1.0f, mu = 0.0f;
        if (adds) {
            if (a.post != RN_NONE) rn_stats<TPR, NV, W>(f, ch, C, a.post, a.eps_post, lds, turn, r, mu);
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                float w[W], b[W];
                V::read(vec, 0, j, w);
                V::read(vec, 1, j, b);
#pragma unroll
                for (int k = 0; k < W; ++k)         // (channels past C: w and b are 0)
                    x[j][k] = __fmaf_rn(g[j][k], __fmaf_rn((f[j][k] - mu) * r, w[k], b[k]), x[j][k]);
            }
        }
        if (outs)
#pragma unroll
            for (int j = 0; j < NV; ++j) piece_store<R, VEC>(outs + row * C, ch.col[j], C, x[j]);
        float r2 = 1.0f, mu2 = 0.0f;
        if (a.pre != RN_NONE) {
            rn_stats<TPR, NV, W>(x, ch, C, a.pre, a.eps_pre, lds, turn, r2, mu2);
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                float y[W], w[W], b[W];
                V::read(vec, 2, j, w);
                V::read(vec, 3, j, b);
#pragma unroll
                for (int k = 0; k < W; ++k) y[k] = __fmaf_rn((x[j][k] - mu2) * r2, w[k], b[k]);
                piece_store<R, VEC>(hs + row * C, ch.col[j], C, y);
            }
        }
        if (a.stats && threadIdx.x % TPR == 0) {
            a.stats[row] = r;
            a.stats[a.rows + row] = mu;
            a.stats[2 * a.rows + row] = r2;
            a.stats[3 * a.rows + row] = mu2;
        }
    }
}

// ---- backward ---------------------------------------------------------------------------------
// KEPT8: x and f come as 8-bit rows.
template <class R, int TPR, int NV, bool VEC, bool KEPT8>
__global__ __launch_bounds__(RnBlock<TPR>::THREADS, rn_waves_bwd(NV * RnPiece<R>::W)) void residual_backward_kernel(
    const ResidualArgs a, const void *__restrict__ d_out_, const void *__restrict__ d_h_,
    void *__restrict__ d_x_, void *__restrict__ d_f_, float *__restrict__ d_gate, float *__restrict__ partial)
{
    typedef typename R::T Tv;
    constexpr int W = RnPiece<R>::W;
    constexpr int TEAMS = RnBlock<TPR>::TEAMS, THREADS = RnBlock<TPR>::THREADS;
    __shared__ float lds[TPR > 64 ? 2 * RN_LDS : 1];
    __shared__ float fold[THREADS * W * NV];
    int turn = 0;
    const int C = a.C, GR = (C + R8_GROUP - 1) / R8_GROUP;
    const Tv *d_outs = (const Tv *)d_out_, *d_hs = a.pre != RN_NONE ? (const Tv *)d_h_ : nullptr;
    Tv *d_xs = (Tv *)d_x_, *d_fs = (Tv *)d_f_;
    const bool has_f = KEPT8 ? a.qf != nullptr : a.f != nullptr;
    RnChannels<TPR, NV, W> ch;
    ch.init(C, a.G);
    // scale w_post, scale b_post, w_pre
    typedef RnVectors<TPR, NV, W, 3> V;
    __shared__ __attribute__((aligned(16))) float vec[3 * V::FLOATS];
    V::fill(vec, 0, a.w_post, C, 1.0f, a.scale);
    V::fill(vec, 1, a.b_post, C, 0.0f, a.scale);
    V::fill(vec, 2, a.w_pre, C, 1.0f);
    __syncthreads();
    // column sums: d gate n, d gate, dh o, dh
    float acc[4][NV][W];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int k = 0; k < W; ++k) acc[i][j][k] = 0.0f;
    const float inv_c = 1.0f / (float)C;

    struct Kept {                           // x or f of a row on its way
        unsigned w[NV][KEPT8 ? W / 4 : 4];
        int e[NV];
    };
    struct Ahead {
        unsigned d[NV][4], h[NV][4];
        Kept x, f;
        RnGate<NV> g;
        float rf, muf, ro, muo;
        bool adds;
    };
    auto kept_load = [&](Kept &k, const int8_t *codes, const uint8_t *exps, const Tv *rows, i64 row) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if constexpr (KEPT8) {
                piece_codes_load<W, VEC>(codes + row * C, ch.col[j], C, k.w[j]);
                k.e[j] = exps[row * GR + min(ch.col[j], C - 1) / R8_GROUP];
            } else {
                piece_load<R, VEC>(rows + row * C, ch.col[j], C, k.w[j]);
            }
        }
    };
    auto kept_values = [&](const Kept &k, float (&v)[NV][W]) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if constexpr (KEPT8) {
#pragma unroll
                for (int i = 0; i < W; ++i) v[j][i] = r8_decode(r8_byte(k.w[j][i / 4], i % 4), k.e[j]);
            } else {
                piece_values<R>(k.w[j], v[j]);
            }
        }
    };
    auto zero = [](unsigned (&w)[NV][4]) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) w[j][i] = 0u;
    };
    auto seen_at = [&](i64 row) { return has_f && (!a.seen || (row < a.rows && a.seen[row])); };
    auto fetch = [&](Ahead &p, i64 row, bool adds) {
        p.adds = adds;
        if (d_outs) {
#pragma unroll
            for (int j = 0; j < NV; ++j) piece_load<R, VEC>(d_outs + row * C, ch.col[j], C, p.d[j]);
        } else {
            zero(p.d);
        }
        if (d_hs) {
#pragma unroll
            for (int j = 0; j < NV; ++j) piece_load<R, VEC>(d_hs + row * C, ch.col[j], C, p.h[j]);
            kept_load(p.x, a.qx, a.ex, (const Tv *)a.x, row);
            p.ro = a.stats[2 * a.rows + row];
            p.muo = a.stats[3 * a.rows + row];
        }
        if (adds) {
            kept_load(p.f, a.qf, a.ef, (const Tv *)a.f, row);
            gate_load(a, row, ch, p.g);
            if (a.post != RN_NONE) {
                p.rf = a.stats[row];
                p.muf = a.stats[a.rows + row];
            }
        }
    };
    const i64 stride = (i64)gridDim.x * TEAMS;
    i64 row = (i64)blockIdx.x * TEAMS + threadIdx.x / TPR;
    Ahead p;
    bool adds_next = false;
    if (row < a.rows) {
        fetch(p, row, seen_at(row));
        adds_next = seen_at(row + stride);
    }
    for (; row < a.rows; row += stride) {
        const bool adds = p.adds;
        const float rf = a.post != RN_NONE ? p.rf : 1.0f, ro = p.ro, muo = p.muo;
        float d[NV][W], n[NV][W], g[NV][W], o[NV][W], dh[NV][W];
#pragma unroll
        for (int j = 0; j < NV; ++j) piece_values<R>(p.d[j], d[j]);
        if (d_hs) {
#pragma unroll
            for (int j = 0; j < NV; ++j) piece_values<R>(p.h[j], dh[j]);
            kept_values(p.x, o);
        }
        if (adds) {
            kept_values(p.f, n);
            gate_values(a, row, ch, p.g, g);
            if (a.post != RN_NONE)
#pragma unroll
                for (int j = 0; j < NV; ++j)
#pragma unroll
                    for (int k = 0; k < W; ++k) n[j][k] = ch.col[j] + k < C ? (n[j][k] - p.muf) * rf : 0.0f;
        } else {
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int k = 0; k < W; ++k) n[j][k] = g[j][k] = 0.0f;
        }
        if (row + stride < a.rows) {
            fetch(p, row + stride, adds_next);
            adds_next = seen_at(row + 2 * stride);
        }
        if (d_hs) {
            float s[2] = {0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                float w[W], b[W], wp[W];
                V::read(vec, 0, j, w);
                V::read(vec, 1, j, b);
                V::read(vec, 2, j, wp);
#pragma unroll
                for (int k = 0; k < W; ++k) {
                    const float u = adds ? __fmaf_rn(g[j][k], __fmaf_rn(n[j][k], w[k], b[k]), o[j][k]) : o[j][k];
                    o[j][k] = ch.col[j] + k < C ? (u - muo) * ro : 0.0f;
                    acc[2][j][k] = __fmaf_rn(dh[j][k], o[j][k], acc[2][j][k]);
                    acc[3][j][k] += dh[j][k];
                    dh[j][k] *= wp[k];
                    s[0] = __fmaf_rn(dh[j][k], o[j][k], s[0]);
                    s[1] += dh[j][k];
                }
            }
            team_sum<TPR, 2>(s, lds, turn);
            const float m0 = s[0] * inv_c, m1 = a.pre == RN_LAYER ? s[1] * inv_c : 0.0f;
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int k = 0; k < W; ++k) d[j][k] += ro * ((dh[j][k] - m1) - o[j][k] * m0);
        }
        if (d_xs)
#pragma unroll
            for (int j = 0; j < NV; ++j) piece_store<R, VEC>(d_xs + row * C, ch.col[j], C, d[j]);
        if (!has_f) continue;               // (the same in every lane)
        float e[NV][W];
        float s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float w[W];
            V::read(vec, 0, j, w);
#pragma unroll
            for (int k = 0; k < W; ++k) {
                const float dg = adds ? d[j][k] * g[j][k] : 0.0f;
                acc[0][j][k] = __fmaf_rn(dg, n[j][k], acc[0][j][k]);
                acc[1][j][k] += dg;
                e[j][k] = dg * w[k];
                s[0] = __fmaf_rn(e[j][k], n[j][k], s[0]);
                s[1] += e[j][k];
            }
        }
        if (d_fs) {
            if (a.post != RN_NONE) {
                team_sum<TPR, 2>(s, lds, turn);
                const float m0 = s[0] * inv_c, m1 = a.post == RN_LAYER ? s[1] * inv_c : 0.0f;
#pragma unroll
                for (int j = 0; j < NV; ++j)
#pragma unroll
                    for (int k = 0; k < W; ++k) e[j][k] = adds ? rf * ((e[j][k] - m1) - n[j][k] * m0) : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < NV; ++j) piece_store<R, VEC>(d_fs + row * C, ch.col[j], C, e[j]);
        }
        if (d_gate) {
            // d scale v of every channel, summed per group: four groups at a time
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                float w[W], b[W];
                V::read(vec, 0, j, w);
                V::read(vec, 1, j, b);
#pragma unroll
                for (int k = 0; k < W; ++k)
                    e[j][k] = adds && ch.col[j] + k < C ? d[j][k] * __fmaf_rn(n[j][k], w[k], b[k]) : 0.0f;
            }
            float pa[NV], pb[NV];           // the piece's part in its first and in its last group
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                pa[j] = pb[j] = 0.0f;
#pragma unroll
                for (int k = 0; k < W; ++k) {
                    pa[j] += k < ch.cut[j] ? e[j][k] : 0.0f;
                    pb[j] += k < ch.cut[j] ? 0.0f : e[j][k];
                }
            }
            for (int q0 = 0; q0 < a.G; q0 += 4) {
                float t[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    t[i] = 0.0f;
                    if (ch.simple()) {
#pragma unroll
                        for (int j = 0; j < NV; ++j) {
                            t[i] += ch.ga[j] == q0 + i ? pa[j] : 0.0f;
                            t[i] += ch.gb[j] == q0 + i ? pb[j] : 0.0f;
                        }
                    } else {
                        const int c0 = (q0 + i) * ch.gw, c1 = c0 + ch.gw;
#pragma unroll
                        for (int j = 0; j < NV; ++j)
#pragma unroll
                            for (int k = 0; k < W; ++k)
                                t[i] += ch.col[j] + k >= c0 && ch.col[j] + k < c1 ? e[j][k] : 0.0f;
                    }
                }
                team_sum<TPR, 4>(t, lds, turn);
                if (threadIdx.x % TPR == 0)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (q0 + i < a.G) d_gate[row * a.G + q0 + i] = t[i];
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
            for (int k = 0; k < W; ++k) fold[(threadIdx.x / TPR * TPR * NV + j * TPR + threadIdx.x % TPR) * W + k] = acc[i][j][k];
        __syncthreads();
        for (int c = threadIdx.x; c < C; c += THREADS) {
            float s = fold[c];
            for (int t = 1; t < TEAMS; ++t) s += fold[t * TPR * NV * W + c];
            partial[((size_t)blockIdx.x * 4 + i) * C + c] = s;
        }
    }
}

// Column gradients from the workgroups' sums: 4 columns and 64 slices of the workgroups a block.
constexpr int RN_FOLD_COLS = 4, RN_FOLD_SLICES = RN_THREADS / RN_FOLD_COLS;
__global__ __launch_bounds__(RN_THREADS) void residual_fold_kernel(
    const float *__restrict__ partial, int nblk, int C, const float *__restrict__ scale,
    const float *__restrict__ w_post, const float *__restrict__ b_post,
    float *__restrict__ d_scale, float *__restrict__ d_w_post, float *__restrict__ d_b_post,
    float *__restrict__ d_w_pre, float *__restrict__ d_b_pre)
{
    __shared__ double red[4][RN_FOLD_SLICES][RN_FOLD_COLS];
    const int c0 = threadIdx.x % RN_FOLD_COLS, slice = threadIdx.x / RN_FOLD_COLS, c = blockIdx.x * RN_FOLD_COLS + c0;
    double s[4] = {0.0, 0.0, 0.0, 0.0};
    if (c < C) {
        int b = slice;
        for (; b + 3 * RN_FOLD_SLICES < nblk; b += 4 * RN_FOLD_SLICES) {
            float v[4][4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) v[u][i] = partial[((size_t)(b + u * RN_FOLD_SLICES) * 4 + i) * C + c];
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[i] += (double)v[u][i];
        }
        for (; b < nblk; b += RN_FOLD_SLICES)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] += (double)partial[((size_t)b * 4 + i) * C + c];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) red[i][slice][c0] = s[i];
    __syncthreads();
    for (int half = RN_FOLD_SLICES / 2; half >= 1; half >>= 1) {
        if (slice < half)
#pragma unroll
            for (int i = 0; i < 4; ++i) red[i][slice][c0] += red[i][slice + half][c0];
        __syncthreads();
    }
    if (slice != 0 || c >= C) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = red[i][0][c0];
    const double sc = scale ? scale[c] : 1.0, w = w_post ? w_post[c] : 1.0, b = b_post ? b_post[c] : 0.0;
    if (d_scale) d_scale[c] = (float)(w * s[0] + b * s[1]);
    if (d_w_post) d_w_post[c] = (float)(sc * s[0]);
    if (d_b_post) d_b_post[c] = (float)(sc * s[1]);
    if (d_w_pre) d_w_pre[c] = (float)s[2];
    if (d_b_pre) d_b_pre[c] = (float)s[3];
}

// Team of a row of C channels, by its pieces of 16 bytes: one to three pieces a lane, so that few lanes
// are idle (35 pieces on 48 places instead of 64: 300000 x 137 float32 forward 287 -> 204 us) and a row
// stays inside one wave as long as it can (sums without barriers: 60000 x 600 float32 backward 291 -> 232
// us).  Backward a lane has one piece where that fills the team: its column sums take four registers a
// channel (500000 x 64: 166 us with two pieces, 153 with one).
struct RnShape { int tpr, nv; };
static RnShape rn_shape(int C, int type, bool forward)
{
    const int p = type == R8_F32 ? (C + 3) / 4 : (C + 7) / 8;       // pieces of a row
    if (p <= 4) return {4, 1};
    if (p <= 8) return {8, 1};
    if (type == R8_F32) {
        if (p <= 16) return forward ? RnShape{8, 2} : RnShape{16, 1};
        if (p <= 24) return {8, 3};
        if (p <= 32) return forward ? RnShape{16, 2} : RnShape{32, 1};
        if (p <= 48) return {16, 3};
        if (p <= 64) return forward ? RnShape{32, 2} : RnShape{64, 1};
        if (p <= 96) return {32, 3};
        if (p <= 128) return {64, 2};
        if (p <= 192) return {64, 3};
        if (p <= 256) return {64, 4};
        return p <= 512 ? RnShape{256, 2} : RnShape{256, 4};
    }
    if (p <= 16) return {16, 1};
    if (p <= 32) return {32, 1};
    if (p <= 64) return {64, 1};
    if (p <= 128) return {64, 2};
    if (p <= 192) return {64, 3};
    return p <= 256 ? RnShape{256, 1} : RnShape{256, 2};
}

static unsigned rn_blocks(i64 rows, RnShape shape, int waves, int most)
{
    int dev = 0, cus = 256;
    if (hipGetDevice(&dev) != hipSuccess ||
        hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus < 1) cus = 256;
    const int teams = shape.tpr > 64 ? 1 : RN_THREADS / shape.tpr;
    const i64 full = (i64)cus * waves;
    i64 n = (rows + teams - 1) / teams;
    if (n > full) n = full;
    if (n > most) n = most;
    return (unsigned)(n < 1 ? 1 : n);
}

static bool rn_vec(const ResidualArgs &a, int type, const void *const *rows, int n)
{
    if (a.C % (type == R8_F32 ? 4 : 8) != 0) return false;
    for (int i = 0; i < n; ++i)
        if ((uintptr_t)rows[i] % 16 != 0) return false;
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

#define MVF_RN_SHAPES_16(R_, V_)                                                                    \
    do {                                                                                            \
        switch (shape.tpr * 16 + shape.nv) {                                                        \
        case 4 * 16 + 1: MVF_RN_LAUNCH(R_, 4, 1, V_); break;                                        \
        case 8 * 16 + 1: MVF_RN_LAUNCH(R_, 8, 1, V_); break;                                        \
        case 16 * 16 + 1: MVF_RN_LAUNCH(R_, 16, 1, V_); break;                                      \
        case 32 * 16 + 1: MVF_RN_LAUNCH(R_, 32, 1, V_); break;                                      \
        case 64 * 16 + 1: MVF_RN_LAUNCH(R_, 64, 1, V_); break;                                      \
        case 64 * 16 + 2: MVF_RN_LAUNCH(R_, 64, 2, V_); break;                                      \
        case 64 * 16 + 3: MVF_RN_LAUNCH(R_, 64, 3, V_); break;                                      \
        case 256 * 16 + 1: MVF_RN_LAUNCH(R_, 256, 1, V_); break;                                    \
        default: MVF_RN_LAUNCH(R_, 256, 2, V_); break;                                              \
        }                                                                                           \
    } while (0)
#define MVF_RN_SHAPES_32(R_, V_)                                                                    \
    do {                                                                                            \
        switch (shape.tpr * 16 + shape.nv) {                                                        \
        case 4 * 16 + 1: MVF_RN_LAUNCH(R_, 4, 1, V_); break;                                        \
        case 8 * 16 + 1: MVF_RN_LAUNCH(R_, 8, 1, V_); break;                                        \
        case 8 * 16 + 3: MVF_RN_LAUNCH(R_, 8, 3, V_); break;                                        \
        case 16 * 16 + 3: MVF_RN_LAUNCH(R_, 16, 3, V_); break;                                      \
        case 32 * 16 + 3: MVF_RN_LAUNCH(R_, 32, 3, V_); break;                                      \
        case 64 * 16 + 2: MVF_RN_LAUNCH(R_, 64, 2, V_); break;                                      \
        case 64 * 16 + 3: MVF_RN_LAUNCH(R_, 64, 3, V_); break;                                      \
        case 64 * 16 + 4: MVF_RN_LAUNCH(R_, 64, 4, V_); break;                                      \
        case 256 * 16 + 2: MVF_RN_LAUNCH(R_, 256, 2, V_); break;                                    \
        MVF_RN_OWN(R_, V_)                                                                          \
        default: MVF_RN_LAUNCH(R_, 256, 4, V_); break;                                              \
        }                                                                                           \
    } while (0)
#define MVF_RN_TYPES()                                                                              \
    do {                                                                                            \
        if (type == R8_F32) { if (vec) MVF_RN_SHAPES_32(RowF32, true); else MVF_RN_SHAPES_32(RowF32, false); }         \
        else if (type == R8_BF16) { if (vec) MVF_RN_SHAPES_16(RowBF16, true); else MVF_RN_SHAPES_16(RowBF16, false); } \
        else { if (vec) MVF_RN_SHAPES_16(RowF16, true); else MVF_RN_SHAPES_16(RowF16, false); }     \
    } while (0)

#define MVF_RN_OWN(R_, V_)                                                                          \
    case 8 * 16 + 2: MVF_RN_LAUNCH(R_, 8, 2, V_); break;                                            \
    case 16 * 16 + 2: MVF_RN_LAUNCH(R_, 16, 2, V_); break;                                          \
    case 32 * 16 + 2: MVF_RN_LAUNCH(R_, 32, 2, V_); break;
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
    const bool vec = rn_vec(a, type, ptrs, 4) && (uintptr_t)x_codes % 8 == 0 && (uintptr_t)f_codes % 8 == 0;
    const RnShape shape = rn_shape(C, type, true);
    const dim3 grid(rn_blocks(rows, shape, rn_waves_fwd(shape.nv * (type == R8_F32 ? 4 : 8)), 1 << 30));
    hipStream_t st = (hipStream_t)stream;
#define MVF_RN_LAUNCH(R_, TPR_, NV_, V_)                                                                          \
    hipLaunchKernelGGL((residual_forward_kernel<R_, TPR_, NV_, V_>), grid, dim3(RnBlock<TPR_>::THREADS), 0, st, a, out, h, x_codes, \
                       x_exps, f_codes, f_exps)
    MVF_RN_TYPES();
#undef MVF_RN_LAUNCH
    MVF_LAUNCH_CHECK();
    return MVF_OK;
}

#undef MVF_RN_OWN

#define MVF_RN_OWN(R_, V_)                                                                          \
    case 16 * 16 + 1: MVF_RN_LAUNCH(R_, 16, 1, V_); break;                                          \
    case 32 * 16 + 1: MVF_RN_LAUNCH(R_, 32, 1, V_); break;                                          \
    case 64 * 16 + 1: MVF_RN_LAUNCH(R_, 64, 1, V_); break;
extern "C" size_t mvf_residual_norm_workspace_bytes(int64_t rows, int32_t C)
{
    if (rows < 1 || C < 1 || C > RN_MAX_C) return 0;
    // (at most one workgroup per row, whatever the type's teams)
    const i64 most = rows < RN_MAX_BLOCKS_BWD ? rows : RN_MAX_BLOCKS_BWD;
    return align_up((size_t)most * 4 * (size_t)C * sizeof(float));
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
    const bool kept8 = x_codes || f_codes;
    MVF_REQUIRE(!kept8 || (!x && !f), "residual_norm_backward: x and f either both as they are or both as 8-bit rows");
    MVF_REQUIRE(!d_gate || gate, "residual_norm_backward: a gradient of the gate without a gate");
    MVF_REQUIRE(!columns || rows == 0 || (workspace && workspace_bytes >= mvf_residual_norm_workspace_bytes(rows, C)),
                "residual_norm_backward: workspace too small");
    hipStream_t st = (hipStream_t)stream;
    const RnShape shape = rn_shape(C, type, false);
    const dim3 grid(rn_blocks(rows, shape, rn_waves_bwd(shape.nv * (type == R8_F32 ? 4 : 8)), RN_MAX_BLOCKS_BWD));
    float *partial = columns ? (float *)workspace : nullptr;
    if (rows > 0) {
        const void *const ptrs[] = {x, f, d_out, d_h, d_x, d_f};
        const bool vec = rn_vec(a, type, ptrs, 6) && (uintptr_t)x_codes % 8 == 0 && (uintptr_t)f_codes % 8 == 0;
#define MVF_RN_LAUNCH(R_, TPR_, NV_, V_)                                                                          \
    do {                                                                                                          \
        if (kept8) hipLaunchKernelGGL((residual_backward_kernel<R_, TPR_, NV_, V_, true>), grid, dim3(RnBlock<TPR_>::THREADS), \
                                      0, st, a, d_out, d_h, d_x, d_f, d_gate, partial);                           \
        else hipLaunchKernelGGL((residual_backward_kernel<R_, TPR_, NV_, V_, false>), grid, dim3(RnBlock<TPR_>::THREADS), \
                                0, st, a, d_out, d_h, d_x, d_f, d_gate, partial);                                 \
    } while (0)
        MVF_RN_TYPES();
#undef MVF_RN_LAUNCH
    }
    if (columns)
        hipLaunchKernelGGL(residual_fold_kernel, dim3(cdiv(C, RN_FOLD_COLS)), dim3(RN_THREADS), 0, st, (const float *)partial,
                           rows > 0 ? (int)grid.x : 0, (int)C, scale, w_post, b_post, d_scale, d_w_post, d_b_post, d_w_pre, d_b_pre);
    MVF_LAUNCH_CHECK();
    return MVF_OK;
}
