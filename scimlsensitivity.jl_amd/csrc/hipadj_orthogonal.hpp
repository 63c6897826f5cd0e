// hipadj_orthogonal.hpp — the orthogonalised update: momentum, then Newton-Schulz products X <- c0 X + (c1 A + c2 A A) X with A = X X'.
//
// With X m x n, m <= n (a tall matrix is taken by its columns: the iteration commutes with transposition), a step is three products on the matrix cores,
//   A = X X' (m x m),   B = c1 A + c2 A A (m x m),   X <- c0 X + B X (m x n),
// each a launch with its linear term in the epilogue.  A and B are symmetric: their tiles on and below the diagonal are computed and stored twice, 3 m m n + m m m operations a step
// instead of 4 m m n + 2 m m m.
//
// Numbers.  The products take F16 factors and accumulate in F32.  F16 rather than BF16 at the same rate: a factor is known to lie within a few powers of two (|X|_2 <= 1.2 for the
// usual coefficients, |B| <= 8), so its 5 exponent bits suffice and its 11-bit significand rounds 8 times finer.  X is held as 2^13 X and A, B as 2^11 A, 2^11 B: small entries
// stay in the normal range and the largest possible ones below 65504.
//   * two terms a factor (SPLIT): v = hi + lo, hi hi + hi lo + lo hi — three products, 22 bits, the accuracy of a plain F32 evaluation (the term left out is 2^-22 of the result);
//   * one term (BF16 output, both sides >= 256): a third of the work.  Two choices keep its error at about that of rounding the output to BF16 (measured 1.2 ... 1.7e-3 of the
//     norm): B is formed from the ROUNDED A, so that it is an exact polynomial of the matrix that is squared; and X in c0 X is the F32 value while small singular values still grow by
//     c0 a step (rounding X there would put noise of the large ones into them), but the rounded one in the last two steps, where X + dX goes through the polynomial as a whole.
// Sums of squares are formed in 64 bits: a gradient of 1e-25 has a norm.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace orth {

typedef _Float16 f16;
typedef __bf16 bf16;
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr float SX = 8192.f, SA = 2048.f;     // X and A, B are stored times these
constexpr int BK = 64;                        // depth of a stage: a row of it is 128 bytes, eight 16-byte chunks
constexpr int PADDED = 128;                   // sides are padded with zeros to multiples of this (the smaller tile), so the products have no edges

struct Mat {                                  // one batch of matrices and the workspace it is computed in
    int64_t m, n, mp, np;                     // m <= n; padded
    int64_t batch;
    bool flip;                                // X is the transpose of the caller's matrix
    f16 *x[2], *xt[2][2], *a[2], *b[2];       // [term]: x [batch][mp][np]; xt[buffer][term] [batch][np][mp]; a, b [batch][mp][mp]
    float* master;                            // 2^13 X in F32, transposed [batch][np][mp]
    double* partial;                          // [batch][NORM_BLOCKS]
};
constexpr int NORM_BLOCKS = 64;

// ---- gradient, momentum, norm -------------------------------------------------------------------------------------------------------------------------------------------
template <class T> struct Io {
    const T* grad; float* mom; T* out;
    int64_t rows, cols, g_b, g_r, m_b, m_r, o_b, o_r;
    float beta, scale;
    int nesterov;
};
template <class T> __device__ inline float moved(const Io<T>& io, int64_t b, int64_t r, int64_t c, bool update) {
    const float g = (float)io.grad[b * io.g_b + r * io.g_r + c];
    if (!io.mom) return g;
    float* mp = io.mom + b * io.m_b + r * io.m_r + c;
    float m = *mp;
    if (update) { m = io.beta * m + g; *mp = m; }
    return io.nesterov ? g + io.beta * m : m;
}

__device__ inline double block_sum(double v) {       // 256 threads, fixed order
    __shared__ double s[4];
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    return (s[0] + s[1]) + (s[2] + s[3]);
}

template <class T> __global__ void __launch_bounds__(256) k_norm(const Io<T> io, double* partial) {
    const int64_t b = blockIdx.y, count = io.rows * io.cols;
    double s = 0;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)NORM_BLOCKS * 256) {
        const float u = moved(io, b, i / io.cols, i % io.cols, true);
        s += (double)u * (double)u;
    }
    s = block_sum(s);
    if (threadIdx.x == 0) partial[b * NORM_BLOCKS + blockIdx.x] = s;
}

template <bool SPLIT> __device__ inline void terms(float v, f16& hi, f16& lo) { hi = (f16)v; if constexpr (SPLIT) lo = (f16)(v - (float)hi); }

// X = u / (|u| + 1e-7) in both orders, padding included.  A workgroup takes a 64 x 64 piece through LDS.
template <class T, bool SPLIT> __global__ void __launch_bounds__(256) k_start(const Io<T> io, const Mat q) {
    __shared__ float tile[64][65];
    const int64_t b = blockIdx.z, i0 = (int64_t)blockIdx.y * 64, j0 = (int64_t)blockIdx.x * 64;      // rows and columns of X
    double s = threadIdx.x < NORM_BLOCKS ? q.partial[b * NORM_BLOCKS + threadIdx.x] : 0.0;
    s = block_sum(s);
    const double inv = (double)SX / (sqrt(s) + 1e-7);
    const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
    for (int r = w; r < 64; r += 4) {                         // lanes run along the caller's rows
        const int64_t i = q.flip ? i0 + l : i0 + r, j = q.flip ? j0 + r : j0 + l;
        float v = 0.f;
        if (i < q.m && j < q.n) v = (float)((double)(q.flip ? moved(io, b, j, i, false) : moved(io, b, i, j, false)) * inv);
        tile[q.flip ? l : r][q.flip ? r : l] = v;
    }
    __syncthreads();
    for (int r = w; r < 64; r += 4) {
        f16 hi, lo;
        terms<SPLIT>(tile[r][l], hi, lo);
        const int64_t at = (b * q.mp + i0 + r) * q.np + j0 + l;
        q.x[0][at] = hi;
        if constexpr (SPLIT) q.x[1][at] = lo;
        const float v = tile[l][r];
        terms<SPLIT>(v, hi, lo);
        const int64_t att = (b * q.np + j0 + r) * q.mp + i0 + l;
        q.xt[0][0][att] = hi;
        if constexpr (SPLIT) q.xt[0][1][att] = lo;
        q.master[att] = v;
    }
}

// ---- products ---------------------------------------------------------------------------------------------------------------------------------------------------------
// C[i][j] = sum_k P[i][k] Q[j][k] over padded sizes: both factors have k next to k.  A workgroup of four waves (2 x 2) takes a BT x BT tile, a wave BT / 2 x BT / 2 of it in
// accumulators; stages of BK go through two LDS buffers, the next one in registers while this one is multiplied.  Chunk c of row r is stored at c ^ (r & 7): the eight
// rows that a read touches together lie in different banks.
enum { GRAM = 0, POLY = 1, APPLY = 2, LAST = 3 };

struct Product {
    const f16 *P[2], *Q[2];                   // terms
    int64_t sP, sQ;                           // matrix strides
    int64_t K, M, N;                          // padded: P [M][K], Q [N][K]
    float c0, c1, c2;
    bool rounded;                             // APPLY, LAST: X in c0 X is the rounded one
    bool keep;                                // APPLY: the next step needs the F32 X
};

__device__ inline f32x16 mfma(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

template <class T, int BT, int EPI, bool SPLIT>
__global__ void __launch_bounds__(256, BT == 256 ? 1 : 2) k_product(const Product g, const Mat q, const Io<T> io, const int from, const int to) {
    constexpr int CH = BT * 8 / 256;          // 16-byte chunks a thread moves per factor and stage
    constexpr int W = BT / 64;                // 32 x 32 accumulators a wave and direction
    __shared__ __align__(16) f16 lds[2][2][BT * BK];
    const int64_t b = blockIdx.z;
    int bi, bj;
    if constexpr (EPI == GRAM || EPI == POLY) {               // tile t of the lower triangle
        const int t = blockIdx.x;
        bi = (int)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
        while ((bi + 1) * (bi + 2) / 2 <= t) ++bi;
        while (bi * (bi + 1) / 2 > t) --bi;
        bj = t - bi * (bi + 1) / 2;
    } else { bi = blockIdx.y; bj = blockIdx.x; }
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, wi = wave >> 1, wj = wave & 1;
    const int64_t i0 = (int64_t)bi * BT, j0 = (int64_t)bj * BT;
    f32x16 acc[W][W];
#pragma unroll
    for (int x = 0; x < W; ++x)
#pragma unroll
        for (int y = 0; y < W; ++y)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[x][y][r] = 0.f;
    f16x8 gp[CH], gq[CH];
    const int per = (int)(g.K / BK), stages = SPLIT ? 3 * per : per;
    auto fetch = [&](int s) {
        const int part = SPLIT ? s / per : 0, k = (SPLIT ? s % per : s) * BK;
        const f16* P = g.P[SPLIT && part == 2 ? 1 : 0] + b * g.sP;
        const f16* Q = g.Q[SPLIT && part == 1 ? 1 : 0] + b * g.sQ;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int id = c * 256 + tid, row = id >> 3, ch = id & 7;
            gp[c] = *(const f16x8*)(P + (i0 + row) * g.K + k + ch * 8);
            gq[c] = *(const f16x8*)(Q + (j0 + row) * g.K + k + ch * 8);
        }
    };
    auto stash = [&](int buf) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int id = c * 256 + tid, row = id >> 3, ch = (id & 7) ^ (row & 7);
            *(f16x8*)&lds[buf][0][row * BK + ch * 8] = gp[c];
            *(f16x8*)&lds[buf][1][row * BK + ch * 8] = gq[c];
        }
    };
    fetch(0);
    stash(0);
    __syncthreads();
    for (int s = 0; s < stages; ++s) {
        if (s + 1 < stages) fetch(s + 1);
        const f16* lp = lds[s & 1][0] + (wi * (BT / 2) + (lane & 31)) * BK;
        const f16* lq = lds[s & 1][1] + (wj * (BT / 2) + (lane & 31)) * BK;
#pragma unroll
        for (int k = 0; k < BK / 16; ++k) {
            const int ch = ((k * 2 + (lane >> 5)) ^ (lane & 7)) * 8;          // (row & 7) == (lane & 7)
            f16x8 fp[W], fq[W];
#pragma unroll
            for (int x = 0; x < W; ++x) { fp[x] = *(const f16x8*)(lp + x * 32 * BK + ch); fq[x] = *(const f16x8*)(lq + x * 32 * BK + ch); }
#pragma unroll
            for (int x = 0; x < W; ++x)
#pragma unroll
                for (int y = 0; y < W; ++y) acc[x][y] = mfma(fp[x], fq[y], acc[x][y]);
        }
        if (s + 1 < stages) stash((s + 1) & 1);
        __syncthreads();
    }
    // a lane holds, of each 32 x 32, column lane & 31 and rows 8 g + 4 (lane >> 5) + 0..3 for g = 0..3
#pragma unroll
    for (int x = 0; x < W; ++x)
#pragma unroll
        for (int y = 0; y < W; ++y) {
            const int64_t j = j0 + wj * (BT / 2) + y * 32 + (lane & 31);
#pragma unroll
            for (int gq4 = 0; gq4 < 4; ++gq4) {
                const int64_t i = i0 + wi * (BT / 2) + x * 32 + gq4 * 8 + (lane >> 5) * 4;
                float v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = acc[x][y][gq4 * 4 + r];
                if constexpr (EPI == GRAM || EPI == POLY) {
                    const int64_t at = b * q.mp * q.mp + j * q.mp + i;            // (j, i .. i + 3): the mirror image, four neighbours
                    f16x4 hi, lo;
                    if constexpr (EPI == GRAM) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) v[r] *= SA / (SX * SX);
                    } else {
                        const f16x4 ah = *(const f16x4*)(q.a[0] + at);
                        f16x4 al = {};
                        if constexpr (SPLIT) al = *(const f16x4*)(q.a[1] + at);
#pragma unroll
                        for (int r = 0; r < 4; ++r) v[r] = g.c1 * ((float)ah[r] + (float)al[r]) + g.c2 * (v[r] * (1.f / SA));
                    }
                    f16* const* dst = EPI == GRAM ? q.a : q.b;
#pragma unroll
                    for (int r = 0; r < 4; ++r) { f16 h, l = 0; terms<SPLIT>(v[r], h, l); hi[r] = h; lo[r] = l; }
                    *(f16x4*)(dst[0] + at) = hi;
                    if constexpr (SPLIT) *(f16x4*)(dst[1] + at) = lo;
                    if (bi != bj) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int64_t d = b * q.mp * q.mp + (i + r) * q.mp + j;
                            dst[0][d] = hi[r];
                            if constexpr (SPLIT) dst[1][d] = lo[r];
                        }
                    }
                } else {
                    const int64_t att = (b * q.np + j) * q.mp + i;
                    f32x4 old;
                    if (g.rounded) {
                        const f16x4 xh = *(const f16x4*)(q.xt[from][0] + att);
#pragma unroll
                        for (int r = 0; r < 4; ++r) old[r] = (float)xh[r];
                    } else old = *(const f32x4*)(q.master + att);
#pragma unroll
                    for (int r = 0; r < 4; ++r) v[r] = g.c0 * old[r] + v[r] * (1.f / SA);
                    if constexpr (EPI == APPLY) {
                        f16x4 hi, lo;
#pragma unroll
                        for (int r = 0; r < 4; ++r) { f16 h, l = 0; terms<SPLIT>(v[r], h, l); hi[r] = h; lo[r] = l; }
                        *(f16x4*)(q.xt[to][0] + att) = hi;
                        if constexpr (SPLIT) *(f16x4*)(q.xt[to][1] + att) = lo;
                        if (g.keep) { f32x4 o; for (int r = 0; r < 4; ++r) o[r] = v[r]; *(f32x4*)(q.master + att) = o; }
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int64_t d = (b * q.mp + i + r) * q.np + j;
                            q.x[0][d] = hi[r];
                            if constexpr (SPLIT) q.x[1][d] = lo[r];
                        }
                    } else {
                        if (j < q.n) {
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                if (i + r < q.m) io.out[b * io.o_b + (q.flip ? j * io.o_r + i + r : (i + r) * io.o_r + j)] = (T)(v[r] * (io.scale * (1.f / SX)));
                        }
                    }
                }
            }
        }
}

}  // namespace orth
