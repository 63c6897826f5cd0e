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
constexpr int BK = 32;                        // depth of a stage: a row of it is 64 bytes, four 16-byte chunks
constexpr int PADDED = 128;                   // sides are padded with zeros to multiples of this (the smaller tile), so the products have no edges

struct Mat {                                  // one batch of matrices and the workspace it is computed in
    int64_t m, n, mp, np;                     // m <= n; padded
    int64_t batch;
    bool flip;                                // X is the transpose of the caller's matrix
    f16 *x[2], *xt[2][2], *a[2], *b[2];       // [term]: x [batch][mp][np]; xt[buffer][term] [batch][np][mp]; a, b [batch][mp][mp]
    float* master;                            // 2^13 X in F32, transposed [batch][np][mp]
    double* partial;                          // [batch][nblocks]
    int nblocks;
};
constexpr int NORM_BLOCKS = 1024;             // at most; Mat::nblocks of them

constexpr int MOST_STEPS = 64;
struct Coefficients { float c[3 * MOST_STEPS]; };

// ---- gradient, momentum, norm -------------------------------------------------------------------------------------------------------------------------------------------
template <class T> struct Io {
    const T* grad; float* mom; T* out;
    int64_t rows, cols, g_b, g_r, m_b, m_r, o_b, o_r;
    float beta, scale;
    int nesterov;
    bool vec;                                 // rows of out start on multiples of four elements
};
template <class T> __device__ inline float moved(const Io<T>& io, int64_t b, int64_t r, int64_t c, bool update) {
    const float g = (float)io.grad[b * io.g_b + r * io.g_r + c];
    if (!io.mom) return g;
    float* mp = io.mom + b * io.m_b + r * io.m_r + c;
    float m = *mp;
    if (update) { m = io.beta * m + g; *mp = m; }
    return io.nesterov ? g + io.beta * m : m;
}

template <int WAVES> __device__ inline double block_sum(double v) {       // fixed order
    __shared__ double s[WAVES];
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    double t = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) t += s[w];
    return t;
}

// Momentum and the partial sums of |u|^2.  A workgroup takes stretches of NORM_SPAN neighbouring elements (host side: matrices without gaps count as one row), 8 a thread with one
// request where rows start on 16 bytes.  Reads 2 or 4 + 4 bytes an element, writes 4: memory-bound (4096 x 4096 bf16 with momentum: 31 us, 5.4 TB/s, part of it from the last-level cache).
constexpr int NORM_SPAN = 2048;
template <class T> __global__ void __launch_bounds__(256) k_norm(const Io<T> io, int64_t rows, int64_t cols, bool vec, double* partial) {
    const int64_t b = blockIdx.y;
    const uint32_t per = (uint32_t)((cols + NORM_SPAN - 1) / NORM_SPAN);
    const int64_t spans = rows * per;
    double s = 0;
    for (int64_t i = blockIdx.x; i < spans; i += gridDim.x) {
        const int64_t r = spans >> 31 ? i / per : (uint32_t)i / per, c0 = (i - r * per) * NORM_SPAN;
        if (vec) {
            const int64_t c = c0 + threadIdx.x * 8;
            if (c < cols) {                                   // cols is a multiple of 8
                T g[8];
                float m[8];
                const T* gp = io.grad + b * io.g_b + r * io.g_r + c;
#pragma unroll
                for (int v = 0; v < 8; v += 16 / (int)sizeof(T)) *(f32x4*)(g + v) = *(const f32x4*)(gp + v);
                float* mp = io.mom + b * io.m_b + r * io.m_r + c;
                if (io.mom) {
                    *(f32x4*)m = *(const f32x4*)mp; *(f32x4*)(m + 4) = *(const f32x4*)(mp + 4);
#pragma unroll
                    for (int v = 0; v < 8; ++v) m[v] = io.beta * m[v] + (float)g[v];
                    *(f32x4*)mp = *(f32x4*)m; *(f32x4*)(mp + 4) = *(f32x4*)(m + 4);
                }
#pragma unroll
                for (int v = 0; v < 8; ++v) { const float u = !io.mom ? (float)g[v] : io.nesterov ? (float)g[v] + io.beta * m[v] : m[v]; s += (double)u * (double)u; }
            }
        } else {
            for (int64_t c = c0 + threadIdx.x; c < cols && c < c0 + NORM_SPAN; c += 256) { const float u = moved(io, b, r, c, true); s += (double)u * (double)u; }
        }
    }
    s = block_sum<4>(s);
    if (threadIdx.x == 0) partial[b * gridDim.x + blockIdx.x] = s;
}

template <bool SPLIT> __device__ inline void terms(float v, f16& hi, f16& lo) { hi = (f16)v; if constexpr (SPLIT) lo = (f16)(v - (float)hi); }

// X = u / (|u| + 1e-7) in both orders, padding included.  A workgroup takes a 64 x 64 piece through LDS: reads 2 or 4 bytes of gradient and momentum an element, writes 2 + 2 (two-term: 4 + 4)
// and the 4 of the FP32 copy; memory-bound where there are many pieces (4096 x 4096 bf16 with momentum, 14 B an element: 50 us, 4.7 TB/s), one piece's latency where there are few.  Hence
// four waves, or 16 up to four pieces a CU: 48 pieces of 333 x 500 7.6 us (four waves: 12.2), 1024 pieces of 16 x 256 x 1024 18.1 (19.5), but 4096 pieces 60.7 (49.6).
template <class T, bool SPLIT, int WAVES> __global__ void __launch_bounds__(WAVES * 64) k_start(const Io<T> io, const Mat q) {
    __shared__ float tile[64][65];
    const int64_t b = blockIdx.z, i0 = (int64_t)blockIdx.y * 64, j0 = (int64_t)blockIdx.x * 64;      // rows and columns of X
    double s = 0;
    for (int i = threadIdx.x; i < q.nblocks; i += WAVES * 64) s += q.partial[b * q.nblocks + i];
    s = block_sum<WAVES>(s);
    const double inv = (double)SX / (sqrt(s) + 1e-7);
    const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
    for (int r = w; r < 64; r += WAVES) {                     // lanes run along the caller's rows
        const int64_t i = q.flip ? i0 + l : i0 + r, j = q.flip ? j0 + r : j0 + l;
        float v = 0.f;
        if (i < q.m && j < q.n) v = (float)((double)(q.flip ? moved(io, b, j, i, false) : moved(io, b, i, j, false)) * inv);
        tile[q.flip ? l : r][q.flip ? r : l] = v;
    }
    __syncthreads();
    for (int r = w; r < 64; r += WAVES) {
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
// accumulators.  Stages of BK go from memory straight into one of four LDS buffers (no registers on the way), three stages ahead of the one that is multiplied.  Four distinct arrays, and
// the stage loop unrolled by four: the compiler then knows that a read of one buffer need not wait for the requests that fill another.
//
// A request of a wave fills 1 KB of LDS in lane order: 16 rows of 64 bytes, four 16-byte chunks each.  Chunk c of row r lies at c ^ (r / 4 & 3): the lanes FETCH in that order, and the
// sixteen rows that a read touches together then lie in different ones of the 64 banks (with r / 2 & 3 half of the LDS cycles were conflicts).
//
// In a stage the factors of its second half are read while the first half is multiplied, and those of the next stage's first half while the second is; the one barrier stands between the
// halves: behind it the next stage has arrived in every wave's part, and no wave still reads this stage's buffer, which stage s + 4 is requested into.
//
// Measured, 4096 x 4096, one term: X X' and the polynomial of A, half their tiles each, 92 and 96 us (745 and 715 TFLOP/s of the half), B X with X out in three forms 156-164 us (840-880).  The
// matrix cores are busy 41-49 % of that time (31 % of B X and 21 % of X X' at 2048 x 8192); a library product of 4096 keeps them busy 72 % of 99 us at the same 1.8-1.9 GHz, so it is not the
// clock: one workgroup a CU leaves them idle during its first stages and its epilogue, and B X stores 8 bytes an element there.  Small sides: a launch of 4-9 us each, most of it the latency of the first stages and of the
// epilogue (two groups of four waves that share a tile and halve K were 10 % slower at every size).
enum { GRAM = 0, POLY = 1, APPLY = 2, LAST = 3, PARTS = 4, JOIN = 5 };        // PARTS, JOIN: GRAM in two launches, parts of K and their sum (in the order of the parts)

struct Product {
    const f16 *P[2], *Q[2];                   // terms
    int64_t sP, sQ;                           // matrix strides
    int64_t K, M, N;                          // padded: P [M][K], Q [N][K]
    int tiles, parts;                         // PARTS, JOIN: tiles of a matrix, parts of K
    float c0, c1, c2;
    bool rounded;                             // APPLY, LAST: X in c0 X is the rounded one
    bool keep;                                // APPLY: the next step needs the F32 X
};

__device__ inline f32x16 mfma(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// Four neighbouring lanes hold four 16-bit values each, lane q those of column q; afterwards lane q holds row q.  Two exchanges of halves, with the lane two and then one apart.
__device__ inline uint64_t across(uint64_t v, int quad) {
    const uint32_t a = (uint32_t)v, b = (uint32_t)(v >> 32);                        // rows 0 1, rows 2 3
    const uint32_t give = quad < 2 ? b : a, keep = quad < 2 ? a : b;
    const uint32_t got = (uint32_t)__builtin_amdgcn_mov_dpp((int)give, 0x4e, 0xf, 0xf, true);      // quad_perm 2 3 0 1
    const uint32_t c0 = quad < 2 ? keep : got, c1 = quad < 2 ? got : keep;          // this lane's two rows: columns (quad & 1), (quad & 1) + 2
    const uint32_t d0 = (uint32_t)__builtin_amdgcn_mov_dpp((int)c0, 0xb1, 0xf, 0xf, true), d1 = (uint32_t)__builtin_amdgcn_mov_dpp((int)c1, 0xb1, 0xf, 0xf, true);
    const uint32_t lo0 = quad & 1 ? (d0 >> 16) | (c0 & 0xffff0000u) : (c0 & 0xffffu) | (d0 << 16);
    const uint32_t lo1 = quad & 1 ? (d1 >> 16) | (c1 & 0xffff0000u) : (c1 & 0xffffu) | (d1 << 16);
    return (uint64_t)lo1 << 32 | lo0;
}

// SLOTS: slices of a stage and factor — the two terms of a split factor, whose three products then share what is read; or two neighbouring slices of K, which halves the number of stages
// where the tile is so small that each stage costs the latency of memory; or one.
template <class T, int BT, int EPI, bool SPLIT, int SLOTS>
__global__ void __launch_bounds__(256, BT == 64 || (BT == 128 && SLOTS == 1) ? 2 : 1) k_product(const Product g, const Mat q, const Io<T> io, const int from, const int to) {
    constexpr int W = BT / 64;                // 32 x 32 accumulators a wave and direction
    constexpr int RQ = BT / 64;               // requests of a wave, factor and stage
    constexpr int SLICE = BT * BK, BUF = 2 * SLOTS * SLICE;   // P's slices, then Q's
    static_assert(!SPLIT || SLOTS == 2, "a slot for each term");
    __shared__ __align__(16) f16 s0[BUF], s1[BUF], s2[BUF], s3[BUF];
    const int64_t b = blockIdx.z;
    int bi, bj;
    constexpr bool LOWER = EPI != APPLY && EPI != LAST;
    int tile = (int)blockIdx.x, part = 0;
    if constexpr (EPI == PARTS) { tile = (int)(blockIdx.x % (uint32_t)g.tiles); part = (int)(blockIdx.x / (uint32_t)g.tiles); }
    if constexpr (LOWER) {                                    // tile t of the lower triangle
        const int t = tile;
        bi = (int)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
        while ((bi + 1) * (bi + 2) / 2 <= t) ++bi;
        while (bi * (bi + 1) / 2 > t) --bi;
        bj = t - bi * (bi + 1) / 2;
    } else {
        // workgroups go round the eight XCDs: each gets a compact part of the tiles (2 x 4 parts), so that its L2 serves its factors' rows to all of them
        const int ti = (int)((g.M + BT - 1) / BT), tj = (int)((g.N + BT - 1) / BT), t = tile;
        if (ti % 2 == 0 && tj % 4 == 0) {
            const int x = t & 7, u = t >> 3, wj4 = tj / 4;
            bi = (x >> 2) * (ti / 2) + u / wj4; bj = (x & 3) * wj4 + u % wj4;
        } else { bi = t / tj; bj = t % tj; }
    }
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, wi = wave >> 1, wj = wave & 1;
    const int64_t i0 = (int64_t)bi * BT, j0 = (int64_t)bj * BT;
    f32x16 acc[W][W];
#pragma unroll
    for (int x = 0; x < W; ++x)
#pragma unroll
        for (int y = 0; y < W; ++y)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[x][y][r] = 0.f;
    // sums of part p of a tile, F32: an accumulator's registers four at a time, lanes next to each other
    f32x4* const parts = (f32x4*)(q.xt[to][0] + b * q.np * q.mp) + (int64_t)tile * (W * W * 1024) + wave * 256 + lane;
    const int64_t part_step = (int64_t)g.tiles * (W * W * 1024);
    if constexpr (EPI == JOIN) {
        for (int p = 0; p < g.parts; ++p)
#pragma unroll
            for (int x = 0; x < W; ++x)
#pragma unroll
                for (int y = 0; y < W; ++y)
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        const f32x4 v = parts[p * part_step + (x * W + y) * 1024 + h * 64];
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[x][y][h * 4 + r] += v[r];
                    }
    } else {
        const int64_t nk = g.K / PADDED, k0 = EPI == PARTS ? nk * part / g.parts * PADDED : 0, k1 = EPI == PARTS ? nk * (part + 1) / g.parts * PADDED : g.K;
        constexpr int DEPTH = SPLIT ? BK : SLOTS * BK;            // of a stage, in k
        const int stages = (int)((k1 - k0) / DEPTH);              // a multiple of four, or of two
        // rows past the last one (the sides are multiples of 128, not of every BT) are requested from the last one, multiplied and not stored
        int64_t row_p[RQ], row_q[RQ];
#pragma unroll
        for (int c = 0; c < RQ; ++c) {
            const int64_t r = (wave * RQ + c) * 16 + (lane >> 2), k = k0 + ((lane & 3) ^ ((lane >> 4) & 3)) * 8;
            row_p[c] = (i0 + r < g.M ? i0 + r : g.M - 1) * g.K + k;
            row_q[c] = (j0 + r < g.N ? j0 + r : g.N - 1) * g.K + k;
        }
        // request n of the 2 SLOTS RQ of a stage; behind the last stage the last one once more, into a buffer that is not read again: the counts stay the same
        constexpr int NREQ = 2 * SLOTS * RQ;
        auto request = [&](int s, f16* buf, int n) {
            s = s < stages ? s : stages - 1;
            const int slice = n / RQ, c = n % RQ, slot = slice % SLOTS, term = SPLIT ? slot : 0;
            const int k = s * DEPTH + (SPLIT ? 0 : slot * BK);
            const f16* from = slice < SLOTS ? g.P[term] + b * g.sP + k + row_p[c] : g.Q[term] + b * g.sQ + k + row_q[c];
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                             (__attribute__((address_space(3))) void*)(buf + slice * SLICE + (wave * RQ + c) * 512), 16, 0, 0);
        };
        const int rp = (wi * (BT / 2) + (lane & 31)) * BK, rq = SLOTS * SLICE + (wj * (BT / 2) + (lane & 31)) * BK;
        const int ch0 = ((lane >> 5) ^ ((lane >> 2) & 3)) * 8, ch1 = ((2 + (lane >> 5)) ^ ((lane >> 2) & 3)) * 8;
        typedef f16x8 Factors[SLOTS][2][W];                       // [slot][P, Q]
        constexpr int NREAD = 2 * SLOTS * W;
        Factors f0, f1;
        auto read = [&](const f16* buf, int ch, Factors& f, int n) {
            const int slot = n / (2 * W), which = n / W % 2, x = n % W;
            f[slot][which][x] = *(const f16x8*)(buf + slot * SLICE + (which ? rq : rp) + x * 32 * BK + ch);
        };
        // half a stage: the products of one half with the reads of the next and half a stage's requests between them, one at a time — issued in a burst they hold the wave, and with it the
        // matrix core, up to the rate of the request queue and of LDS
        constexpr int SETS = SPLIT ? 3 : SLOTS, NM = SETS * W * W;
        auto half = [&](const Factors& f, const f16* rbuf, int ch, Factors& nf, int rs, f16* qbuf, int n0) {
            int reads = 0, requests = 0;
#pragma unroll
            for (int m = 0; m < NM; ++m) {
                const int set = m / (W * W), x = m / W % W, y = m % W;
                const int tp = SPLIT ? set == 1 : set, tq = SPLIT ? set == 0 : set;    // split: hi lo, lo hi, hi hi
                acc[x][y] = mfma(f[tp][0][x], f[tq][1][y], acc[x][y]);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (; reads < NREAD && reads * 2 * NM < (m + 1) * NREAD * 3; ++reads) read(rbuf, ch, nf, reads);     // all within the first two thirds
#pragma unroll
                for (; requests < NREQ / 2 && (requests + 1) * NM <= (m + 1) * (NREQ / 2); ++requests) request(rs, qbuf, n0 + requests);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        // the oldest stage in flight has arrived in this wave's part (those of two later ones may still be on the way) and its LDS reads are done; then in all waves
        auto arrive = [&]() {
            static_assert(NREQ == 4 || NREQ == 6 || NREQ == 8, "the counts below");
            __builtin_amdgcn_s_waitcnt(NREQ == 8 ? 0x4070 : NREQ == 6 ? 0x007c : 0x0078);        // vmcnt(2 NREQ) lgkmcnt(0)
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_sched_barrier(0);
        };
        // behind the barrier no wave reads `now` any more: its next stage is requested half there, half in the first half of the next stage
        auto stage = [&](int s, f16* prev, f16* now, const f16* next) {
            half(f0, now, ch1, f1, s + 3, prev, NREQ / 2);
            arrive();
            half(f1, next, ch0, f0, s + 4, now, 0);
        };
        auto all = [&](int s, f16* buf, int from, int to) {
#pragma unroll
            for (int n = from; n < to; ++n) request(s, buf, n);
        };
        all(0, s0, 0, NREQ); all(1, s1, 0, NREQ); all(2, s2, 0, NREQ);
        __builtin_amdgcn_sched_barrier(0);
        arrive();
        all(3, s3, 0, NREQ / 2);
#pragma unroll
        for (int n = 0; n < NREAD; ++n) read(s0, ch0, f0, n);
        int s = 0;
        for (; s + 4 <= stages; s += 4) {
            stage(s, s3, s0, s1);
            stage(s + 1, s0, s1, s2);
            stage(s + 2, s1, s2, s3);
            stage(s + 3, s2, s3, s0);
        }
        if constexpr (SLOTS == 2 && !SPLIT)                       // K is a multiple of 128: two stages of 64 may be left
            if (s < stages) {
                stage(s, s3, s0, s1);
                stage(s + 1, s0, s1, s2);
            }
        __builtin_amdgcn_s_waitcnt(0x0070);                       // nothing is on the way to LDS when the workgroup ends
    }
    if constexpr (EPI == PARTS) {
#pragma unroll
        for (int x = 0; x < W; ++x)
#pragma unroll
            for (int y = 0; y < W; ++y)
#pragma unroll
                for (int h = 0; h < 4; ++h)
                    parts[part * part_step + (x * W + y) * 1024 + h * 64] = f32x4{acc[x][y][h * 4], acc[x][y][h * 4 + 1], acc[x][y][h * 4 + 2], acc[x][y][h * 4 + 3]};
        return;
    }
    // A lane holds, of each 32 x 32, column lane & 31 and rows 8 g + 4 (lane >> 5) + 0..3 for g = 0..3: four neighbours of the transposed order.  For the other order four lanes
    // exchange theirs, so that both are stored eight bytes at a time.  What a row of accumulators needs from memory is requested before any of it is used.
    const int64_t jw = j0 + wj * (BT / 2) + (lane & 31), iw = i0 + wi * (BT / 2) + (lane >> 5) * 4;
    const int quad = lane & 3;
    int64_t jc[W];                                            // columns that are read: inside
#pragma unroll
    for (int y = 0; y < W; ++y) jc[y] = jw + y * 32 < g.N ? jw + y * 32 : jw < g.N ? jw : 0;
#pragma unroll
    for (int x = 0; x < W; ++x) {
        if (i0 + wi * (BT / 2) + x * 32 >= g.M) continue;     // the same for all lanes
        f32x4 old[W][4];
        if constexpr (EPI == POLY) {
            f16x4 ah[W][4], al[W][4];
#pragma unroll
            for (int y = 0; y < W; ++y)
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    const int64_t at = b * q.mp * q.mp + jc[y] * q.mp + iw + x * 32 + h * 8;
                    ah[y][h] = *(const f16x4*)(q.a[0] + at);
                    if constexpr (SPLIT) al[y][h] = *(const f16x4*)(q.a[1] + at);
                }
#pragma unroll
            for (int y = 0; y < W; ++y)
#pragma unroll
                for (int h = 0; h < 4; ++h)
#pragma unroll
                    for (int r = 0; r < 4; ++r) old[y][h][r] = SPLIT ? (float)ah[y][h][r] + (float)al[y][h][r] : (float)ah[y][h][r];
        } else if constexpr (EPI == APPLY || EPI == LAST) {
            if (!SPLIT && g.rounded) {
                f16x4 xh[W][4];
#pragma unroll
                for (int y = 0; y < W; ++y)
#pragma unroll
                    for (int h = 0; h < 4; ++h) xh[y][h] = *(const f16x4*)(q.xt[from][0] + (b * q.np + jc[y]) * q.mp + iw + x * 32 + h * 8);
#pragma unroll
                for (int y = 0; y < W; ++y)
#pragma unroll
                    for (int h = 0; h < 4; ++h)
#pragma unroll
                        for (int r = 0; r < 4; ++r) old[y][h][r] = (float)xh[y][h][r];
            } else {
#pragma unroll
                for (int y = 0; y < W; ++y)
#pragma unroll
                    for (int h = 0; h < 4; ++h) old[y][h] = *(const f32x4*)(q.master + (b * q.np + jc[y]) * q.mp + iw + x * 32 + h * 8);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int y = 0; y < W; ++y) {
            if (j0 + wj * (BT / 2) + y * 32 >= g.N) continue;
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                const int64_t i = iw + x * 32 + h * 8, j = jw + y * 32;            // rows i .. i + 3 of column j
                f32x4 v;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    v[r] = acc[x][y][h * 4 + r];
                    if constexpr (EPI == GRAM || EPI == JOIN) v[r] *= SA / (SX * SX);
                    else if constexpr (EPI == POLY) v[r] = g.c1 * old[y][h][r] + g.c2 * (v[r] * (1.f / SA));
                    else v[r] = g.c0 * old[y][h][r] + v[r] * (1.f / SA);
                }
                if constexpr (EPI == LAST) {
                    const float f = io.scale * (1.f / SX);
                    T o[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[r] = (T)(v[r] * f);
                    if (q.flip) {
                        if (j < q.n) {
                            T* dst = io.out + b * io.o_b + j * io.o_r + i;
                            if (io.vec && i + 4 <= q.m) {
                                if constexpr (sizeof(T) == 2) *(uint64_t*)dst = __builtin_bit_cast(uint64_t, *(f16x4*)o); else *(f32x4*)dst = *(f32x4*)o;
                            } else {
#pragma unroll
                                for (int r = 0; r < 4; ++r) if (i + r < q.m) dst[r] = o[r];
                            }
                        }
                    } else {
                        if constexpr (sizeof(T) == 2) {
                            const uint64_t row = across(__builtin_bit_cast(uint64_t, *(f16x4*)o), quad);
                            const int64_t jq = j - quad;
                            if (i + quad < q.m) {
                                T* dst = io.out + b * io.o_b + (i + quad) * io.o_r + jq;
                                if (io.vec && jq + 4 <= q.n) *(uint64_t*)dst = row;
                                else {
#pragma unroll
                                    for (int r = 0; r < 4; ++r) if (jq + r < q.n) ((uint16_t*)dst)[r] = (uint16_t)(row >> (16 * r));
                                }
                            }
                        } else if (j < q.n) {
#pragma unroll
                            for (int r = 0; r < 4; ++r) if (i + r < q.m) io.out[b * io.o_b + (i + r) * io.o_r + j] = o[r];
                        }
                    }
                } else {
                    f16x4 hi, lo;
#pragma unroll
                    for (int r = 0; r < 4; ++r) { f16 e, l = 0; terms<SPLIT>(v[r], e, l); hi[r] = e; lo[r] = l; }
                    constexpr bool SQUARE = LOWER;
                    f16* const* direct = EPI == POLY ? q.b : SQUARE ? q.a : q.x;
                    f16* const* turned = EPI == POLY ? q.b : SQUARE ? q.a : q.xt[to];
                    const int64_t att = SQUARE ? (b * q.mp + j) * q.mp + i : (b * q.np + j) * q.mp + i;
                    const int64_t atd = SQUARE ? (b * q.mp + i + quad) * q.mp + j - quad : (b * q.mp + i + quad) * q.np + j - quad;
                    *(f16x4*)(turned[0] + att) = hi;
                    if constexpr (SPLIT) *(f16x4*)(turned[1] + att) = lo;
                    if constexpr (EPI == APPLY) { if (g.keep) *(f32x4*)(q.master + att) = v; }
                    if (!SQUARE || bi != bj) {
                        *(uint64_t*)(direct[0] + atd) = across(__builtin_bit_cast(uint64_t, hi), quad);
                        if constexpr (SPLIT) *(uint64_t*)(direct[1] + atd) = across(__builtin_bit_cast(uint64_t, lo), quad);
                    }
                }
            }
        }
    }
}

// ---- small matrices ---------------------------------------------------------------------------------------------------------------------------------------------------
// Both sides at most 128: one workgroup does a matrix in one launch (17 otherwise: 48.6 us against 205 at 128 x 128).  X, A and B live in LDS as two F16 terms and 32 x 32 pieces of X
// stay in the F32 registers of the waves that own them.  X is needed by rows for X X' and by columns for B X, never at once, and A, B never next to X by rows: two regions, 128 KB at
// a side of 128.  Symmetric matrices are stored transposed, which is their own order, four neighbours at a time.
template <class T, int S> __global__ void __launch_bounds__((S / 32) * (S / 32) * 64) k_small(const Io<T> io, const int64_t m, const int64_t n, const bool flip, const int steps, const Coefficients co) {
    constexpr int WS = S / 32, NWAVE = WS * WS, CHUNKS = S / 8;
    __shared__ __align__(16) f16 x[2][S * S], a[2][S * S];
    __shared__ double part[NWAVE];
    const int64_t b = blockIdx.x;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, wi = wave / WS, wj = wave % WS, quad = lane & 3;
    const int j = wj * 32 + (lane & 31), i0 = wi * 32 + (lane >> 5) * 4;            // this lane's elements: rows i0 + 8 h + r of column j
    // place of the 16-byte chunk c of a row
    auto at = [](int row, int c) { return row * S + ((c ^ (S == 128 ? row & 15 : S == 64 ? row >> 1 & 7 : row >> 2 & 3)) * 8); };
    float v[4][4];
    double sum = 0;
#pragma unroll
    for (int h = 0; h < 4; ++h)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = i0 + 8 * h + r;
            v[h][r] = i < m && j < n ? (flip ? moved(io, b, j, i, true) : moved(io, b, i, j, true)) : 0.f;
            sum += (double)v[h][r] * (double)v[h][r];
        }
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    if (lane == 0) part[wave] = sum;
    __syncthreads();
    sum = 0;
    for (int w = 0; w < NWAVE; ++w) sum += part[w];
    const double inv = (double)SX / (sqrt(sum) + 1e-7);
#pragma unroll
    for (int h = 0; h < 4; ++h)
#pragma unroll
        for (int r = 0; r < 4; ++r) v[h][r] = (float)((double)v[h][r] * inv);
    auto split = [&](const float (&f)[4], uint64_t& hi, uint64_t& lo) {
        f16x4 eh, el;
#pragma unroll
        for (int r = 0; r < 4; ++r) { f16 p, q; terms<true>(f[r], p, q); eh[r] = p; el[r] = q; }
        hi = __builtin_bit_cast(uint64_t, eh); lo = __builtin_bit_cast(uint64_t, el);
    };
    auto put_columns = [&](f16 (&dst)[2][S * S], const float (&f)[4][4]) {          // (column j, rows i ..): by columns, or a symmetric matrix
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            uint64_t hi, lo;
            split(f[h], hi, lo);
            const int i = i0 + 8 * h, w = at(j, i >> 3) + (i & 7);
            *(uint64_t*)&dst[0][w] = hi; *(uint64_t*)&dst[1][w] = lo;
        }
    };
    auto put_rows = [&](f16 (&dst)[2][S * S], const float (&f)[4][4]) {
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            uint64_t hi, lo;
            split(f[h], hi, lo);
            const int i = i0 + 8 * h + quad, jq = j - quad, w = at(i, jq >> 3) + (jq & 7);
            *(uint64_t*)&dst[0][w] = across(hi, quad); *(uint64_t*)&dst[1][w] = across(lo, quad);
        }
    };
    auto product = [&](const f16 (&P)[2][S * S], const f16 (&Q)[2][S * S]) {        // rows 32 wi .. of P times rows 32 wj .. of Q
        f32x16 acc;
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[r] = 0.f;
        const int rp = wi * 32 + (lane & 31), rq = wj * 32 + (lane & 31);
#pragma unroll 2
        for (int c = 0; c < CHUNKS; c += 2) {
            const int k = c + (lane >> 5);
            const f16x8 ph = *(const f16x8*)&P[0][at(rp, k)], pl = *(const f16x8*)&P[1][at(rp, k)], qh = *(const f16x8*)&Q[0][at(rq, k)], ql = *(const f16x8*)&Q[1][at(rq, k)];
            acc = mfma(ph, ql, acc); acc = mfma(pl, qh, acc); acc = mfma(ph, qh, acc);
        }
        return acc;
    };
    put_rows(x, v);
    for (int s = 0; s < steps; ++s) {
        const float c0 = co.c[3 * s], c1 = co.c[3 * s + 1], c2 = co.c[3 * s + 2];
        float g[4][4];
        __syncthreads();
        f32x16 acc = product(x, x);
#pragma unroll
        for (int e = 0; e < 16; ++e) g[e >> 2][e & 3] = acc[e] * (SA / (SX * SX));
        put_columns(a, g);
        __syncthreads();
        acc = product(a, a);
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 16; ++e) g[e >> 2][e & 3] = c1 * g[e >> 2][e & 3] + c2 * (acc[e] * (1.f / SA));
        put_columns(a, g);
        put_columns(x, v);
        __syncthreads();
        acc = product(a, x);
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e >> 2][e & 3] = c0 * v[e >> 2][e & 3] + acc[e] * (1.f / SA);
        if (s + 1 < steps) { __syncthreads(); put_rows(x, v); }
    }
    const float f = io.scale * (1.f / SX);
#pragma unroll
    for (int h = 0; h < 4; ++h)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = i0 + 8 * h + r;
            if (i < m && j < n) io.out[b * io.o_b + (flip ? (int64_t)j * io.o_r + i : (int64_t)i * io.o_r + j)] = (T)(v[h][r] * f);
        }
}

}  // namespace orth
