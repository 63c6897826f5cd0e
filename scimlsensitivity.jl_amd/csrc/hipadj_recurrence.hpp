// hipadj_recurrence.hpp — the gated linear recurrence: the exactly stepped diagonal linear system of a sequence model, its adjoint and its single step.
//
//   h_t = a_t h_{t-1} + b_t,   a = g | exp(g) | sigmoid(g),   b = x | (1 - a) x
//
// and, with the cotangents dh_t of all states and dh_T of the last one,
//
//   G_t = dh_t + R_{t+1},  R_t = a_t G_t  (R_{T+1} = dh_T),   dx_t = G_t (1 - a_t or 1),   da_t = G_t (h_{t-1} [- x_t]),   dh_0 = R_1.
//
// Both directions are scans of affine maps h -> A h + H, whose composition is associative, so the time axis can be cut:
//   * a workgroup takes a TILE of NW * TS rows (TS: TSF or TSA) by 64 * V channels; wave w holds rows [w TS, (w + 1) TS) of it in registers, every lane V neighbouring channels, so that each
//     row of a wave is one contiguous request and every input is read from memory ONCE;
//   * the NW partial maps of a tile are joined through LDS;
//   * the tiles of one (batch row, channel group) form a CHAIN.  A tile first publishes its own map (A, H); the state at its start is the state at the start of its group of
//     GS tiles carried through the maps of the group's earlier tiles, in this fixed order — the result does not depend on which tile ran first — and the last tile of a group
//     publishes the state at the next group's start.  A long axis therefore costs one exchange per GROUP on the critical path, not one per tile.
// Tiles are handed out by a ticket (one atomic increment per workgroup) in an order where a tile only ever waits for tiles with lower tickets: those already run, and the
// publication of a map waits for nothing, so every wait ends.  Published values travel in 64-bit words that also say that they are there, written and read as relaxed
// device-scope atomics: a word is complete or absent, nothing orders one word against another and no cache has to be written back.  The words are zeroed by a launch of their own.
//
// The adjoint does not read h: the forward pass leaves the state at the start of every TTA rows (the checkpoints, 1 / TTA of h in 32 bits) and a tile of the adjoint re-solves its rows from there in
// registers — the bytes of reading h back are those of reading x, and the states are the unrounded ones.
// Bound: memory, 3 streams forward and 5 in the adjoint, where the axes are long and many; the exchanges along the chain where there are few.  Measured on an MI355X (a copy: 5.10 TB/s), the
// launch of k_zero (2-6 us) not counted:
//   forward  1 x 65536 x 2048 BF16, exp gate            197 us, 4.09 TB/s        8 x 4096 x 2048 BF16, coupled sigmoid, with checkpoints  103 us, 3.95 TB/s
//            37 packed sequences, 16381 x 1024 F16       40 us, 2.5 TB/s         2 x 2047 x 777 F32                                        16 us, 2.4 TB/s
//            1 x 512 x 2048 BF16                        9.1 us: four tiles a chain, latency
//   adjoint  8 x 4096 x 2048 BF16, coupled sigmoid      185 us, 3.7 TB/s         2 x 2047 x 777 F32                                        27 us, 2.3 TB/s
// (averages of 13 calls; the vector units are busy 41 % of the time in the first of these, 55 % in the second and 74 % in the adjoint of 16-bit data).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace rec {

constexpr int NW = 8;             // waves of a workgroup = time pieces of a tile
constexpr int TSF = 16;           // rows of a piece, forward: (a, b) of 16 x V cells fit the 128 registers that leave room for two workgroups a CU
constexpr int TSA = 8;            // rows of a piece, adjoint: five values a cell, so half as many (16 spilled 47 ... 101 registers and left one workgroup a CU)
constexpr int TTF = NW * TSF, TTA = NW * TSA;                 // rows of a tile; a checkpoint every TTA rows
constexpr int NT = NW * 64;
constexpr int MOST_GS = 32;       // tiles of a group: a multiple of NW up to this

typedef __bf16 bf16;
typedef _Float16 f16;

struct Args {
    const void *x, *gate, *h0, *dh, *dh_final;
    void *h, *h_final, *dx, *dgate, *dh0, *ckpt;
    const void* offsets;                                     // [nseq + 1], offsets64: 64-bit
    int64_t x_sb, x_st, g_sb, g_st, h_sb, h_st, dh_sb, dh_st, dx_sb, dx_st, dg_sb, dg_st;
    int64_t L, D, nseq;
    int32_t offsets64, ntiles, nckpt, ncg, nchains, GS;      // nckpt: checkpoints of a batch row; ncg: channel groups; nchains = batch * ncg; GS: tiles of a group
    uint64_t *agg, *car;                                     // [nchains][ntiles][WPM][CW], [nchains][ngroups][WPV][CW]
    uint32_t* ticket;
};

template <class T, int V> struct alignas(sizeof(T) * V) Pack { T v[V]; };

// ---- values -----------------------------------------------------------------------------------------------------------------------------------------------------

// exp in 32 bits: exp2 of p = g log2(e), times 1 + (g - p ln 2), which makes up for p's rounding and the constant's: strong decays keep their digits (without it exp(-14) is off by 10 units
// of its last place).  ln 2 in one number leaves |g| 3e-9, two units at -80, which 16-bit data (FAST) do with; wider ones have it in two.  The difference is no number where p overflows, where
// exp2 is 0 or infinite: the smaller of NaN and 1 is 1.  NaN stays NaN.  NEG: g <= 0, nothing overflows upwards and the product takes one instruction less.
template <bool FAST, bool NEG> __device__ inline float exp_(float g) {
    const float p = g * 1.44269504f, r = __builtin_amdgcn_exp2f(p);
    float e = fmaf(-p, 0.693147182f, g);
    if constexpr (!FAST) e = fmaf(p, 1.90465433e-9f, e);
    e = fminf(e, 1.f);
    return NEG ? fmaf(r, e, r) : r * (1.f + e);
}
template <bool FAST, bool NEG> __device__ inline double exp_(double g) { return exp(g); }
// exp(g) and 1 - exp(g), the latter without the cancellation at small |g| (Taylor series; the first term left out is below 2e-8 of the value at 0.35, FAST: 5e-8 at 0.25)
template <bool FAST> __device__ inline void exp_rest(float g, float& a, float& rest) {
    a = exp_<FAST, false>(g);
    float s;
    s = FAST ? 1.f / 720.f : fmaf(g, 1.f / 5040.f, 1.f / 720.f);
    s = fmaf(s, g, 1.f / 120.f); s = fmaf(s, g, 1.f / 24.f); s = fmaf(s, g, 1.f / 6.f); s = fmaf(s, g, 0.5f); s = fmaf(s, g, 1.f);
    const bool near = fabsf(g) < (FAST ? 0.25f : 0.35f);
    rest = near ? -g * s : 1.f - a;
    a = near ? 1.f - rest : a;
}
template <bool FAST> __device__ inline void exp_rest(double g, double& a, double& rest) { a = exp(g); rest = -expm1(g); }
__device__ inline float recip(float x) { return __builtin_amdgcn_rcpf(x); }
__device__ inline double recip(double x) { return 1.0 / x; }
__device__ inline float neg_abs(float x) { return -fabsf(x); }
__device__ inline double neg_abs(double x) { return -fabs(x); }

// a and 1 - a of a gate; `rest` is only formed where it is used.  A decay next to one acts over hundreds of rows, so its last bit counts: where 1 - a is the smaller one it is formed
// first, with its own relative accuracy, and a as its difference from one, within half a unit of the last place.
template <int FORM, bool REST, bool FAST, class S> __device__ inline void decay(S g, S& a, S& rest) {
    if constexpr (FORM == 0) { a = g; if constexpr (REST) rest = S(1) - g; }
    else if constexpr (FORM == 1) { if constexpr (REST) exp_rest<FAST>(g, a, rest); else a = exp_<FAST, false>(g); }
    else { const S e = exp_<FAST, true>(neg_abs(g)), s = e * recip(S(1) + e), l = S(1) - s; a = g >= S(0) ? l : s; if constexpr (REST) rest = g >= S(0) ? s : l; }
}

// ---- published words ----------------------------------------------------------------------------------------------------------------------------------------------

template <class S> constexpr int WPV = sizeof(S) / 4;         // words of a value
__device__ inline void put(uint64_t* w, uint64_t v) { __hip_atomic_store(w, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ inline uint64_t get(const uint64_t* w) { return __hip_atomic_load(const_cast<uint64_t*>(w), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ inline void publish(uint64_t* w, int64_t cw, float v, uint32_t tag) { put(w, (uint64_t(tag) << 32) | __float_as_uint(v)); }
__device__ inline void publish(uint64_t* w, int64_t cw, double v, uint32_t tag) {
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    put(w, (uint64_t(tag) << 32) | (b & 0xffffffffu)); put(w + cw, (uint64_t(tag) << 32) | (b >> 32));
}
// waits for a published value; every wave that waits does so for a tile with a lower ticket (top of this file)
__device__ inline uint32_t await_value(const uint64_t* w, int64_t, float& v) {
    uint64_t q;
    while (!((q = get(w)) >> 32)) __builtin_amdgcn_s_sleep(1);
    v = __uint_as_float((uint32_t)q);
    return (uint32_t)(q >> 32);
}
__device__ inline uint32_t await_value(const uint64_t* w, int64_t cw, double& v) {
    uint64_t q, r;
    while (!((q = get(w)) >> 32)) __builtin_amdgcn_s_sleep(1);
    while (!((r = get(w + cw)) >> 32)) __builtin_amdgcn_s_sleep(1);
    v = __longlong_as_double((long long)((q & 0xffffffffu) | (r << 32)));
    return (uint32_t)(q >> 32);
}
// A map (A, H); CUT: no state passes (a sequence starts inside), H alone counts, whatever A and the state are.  In 32 bits it is one word, and every A but the payload of a NaN passes
// exactly (a held state is multiplied by the A of each tile: one that is off by a last bit would let it grow along the axis): the bits of A are inverted, so that the two patterns
// that no NaN is stored as stand for "absent" (a zeroed word) and for CUT.
constexpr uint32_t TAG_VALUE = 1, TAG_CUT = 2;
constexpr uint32_t MAP_CUT = ~0x7fffffffu;
template <class S> constexpr int WPM = sizeof(S) == 4 ? 1 : 4;         // words of a map
__device__ inline void publish_map(uint64_t* w, int64_t, float A, float H, uint32_t cut) {
    const uint32_t a = A != A ? 0x7fc00000u : __float_as_uint(A);
    put(w, (uint64_t(__float_as_uint(H)) << 32) | (cut ? MAP_CUT : ~a));
}
__device__ inline void publish_map(uint64_t* w, int64_t cw, double A, double H, uint32_t cut) { publish(w, cw, A, cut ? TAG_CUT : TAG_VALUE); publish(w + 2 * cw, cw, H, TAG_VALUE); }
// `seen`: the first look at the word, taken earlier so that several are on their way together (64 bits: none)
__device__ inline uint32_t await_map(const uint64_t* w, int64_t, uint64_t seen, float& A, float& H) {
    uint64_t q = seen;
    while (!(uint32_t)q) { __builtin_amdgcn_s_sleep(1); q = get(w); }
    A = __uint_as_float(~(uint32_t)q); H = __uint_as_float((uint32_t)(q >> 32));
    return (uint32_t)q == MAP_CUT;
}
__device__ inline uint32_t await_map(const uint64_t* w, int64_t cw, uint64_t, double& A, double& H) {
    const uint32_t q = await_value(w, cw, A);
    await_value(w + 2 * cw, cw, H);
    return q == TAG_CUT;
}

// ---- packed sequences ---------------------------------------------------------------------------------------------------------------------------------------------

struct Offset { uint32_t lo, hi; };                           // as it arrives (32 bits: twice the same word), so that nothing waits where it is requested
__device__ inline Offset request_offset(const Args& p, int64_t i) {
    const uint32_t* w = (const uint32_t*)p.offsets + (i << p.offsets64);
    return {w[0], w[p.offsets64]};
}
__device__ inline int64_t value_of(const Args& p, Offset o) { return p.offsets64 ? (int64_t)((uint64_t)o.hi << 32 | o.lo) : (int64_t)(int32_t)o.lo; }
__device__ inline int64_t offset_at(const Args& p, int64_t i) { return value_of(p, request_offset(p, i)); }

// The first sequence that ends behind row t (nseq: none) is among lo ... lo + 63: a 64-ary search over the ends.  Offsets that do not ascend give some number in [0, nseq].
__device__ inline int64_t narrow(const Args& p, int64_t t) {
    int64_t lo = 0, n = p.nseq;                               // it is in [lo, lo + n]
    const int lane = threadIdx.x & 63;
    while (n > 63) {
        const int64_t step = (n + 63) / 64;
        const int64_t i = lo + lane * step;
        const bool in = lane * step < n;
        const int64_t last = i + step - 1 < lo + n ? i + step - 1 : lo + n - 1;
        const bool before = in && offset_at(p, last + 1) <= t;                      // the whole stretch ends at t or earlier
        const int k = __popcll(__ballot(before));
        const int64_t at = (int64_t)k * step;
        if (at >= n) return lo + n;
        lo += at;
        n = (step < n - at ? step : n - at) - 1;                                    // its last one ends behind t
    }
    return lo;
}
__device__ inline int64_t of_lane(int64_t v, int lane) {
    return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)v, lane) | (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32);
}

struct Marks { uint32_t start, end, out; };                   // bits of a piece's rows: first of a sequence, last of one, of none
// The bounds of 64 neighbouring sequences, one a lane, among them the first that ends behind row t: one exchange with memory for up to 63 sequences.  Requested BEFORE the rows: requests
// return in order, and behind the rows' they would keep the arithmetic waiting for the last row (1 x 16384 x 1024 F16, one sequence: 44 us instead of 40).
struct Window { int64_t lo; Offset start, end; bool in; };
__device__ inline Window window_of(const Args& p, int64_t t) {
    Window w{};
    w.lo = narrow(p, t);
    const int64_t s = w.lo + (threadIdx.x & 63);
    w.in = s < p.nseq;
    const int64_t i = w.in ? s : p.nseq - 1;
    w.start = request_offset(p, i); w.end = request_offset(p, i + 1);
    return w;
}
// seq[i]: the sequence that row i, first or last of it, belongs to; in LDS, where the few rows that need it find it without a search (a search at each of those places made the adjoint of 37
// sequences of 16384 x 1024 F16 take 78-96 us instead of 64)
template <int TS> __device__ inline Marks marks_of(const Args& p, int64_t t0, Window w, int64_t (&seq)[TS]) {
    Marks m{0, 0, (1u << TS) - 1};
    int64_t pos = t0, start = value_of(p, w.start), end = value_of(p, w.end);
    while (pos < t0 + TS && pos < p.L) {                      // pos advances in every turn, whatever the offsets hold
        int k = __popcll(__ballot(w.in && end <= pos));
        if (k == 64) {
            w = window_of(p, pos);
            start = value_of(p, w.start); end = value_of(p, w.end);
            k = __popcll(__ballot(w.in && end <= pos));
        }
        if (k == 64 || w.lo + k >= p.nseq) break;
        const int64_t st = of_lane(start, k), en = of_lane(end, k);
        const int64_t from = st > pos ? st : pos, to = en < t0 + TS ? en : t0 + TS;
        if (from < to) m.out &= ~((1u << (int)(to - t0)) - (1u << (int)(from - t0)));      // bits from - t0 ... to - t0 - 1; both at most TS <= 16
        if (st >= t0 && st < to) { m.start |= 1u << (int)(st - t0); seq[(int)(st - t0)] = w.lo + k; }
        if (en - 1 >= from && en - 1 < t0 + TS) { m.end |= 1u << (int)(en - 1 - t0); seq[(int)(en - 1 - t0)] = w.lo + k; }
        pos = en > pos ? en : pos + 1;
    }
    const int inside = p.L - t0 >= TS ? TS : p.L > t0 ? (int)(p.L - t0) : 0;
    const uint32_t rows = (1u << inside) - 1;                 // rows behind the end belong to none
    m.out |= ((1u << TS) - 1) & ~rows; m.start &= rows; m.end &= rows;
    m.start = __builtin_amdgcn_readfirstlane(m.start); m.end = __builtin_amdgcn_readfirstlane(m.end); m.out = __builtin_amdgcn_readfirstlane(m.out);
    return m;
}
__device__ inline int64_t uniform(int64_t v) { return of_lane(v, 0); }
// Packed rows in two forms: most pieces have no mark and run as those of one long sequence.
template <bool B> struct Flag { static constexpr bool value = B; };
template <bool PACKED, class F> __device__ inline void by_marks(const Marks& m, F f) {
    if constexpr (PACKED) { if (m.start | m.end | m.out) f(Flag<true>{}); else f(Flag<false>{}); }
    else f(Flag<false>{});
}

// ---- the scan over the tiles of a chain -----------------------------------------------------------------------------------------------------------------------------

template <class S, int V> struct Lds {
    S A[NW][64 * V], H[NW][64 * V];                           // maps of the pieces
    S pA[NW][64 * V], pH[NW][64 * V];                         // maps of the group's earlier tiles, NW at a time
    S c[64 * V];                                              // state at the group's start
    uint32_t cut[NW], pcut[NW];
    uint32_t ticket;
};

// A state of exactly zero leaves H whatever A is: decays above one may have overflowed in A over the rows, and where one of them is not finite itself H says so already (it starts from
// the same zero).
template <class S> __device__ inline S through(S A, S H, uint32_t cut, S c) { return cut || c == S(0) ? H : A * c + H; }
// Over a tile and more the product of the decays may fall below the smallest number.  What it leaves of a finite state is nothing, but an infinite one stays infinite unless a decay is zero
// itself: such a product is kept as the smallest number there is, which acts as zero on finite states.  `least` is the smallest of its factors.
template <class S> constexpr S LEAST = sizeof(S) == 4 ? S(1.40129846e-45f) : S(4.94065645841246544e-324);
template <class S> __device__ inline S product(S A, S least) { return A == S(0) && least > S(0) ? LEAST<S> : A; }
template <class S> __device__ inline S far_through(S A, S H, uint32_t cut, S c) { return through(A, H, cut, fabs(A) <= LEAST<S> && fabs(c) < S(INFINITY) ? S(0) : c); }

// The state at the start of position `k` of chain `c` (positions are in scan order; the adjoint counts tiles from the end), given the maps of its NW pieces in sh.A / sh.H / sh.cut
// (piece order is scan order too).  `first`: the state at the chain's start.  Publishes what later tiles of the chain wait for.  Returns with all pieces' waves past a barrier.
template <class S, int V> __device__ inline void chain(const Args& p, Lds<S, V>& sh, int64_t c, int k, const S (&first)[V], S (&carry)[V]) {
    constexpr int CW = 64 * V, W = WPV<S>, WM = WPM<S>;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, ch = lane * V;
    const int g = k / p.GS, base = g * p.GS, before = k - base, ngroups = (p.ntiles + p.GS - 1) / p.GS;
    const bool last = k == p.ntiles - 1, closes = !last && before == p.GS - 1;
    __syncthreads();
    S A[V], H[V], least[V];
    uint32_t cut = 0;
    if (wave == 0 && !last) {                                 // the tile's own map
#pragma unroll
        for (int v = 0; v < V; ++v) { A[v] = least[v] = S(1); H[v] = S(0); }
        for (int w = 0; w < NW; ++w) {
            const uint32_t q = sh.cut[w];
            cut |= q;
#pragma unroll
            for (int v = 0; v < V; ++v) { H[v] = through(sh.A[w][ch + v], sh.H[w][ch + v], q, H[v]); A[v] *= sh.A[w][ch + v]; least[v] = fmin(least[v], fabs(sh.A[w][ch + v])); }
        }
#pragma unroll
        for (int v = 0; v < V; ++v) A[v] = product(A[v], least[v]);
        if (!closes) {                                        // (only later tiles of the same group read it)
            uint64_t* dst = p.agg + (c * p.ntiles + k) * WM * CW + ch;
#pragma unroll
            for (int v = 0; v < V; ++v) publish_map(dst + v, CW, A[v], H[v], cut);
        }
    }
    // the maps of the group's earlier tiles: a wave takes GS / NW neighbouring ones, all requested before the first is waited for, and composes them; the waves' maps are composed to (B, G)
    const int per = p.GS / NW, j0 = wave * per;
    if (j0 < before) {
        const uint64_t* src = p.agg + (c * p.ntiles + base + j0) * WM * CW + ch;
        uint64_t seen[MOST_GS / NW][V];
#pragma unroll
        for (int m = 0; m < MOST_GS / NW; ++m)
#pragma unroll
            for (int v = 0; v < V; ++v) seen[m][v] = sizeof(S) == 4 && m < per && j0 + m < before ? get(src + m * WM * CW + v) : 0;
        S a[V], h[V];
        uint32_t q = 0;
#pragma unroll
        for (int v = 0; v < V; ++v) { a[v] = least[v] = S(1); h[v] = S(0); }
#pragma unroll
        for (int m = 0; m < MOST_GS / NW; ++m)
            if (m < per && j0 + m < before) {
                uint32_t qm = 0;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    S am, hm;
                    qm = await_map(src + m * WM * CW + v, CW, seen[m][v], am, hm);
                    h[v] = far_through(am, hm, qm, h[v]); a[v] *= am; least[v] = fmin(least[v], fabs(am));
                }
                q |= qm;
            }
#pragma unroll
        for (int v = 0; v < V; ++v) { sh.pA[wave][ch + v] = product(a[v], least[v]); sh.pH[wave][ch + v] = h[v]; }
        if (lane == 0) sh.pcut[wave] = q;
    }
    S B[V], G[V];
    uint32_t gcut = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) { B[v] = least[v] = S(1); G[v] = S(0); }
    if (before > 0) {
        __syncthreads();
        for (int i = 0; i * per < before; ++i) {
            const uint32_t q = sh.pcut[i];
            gcut |= q;
#pragma unroll
            for (int v = 0; v < V; ++v) { G[v] = far_through(sh.pA[i][ch + v], sh.pH[i][ch + v], q, G[v]); B[v] *= sh.pA[i][ch + v]; least[v] = fmin(least[v], fabs(sh.pA[i][ch + v])); }
        }
#pragma unroll
        for (int v = 0; v < V; ++v) B[v] = product(B[v], least[v]);
    }
    // the state at the group's start: wave 0 waits for it and, in the group's last tile, has the next group's on its way two operations later
    if (g > 0) {
        if (wave == 0) {
            const uint64_t* src = p.car + (c * ngroups + g) * W * CW + ch;
            uint64_t* dst = p.car + (c * ngroups + g + 1) * W * CW + ch;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                S s;
                await_value(src + v, CW, s);
                if (closes) publish(dst + v, CW, far_through(A[v], H[v], cut, far_through(B[v], G[v], gcut, s)), TAG_VALUE);
                sh.c[ch + v] = s;
            }
        }
        __syncthreads();
#pragma unroll
        for (int v = 0; v < V; ++v) carry[v] = far_through(B[v], G[v], gcut, sh.c[ch + v]);
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            carry[v] = far_through(B[v], G[v], gcut, first[v]);
            if (wave == 0 && closes) publish(p.car + (c * ngroups + g + 1) * W * CW + ch + v, CW, far_through(A[v], H[v], cut, carry[v]), TAG_VALUE);
        }
    }
}

// The tile of this workgroup.  Tile t: chain t % nchains, position t / nchains in scan order.  (Workgroups that stay and request the next tile's inputs while they wait for a state were
// slower: a tile that is taken early and begun late holds up its chain; 226 us against 201 for one sequence of 65536 rows.)
__device__ inline uint32_t take(const Args& p, uint32_t* slot) {
    if (p.ntiles == 1) return blockIdx.x;
    if (threadIdx.x == 0) *slot = atomicAdd(p.ticket, 1u);
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(*slot);
}

// A row is addressed by a wave-uniform base and a 32-bit byte offset of the lane: the row's part of the address is scalar arithmetic.
// What is on its way stays one integer a lane (two 16-bit values split up would take two registers), and `arrived` keeps the compiler from splitting it, and so waiting for it, where it
// is requested instead of where it is used.
template <int BYTES> struct Bits;
template <> struct Bits<2> { typedef uint16_t memory; typedef uint32_t type; };
template <> struct Bits<4> { typedef uint32_t memory, type; };
template <> struct Bits<8> { typedef uint64_t memory, type; };
template <class T, int V> using Raw = typename Bits<sizeof(T) * V>::type;
template <class T, int V> using RawMemory = typename Bits<sizeof(T) * V>::memory;
template <class T, int V> __device__ inline Raw<T, V> read(const T* row, uint32_t lane_bytes) { return *(const RawMemory<T, V>*)((const char*)row + lane_bytes); }
template <class T, int V> __device__ inline T part(Raw<T, V> r, int v) { return __builtin_bit_cast(Pack<T, V>, (RawMemory<T, V>)r).v[v]; }
template <class R, int N> __device__ inline void arrived(R (&r)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+v"(r[i]));
}
template <class T, int V> __device__ inline void write(T* row, uint32_t lane_bytes, const Pack<T, V>& v) { *(Pack<T, V>*)((char*)row + lane_bytes) = v; }

// ---- forward ------------------------------------------------------------------------------------------------------------------------------------------------------

// where a piece of a tile lies
struct Piece { int64_t b, c0, t0; int k, rows, channels; };
template <int V, int TS> __device__ inline Piece piece_of(const Args& p, uint32_t tile, int wave, bool backwards) {
    Piece q;
    const uint32_t c = tile % (uint32_t)p.nchains;
    q.k = (int)(tile / (uint32_t)p.nchains);
    q.b = c / (uint32_t)p.ncg; q.c0 = (int64_t)(c % (uint32_t)p.ncg) * (64 * V);
    q.channels = (int)(p.D - q.c0 < 64 * V ? p.D - q.c0 : 64 * V);
    q.t0 = (int64_t)(backwards ? p.ntiles - 1 - q.k : q.k) * (NW * TS) + wave * TS;
    q.rows = (int)(p.L - q.t0 < TS ? (p.L > q.t0 ? p.L - q.t0 : 0) : TS);
    return q;
}
// the piece's rows of one input; behind the end the last row again (L > 0), which nothing uses
template <class T, int V, int TS> __device__ inline void fetch(const Args& p, const void* base, int64_t sb, int64_t st, const Piece& q, uint32_t lane_bytes, Raw<T, V> (&r)[TS]) {
    const int64_t t = q.t0 < p.L ? q.t0 : p.L - 1;
    const T* row = (const T*)base + (q.b * sb + t * st + q.c0);
#pragma unroll
    for (int i = 0; i < TS; ++i) {
        r[i] = read<T, V>(row, lane_bytes);
        row += i + 1 < q.rows ? st : 0;                       // (stepped: TS multiples of st would be kept, and spilled, across the tiles)
    }
}

template <class T, class TG, class S, int V, int FORM, bool COUPLED, bool PACKED>
__global__ void __launch_bounds__(NT, sizeof(S) == 8 ? 2 : 4) k_forward(const Args p) {
    __shared__ Lds<S, V> sh;
    constexpr int TS = TSF;
    __shared__ int64_t seqs[PACKED ? NW : 1][TS];
    constexpr bool FAST = sizeof(T) == 2 && sizeof(TG) == 2;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const uint32_t tile = take(p, &sh.ticket);
    const Piece q = piece_of<V, TS>(p, tile, wave, false);
    const int64_t b = q.b, c = tile % (uint32_t)p.nchains, t0 = q.t0, c0 = q.c0;
    const int k = q.k, rows = q.rows;
    const bool on = lane * V < q.channels;
    const uint32_t lv = on ? lane * V : 0, lt = lv * sizeof(T);     // lanes past the last channel read the first one and write nothing
    Raw<T, V> rx[TS]; Raw<TG, V> rg[TS];
    Window win{};
    if constexpr (PACKED) { win = window_of(p, t0); __builtin_amdgcn_sched_barrier(0); }
    fetch<TG, V, TS>(p, p.gate, p.g_sb, p.g_st, q, lv * sizeof(TG), rg);
    fetch<T, V, TS>(p, p.x, p.x_sb, p.x_st, q, lt, rx);
    Marks m{0, 0, 0};
    if constexpr (PACKED) m = marks_of<TS>(p, t0, win, seqs[wave]);
    const uint32_t cuts = PACKED ? (m.start | m.out) : 0;
    arrived(rg); arrived(rx);
    S a[TS][V], u[TS][V];                                     // (a, b) of each row
#pragma unroll
    for (int i = 0; i < TS; ++i)
#pragma unroll
        for (int v = 0; v < V; ++v) {
            S rest = S(0);
            decay<FORM, COUPLED, FAST, S>((S)part<TG, V>(rg[i], v), a[i][v], rest);
            u[i][v] = COUPLED ? rest * (S)part<T, V>(rx[i], v) : (S)part<T, V>(rx[i], v);
        }
    if (rows < TS) {                                          // rows behind the end pass a state on
#pragma unroll
        for (int i = 0; i < TS; ++i) if (i >= rows) {
#pragma unroll
            for (int v = 0; v < V; ++v) { a[i][v] = S(1); u[i][v] = S(0); }
        }
    }
    if constexpr (PACKED) if (cuts) {
#pragma unroll
        for (int i = 0; i < TS; ++i) {
            if ((m.start >> i) & 1) {
                const int64_t s = uniform(seqs[wave][i]);
                if (p.h0) {
#pragma unroll
                    for (int v = 0; v < V; ++v) u[i][v] += a[i][v] * ((const S*)p.h0 + (s * p.D + c0))[lv + v];
                } else {
#pragma unroll
                    for (int v = 0; v < V; ++v) u[i][v] += a[i][v] * S(0);
                }
            }
            if ((m.out >> i) & 1) {
#pragma unroll
                for (int v = 0; v < V; ++v) u[i][v] = S(0);
            }
        }
    }
    S A[V], H[V];
#pragma unroll
    for (int v = 0; v < V; ++v) { A[v] = S(1); H[v] = S(0); }
    by_marks<PACKED>(m, [&](auto marked) {
#pragma unroll
        for (int i = 0; i < TS; ++i)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const bool cut = marked.value && ((cuts >> i) & 1);
                H[v] = cut ? u[i][v] : a[i][v] * H[v] + u[i][v];
                A[v] *= a[i][v];                              // not used where the piece is cut
            }
    });
#pragma unroll
    for (int v = 0; v < V; ++v) { sh.A[wave][lane * V + v] = A[v]; sh.H[wave][lane * V + v] = H[v]; }
    if (lane == 0) sh.cut[wave] = cuts != 0;
    S first[V], st[V];
#pragma unroll
    for (int v = 0; v < V; ++v) first[v] = (!PACKED && p.h0) ? ((const S*)p.h0 + (b * p.D + c0))[lv + v] : S(0);
    chain<S, V>(p, sh, c, k, first, st);
    for (int w = 0; w < wave; ++w) {
        const uint32_t z = sh.cut[w];
#pragma unroll
        for (int v = 0; v < V; ++v) st[v] = through(sh.A[w][lane * V + v], sh.H[w][lane * V + v], z, st[v]);
    }
    if (p.ckpt && on && wave * TS % TTA == 0 && t0 / TTA < p.nckpt) {
#pragma unroll
        for (int v = 0; v < V; ++v) ((S*)p.ckpt + ((b * p.nckpt + t0 / TTA) * p.D + c0))[lv + v] = st[v];
    }
    T* hr = (T*)p.h + (b * p.h_sb + t0 * p.h_st + c0);
    by_marks<PACKED>(m, [&](auto marked) {
#pragma unroll
        for (int i = 0; i < TS; ++i) {
            Pack<T, V> o;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                st[v] = (marked.value && ((cuts >> i) & 1)) ? u[i][v] : a[i][v] * st[v] + u[i][v];
                o.v[v] = (T)st[v];
            }
            if (on && i < rows) write<T, V>(hr, lt, o);
            hr += p.h_st;
            if constexpr (marked.value) {
                if ((m.end >> i) & 1) {
                    const int64_t s = uniform(seqs[wave][i]);
                    if (on) {
#pragma unroll
                        for (int v = 0; v < V; ++v) ((S*)p.h_final + (s * p.D + c0))[lv + v] = st[v];
                    }
                }
            }
        }
    });
    if constexpr (PACKED) {                                   // a sequence without rows ends where it starts
        for (int64_t s = (int64_t)k * NW + wave; s < p.nseq; s += (int64_t)p.ntiles * NW)
            if (offset_at(p, s + 1) <= offset_at(p, s) && on) {
#pragma unroll
                for (int v = 0; v < V; ++v) ((S*)p.h_final + (s * p.D + c0))[lv + v] = p.h0 ? ((const S*)p.h0 + (s * p.D + c0))[lv + v] : S(0);
            }
    } else if (on && k == p.ntiles - 1 && t0 <= p.L - 1 && t0 + TS > p.L - 1) {
#pragma unroll
        for (int v = 0; v < V; ++v) ((S*)p.h_final + (b * p.D + c0))[lv + v] = st[v];
    }
}

// ---- adjoint ------------------------------------------------------------------------------------------------------------------------------------------------------
// Where both a and 1 - a are needed, 16-bit data keep the smaller one in registers, with its own digits, and the larger one is its difference from one, good to half a unit: both are factors
// of gradients, and 1 - (1 - a) would have none of a's digits left at exp(-17).  (Packed rows keep both: their scalar registers have no room for the masks, which made 87 us of 65-68.)  Wider
// data keep a and evaluate the gate again at the end.  16-bit data also leave x and dh
// as they arrived and make 32-bit values of them each time they are used (`again` hides that they are the same values), and read dh a second time, from L2: then three workgroups share
// a CU instead of two (80 registers), and the adjoint of 8 x 4096 x 2048 BF16 takes 185 us instead of 204 (two workgroups a CU with both values in registers).  Packed rows that keep both
// have two: 69-83 us for 37 ... 512 sequences of 16384 x 1024 F16.
template <class T, class TG, class S, int V, int FORM, bool COUPLED, bool PACKED>
__global__ void __launch_bounds__(NT, sizeof(S) == 8 ? 2 : sizeof(T) == 2 && sizeof(TG) == 2 && !(PACKED && (COUPLED || FORM == 2)) ? 6 : 4) k_adjoint(const Args p) {
    __shared__ Lds<S, V> sh;
    constexpr int TS = TSA;
    __shared__ int64_t seqs[PACKED ? NW : 1][TS];
    constexpr bool FAST = sizeof(T) == 2 && sizeof(TG) == 2, REST = COUPLED || FORM == 2, KEEP = REST && FAST, LATE = KEEP || !COUPLED;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const uint32_t taken = take(p, &sh.ticket);
    const Piece q = piece_of<V, TS>(p, taken, wave, true);
    const int64_t b = q.b, c = taken % (uint32_t)p.nchains, t0 = q.t0, c0 = q.c0;
    const int k = q.k, rows = q.rows, tile = p.ntiles - 1 - k;      // the scan runs from the end: position 0 is the last tile
    const bool on = lane * V < q.channels;
    const uint32_t lv = on ? lane * V : 0, lt = lv * sizeof(T), lg = lv * sizeof(TG);
    Raw<T, V> rx[TS], rd[TS]; Raw<TG, V> rg[TS];
    Window win{};
    if constexpr (PACKED) { win = window_of(p, t0); __builtin_amdgcn_sched_barrier(0); }
    fetch<TG, V, TS>(p, p.gate, p.g_sb, p.g_st, q, lg, rg);
    fetch<T, V, TS>(p, p.x, p.x_sb, p.x_st, q, lt, rx);
    if (p.dh) fetch<T, V, TS>(p, p.dh, p.dh_sb, p.dh_st, q, lt, rd);
    else {
#pragma unroll
        for (int i = 0; i < TS; ++i) rd[i] = 0;
    }
    Marks m{0, 0, 0};
    if constexpr (PACKED) m = marks_of<TS>(p, t0, win, seqs[wave]);
    const uint32_t cuts = PACKED ? (m.start | m.out) : 0;
    arrived(rg); arrived(rx); arrived(rd);
    constexpr bool PAIR = KEEP && FORM != 0, BOTH = PAIR && PACKED;      // (a given decay is kept itself, 1 - a is its difference from one by definition)
    S kept[TS][V], rests[BOTH ? TS : 1][V];                   // a or (PAIR) the smaller of a and 1 - a of each row, or both
    S before[TS][V];                                          // the state before each row; till then its b unless that is made again from x (LATE)
    bool low[TS][V];                                          // PAIR: a is what is kept: a mask a row in scalar registers
    auto a = [&](int i, int v) -> S { return PAIR && !low[i][v] ? S(1) - kept[i][v] : kept[i][v]; };
    auto rest_of = [&](int i, int v) -> S {                   // KEEP
        if constexpr (BOTH) return rests[i][v];
        else return PAIR && !low[i][v] ? kept[i][v] : S(1) - kept[i][v];
    };
    auto b_of = [&](int i, int v) -> S {
        if constexpr (!LATE) return before[i][v];
        const S x = (S)part<T, V>(rx[i], v);
        return COUPLED ? rest_of(i, v) * x : x;
    };
    auto again = [&]() {
        if constexpr (sizeof(T) == 2) arrived(rx);
        if constexpr (KEEP)
#pragma unroll
            for (int i = 0; i < TS; ++i) { arrived(kept[i]); if constexpr (BOTH) arrived(rests[i]); }
    };
    auto at_seq = [&](const void* of, int i, int v) -> S {    // of the sequence that row i belongs to, in h0 or dh_final
        const int64_t s = uniform(seqs[wave][i]);
        return of ? ((const S*)of + (s * p.D + c0))[lv + v] : S(0);
    };
    // the cotangent of a row's state from outside the recurrence (a sequence's last row also feeds its final state); nothing in a row of no sequence
    auto cot = [&](auto marked, int i, int v) -> S {
        S d = (S)part<T, V>(rd[i], v);
        if constexpr (marked.value) {
            if ((m.out >> i) & 1) d = S(0);
            if ((m.end >> i) & 1) d += at_seq(p.dh_final, i, v);
        }
        return d;
    };
#pragma unroll
    for (int i = 0; i < TS; ++i)
#pragma unroll
        for (int v = 0; v < V; ++v) {
            S aa, rest = S(0);
            decay<FORM, REST, FAST, S>((S)part<TG, V>(rg[i], v), aa, rest);
            low[i][v] = PAIR && (BOTH || aa < S(0.5));
            kept[i][v] = PAIR && !low[i][v] ? rest : aa;
            if constexpr (BOTH) rests[i][v] = rest;
            if constexpr (!LATE) before[i][v] = rest * (S)part<T, V>(rx[i], v);
        }
    if (rows < TS) {                                          // rows behind the end pass a state on
#pragma unroll
        for (int i = 0; i < TS; ++i) if (i >= rows) {
            rx[i] = 0; rd[i] = 0;
#pragma unroll
            for (int v = 0; v < V; ++v) { low[i][v] = BOTH; kept[i][v] = PAIR && !BOTH ? S(0) : S(1); if constexpr (BOTH) rests[i][v] = S(0); if constexpr (!LATE) before[i][v] = S(0); }
        }
    }
    if constexpr (PACKED) if (m.out) {
#pragma unroll
        for (int i = 0; i < TS; ++i) if ((m.out >> i) & 1) {
            rx[i] = 0;
#pragma unroll
            for (int v = 0; v < V; ++v) if constexpr (!LATE) before[i][v] = S(0);
        }
    }
    // the rows' forward map, for the states
    S A[V], H[V], F[V];
#pragma unroll
    for (int v = 0; v < V; ++v) { A[v] = S(1); H[v] = S(0); }
    by_marks<PACKED>(m, [&](auto marked) {
#pragma unroll
        for (int i = 0; i < TS; ++i)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const S ai = a(i, v);
                S bb = (marked.value && ((m.out >> i) & 1)) ? S(0) : b_of(i, v);
                if constexpr (marked.value) { if ((m.start >> i) & 1) bb += ai * at_seq(p.h0, i, v); }
                H[v] = (marked.value && ((cuts >> i) & 1)) ? bb : ai * H[v] + bb;
                A[v] *= ai;
            }
    });
#pragma unroll
    for (int v = 0; v < V; ++v) { sh.A[wave][lane * V + v] = A[v]; sh.H[wave][lane * V + v] = H[v]; }
    if (lane == 0) sh.cut[wave] = cuts != 0;
    __syncthreads();
#pragma unroll
    for (int v = 0; v < V; ++v) F[v] = ((const S*)p.ckpt + ((b * p.nckpt + tile) * p.D + c0))[lv + v];
    for (int w = 0; w < wave; ++w) {
        const uint32_t z = sh.cut[w];
#pragma unroll
        for (int v = 0; v < V; ++v) F[v] = through(sh.A[w][lane * V + v], sh.H[w][lane * V + v], z, F[v]);
    }
    __syncthreads();
    // the rows' reverse map R -> A R + H with the same product A
    again();
#pragma unroll
    for (int v = 0; v < V; ++v) H[v] = S(0);
    by_marks<PACKED>(m, [&](auto marked) {
#pragma unroll
        for (int i = TS - 1; i >= 0; --i) {
#pragma unroll
            for (int v = 0; v < V; ++v) { const S d = cot(marked, i, v); H[v] = (marked.value && ((cuts >> i) & 1)) ? S(0) : a(i, v) * (d + H[v]); }
        }
    });
    again();
    const int rw = NW - 1 - wave;                             // the piece's place in scan order
#pragma unroll
    for (int v = 0; v < V; ++v) { sh.A[rw][lane * V + v] = A[v]; sh.H[rw][lane * V + v] = H[v]; }
    if (lane == 0) sh.cut[rw] = cuts != 0;
    S first[V], R[V];
#pragma unroll
    for (int v = 0; v < V; ++v) first[v] = (!PACKED && p.dh_final) ? ((const S*)p.dh_final + (b * p.D + c0))[lv + v] : S(0);
    chain<S, V>(p, sh, c, k, first, R);
    for (int w = 0; w < rw; ++w) {
        const uint32_t z = sh.cut[w];
#pragma unroll
        for (int v = 0; v < V; ++v) R[v] = through(sh.A[w][lane * V + v], sh.H[w][lane * V + v], z, R[v]);
    }
    again();
    if constexpr (sizeof(T) == 2) {
        if (p.dh) fetch<T, V, TS>(p, p.dh, p.dh_sb, p.dh_st, q, lt, rd);
        if (rows < TS) {
#pragma unroll
            for (int i = 0; i < TS; ++i) if (i >= rows) rd[i] = 0;
        }
    }
    // the states before each row, then the rows from the last to the first
    by_marks<PACKED>(m, [&](auto marked) {
#pragma unroll
        for (int i = 0; i < TS; ++i) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                if (marked.value && ((m.start >> i) & 1)) F[v] = at_seq(p.h0, i, v);
                const S bb = b_of(i, v);
                before[i][v] = F[v];
                F[v] = a(i, v) * F[v] + bb;
                if (marked.value && ((m.out >> i) & 1)) F[v] = S(0);
            }
        }
        again();
        T* dxr = (T*)p.dx + (b * p.dx_sb + (t0 + TS - 1) * p.dx_st + c0);
        TG* dgr = (TG*)p.dgate + (b * p.dg_sb + (t0 + TS - 1) * p.dg_st + c0);
#pragma unroll
        for (int i = TS - 1; i >= 0; --i) {
            Pack<T, V> ox; Pack<TG, V> og;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const S G = cot(marked, i, v) + R[v], ai = a(i, v);
                S aa, rest = S(1);
                if constexpr (KEEP) rest = rest_of(i, v);
                else if constexpr (REST) decay<FORM, true, FAST, S>((S)part<TG, V>(rg[i], v), aa, rest);
                S da = G * (COUPLED ? before[i][v] - (S)part<T, V>(rx[i], v) : before[i][v]);
                if constexpr (FORM == 1) da *= ai;
                if constexpr (FORM == 2) da *= ai * rest;
                S dx = COUPLED ? G * rest : G;
                R[v] = ai * G;
                if (marked.value && ((m.out >> i) & 1)) { da = S(0); dx = S(0); R[v] = S(0); }
                ox.v[v] = (T)dx; og.v[v] = (TG)da;
            }
            if (on && i < rows) {
                if (p.dx) write<T, V>(dxr, lt, ox);
                if (p.dgate) write<TG, V>(dgr, lg, og);
            }
            dxr -= p.dx_st; dgr -= p.dg_st;
            if constexpr (marked.value) {
                if ((m.start >> i) & 1) {
                    const int64_t s = uniform(seqs[wave][i]);
                    if (on && p.dh0) {
#pragma unroll
                        for (int v = 0; v < V; ++v) ((S*)p.dh0 + (s * p.D + c0))[lv + v] = R[v];
                    }
#pragma unroll
                    for (int v = 0; v < V; ++v) R[v] = S(0);
                }
            }
        }
    });
    if constexpr (PACKED) {
        for (int64_t s = (int64_t)k * NW + wave; s < p.nseq; s += (int64_t)p.ntiles * NW)
            if (offset_at(p, s + 1) <= offset_at(p, s) && on && p.dh0) {
#pragma unroll
                for (int v = 0; v < V; ++v) ((S*)p.dh0 + (s * p.D + c0))[lv + v] = p.dh_final ? ((const S*)p.dh_final + (s * p.D + c0))[lv + v] : S(0);
            }
    } else if (on && tile == 0 && wave == 0 && p.dh0) {
#pragma unroll
        for (int v = 0; v < V; ++v) ((S*)p.dh0 + (b * p.D + c0))[lv + v] = R[v];
    }
}

// ---- single step --------------------------------------------------------------------------------------------------------------------------------------------------
// One row per sequence: state[slot] = a state[slot] + b, h = the new state.  Rows that name the same slot are steps of one sequence in the order of the rows: the first of them
// takes all, so no two workgroups touch a state.  A slot outside [0, nslots) (-1 pads a batch) has no state: its h is zero.
// A row is read, updated and written by neighbouring lanes of workgroups of their own: 14 bytes a BF16 channel.  256 rows x 4096 channels 6.7 us (2.2 TB/s; a launch alone is 2.2 us, which
// is one row of 2048 channels).
struct StepArgs {
    const void *x, *gate, *slots;
    void *state, *h;
    int64_t x_s, g_s, st_s, h_s, B, D, nslots;
    int32_t slots64;
};
constexpr int NS = 256;
template <class T, class TG, class S, int V, int FORM, bool COUPLED>
__global__ void __launch_bounds__(NS) k_step(const StepArgs p, int ncg) {
    const int64_t r = blockIdx.x / (uint32_t)ncg, ch = ((int64_t)(blockIdx.x % (uint32_t)ncg) * NS + threadIdx.x) * V;
    const bool on = ch < p.D;
    auto slot_of = [&](int64_t i) -> int64_t { return p.slots64 ? ((const int64_t*)p.slots)[i] : (int64_t)((const int32_t*)p.slots)[i]; };
    const int64_t slot = p.slots ? slot_of(r) : r;
    if (slot < 0 || slot >= p.nslots) {
        if (on) {
            Pack<T, V> o;
#pragma unroll
            for (int v = 0; v < V; ++v) o.v[v] = (T)S(0);
            *(Pack<T, V>*)((T*)p.h + r * p.h_s + ch) = o;
        }
        return;
    }
    bool more = false;
    if (p.slots) {
        bool earlier = false, later = false;
        for (int64_t i = threadIdx.x; i < p.B; i += NS) if (i != r && slot_of(i) == slot) { if (i < r) earlier = true; else later = true; }
        if (__syncthreads_or(earlier)) return;
        more = __syncthreads_or(later);
    }
    if (!on) return;
    S st[V];
    S* sp = (S*)p.state + slot * p.st_s + ch;
    {
        const Pack<S, V> q = *(const Pack<S, V>*)sp;
#pragma unroll
        for (int v = 0; v < V; ++v) st[v] = q.v[v];
    }
    for (int64_t i = r; i < p.B; ++i) {
        if (i != r) { if (!more) break; if (slot_of(i) != slot) continue; }
        const Pack<T, V> x = *(const Pack<T, V>*)((const T*)p.x + i * p.x_s + ch);
        const Pack<TG, V> g = *(const Pack<TG, V>*)((const TG*)p.gate + i * p.g_s + ch);
        Pack<T, V> o;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            S a, rest = S(0);
            decay<FORM, COUPLED, sizeof(T) == 2 && sizeof(TG) == 2, S>((S)g.v[v], a, rest);
            st[v] = a * st[v] + (COUPLED ? rest * (S)x.v[v] : (S)x.v[v]);
            o.v[v] = (T)st[v];
        }
        *(Pack<T, V>*)((T*)p.h + i * p.h_s + ch) = o;
    }
    Pack<S, V> q;
#pragma unroll
    for (int v = 0; v < V; ++v) q.v[v] = st[v];
    *(Pack<S, V>*)sp = q;
}

// one launch per (types, vector width, form, coupled, packed); translation units instantiate these (hipadj_tu_recurrence.hip)
enum { PAIR_F64 = 0, PAIR_F32, PAIR_BF16, PAIR_BF16_F32, PAIR_F16, PAIR_F16_F32 };     // (x, gate)
template <int PAIR> struct Types;
template <> struct Types<PAIR_F64> { typedef double T, TG, S; static constexpr int V = 1; };
template <> struct Types<PAIR_F32> { typedef float T, TG, S; static constexpr int V = 1; };
template <> struct Types<PAIR_BF16> { typedef bf16 T, TG; typedef float S; static constexpr int V = 2; };
template <> struct Types<PAIR_BF16_F32> { typedef bf16 T; typedef float TG, S; static constexpr int V = 2; };
template <> struct Types<PAIR_F16> { typedef f16 T, TG; typedef float S; static constexpr int V = 2; };
template <> struct Types<PAIR_F16_F32> { typedef f16 T; typedef float TG, S; static constexpr int V = 2; };

template <int PAIR> void launch(const Args& a, bool adjoint, bool wide, int form, bool coupled, bool packed, hipStream_t stream);
template <int PAIR> void launch_step(const StepArgs& a, bool wide, int form, bool coupled, hipStream_t stream);

}  // namespace rec
