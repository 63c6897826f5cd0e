// hipadj_tu_orthogonal.hip — the orthogonalised update: launches and C entry points.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include "hipadj_ops.hpp"
#include "hipadj_orthogonal.hpp"

namespace orth {

struct Plan { Mat q; bool split, small; int64_t bytes; };

static int64_t padded(int64_t v) { return (v + PADDED - 1) / PADDED * PADDED; }

// One F16 term a factor where BF16 rounds the output anyway and the matrix is large enough for the products to be what it costs; see hipadj_orthogonal.hpp for the error
static bool one_term(const hipadj_orthogonal* o) { return o->dtype == HIPADJ_BF16 && std::min(o->rows, o->cols) >= 256; }

static Plan plan_of(const hipadj_orthogonal* o, char* base) {
    Plan p;
    Mat& q = p.q;
    q.flip = o->rows > o->cols;
    q.m = std::min(o->rows, o->cols); q.n = std::max(o->rows, o->cols);
    q.mp = padded(q.m); q.np = padded(q.n);
    q.batch = o->batch;
    p.split = !one_term(o);
    p.small = q.n <= 128;
    p.bytes = 0;
    if (p.small) return p;
    int64_t at = 0;
    auto take = [&](int64_t bytes) { char* r = base + at; at += (bytes + 255) / 256 * 256; return r; };
    const int T = p.split ? 2 : 1;
    q.x[1] = q.xt[0][1] = q.xt[1][1] = q.a[1] = q.b[1] = nullptr;
    for (int t = 0; t < T; ++t) {
        q.x[t] = (f16*)take(q.batch * q.mp * q.np * 2);
        q.xt[0][t] = (f16*)take(q.batch * q.mp * q.np * 2);
        q.xt[1][t] = (f16*)take(q.batch * q.mp * q.np * 2);
        q.a[t] = (f16*)take(q.batch * q.mp * q.mp * 2);
        q.b[t] = (f16*)take(q.batch * q.mp * q.mp * 2);
    }
    q.master = (float*)take(q.batch * q.mp * q.np * 4);
    q.nblocks = (int)std::max<int64_t>(1, std::min<int64_t>({NORM_BLOCKS, (q.m * q.n + NORM_SPAN - 1) / NORM_SPAN, std::max<int64_t>(1, 2048 / std::max<int64_t>(1, q.batch))}));
    q.partial = (double*)take(q.batch * q.nblocks * 8);
    p.bytes = at;
    return p;
}

static int64_t tiles_of(const Product& g, int64_t batch, bool lower, int64_t BT) {
    const int64_t ti = (g.M + BT - 1) / BT, tj = (g.N + BT - 1) / BT;
    return (lower ? ti * (ti + 1) / 2 : ti * tj) * batch;
}
template <class T, int BT, int EPI, bool SPLIT, int SLOTS> static void product(const Product& g, const Mat& q, const Io<T>& io, int from, int to, hipStream_t s) {
    const dim3 grid((uint32_t)(tiles_of(g, 1, EPI != APPLY && EPI != LAST, BT) * (EPI == PARTS ? g.parts : 1)), 1, (uint32_t)q.batch);
    ops_launch(k_product<T, BT, EPI, SPLIT, SLOTS>, grid, dim3(256), s, g, q, io, from, to);
}

// The time of a product by tiles of BT, microseconds: rounds over the 256 CUs, each with a fixed part (first requests, epilogue) and one for every row of K, which grows with the share
// of the CUs at work (they share L2 and power).  Fitted to 12 shapes from 256 x 256 to 4096 x 4096 with every tile, within 15 % where the choice is between near ones.  Larger tiles read
// less a product, smaller ones leave fewer CUs without work: 4096 x 4096 takes 253 tiles of 192 for a symmetric product (87 us; 528 of 128: 119, 136 of 256: 117) and 256 of 256 for
// B X (147; of 192: 167), 512 x 512 takes tiles of 64 (5 us; of 128: 9, of 256: 27).
struct TileCost { int BT; double fixed, round, row, load; };
static constexpr TileCost ONE_TERM[] = {{64, 2.0, 2.2, 3.0e-3, 0.5}, {128, 2.0, 3.5, 6.0e-3, 0.65}, {192, 3.0, 8.0, 9.8e-3, 0.9}, {256, 4.0, 14.0, 16.3e-3, 0.9}};
static constexpr TileCost TWO_TERMS[] = {{64, 2.0, 2.5, 7.5e-3, 0.2}, {128, 3.0, 7.5, 13.0e-3, 0.5}};
static double cost_of(const TileCost& c, const Product& g, int64_t batch, bool lower, int parts) {
    const int64_t n = tiles_of(g, batch, lower, c.BT) * parts, rounds = (n + 255) / 256;
    return c.fixed + (double)rounds * (c.round + (double)g.K / parts * c.row * (1.0 + c.load * (double)n / (256.0 * (double)rounds)));
}
template <int N> static const TileCost& best_tile(const TileCost (&table)[N], const Product& g, int64_t batch, bool lower) {
    const TileCost* best = table;
    for (const TileCost& c : table) if (cost_of(c, g, batch, lower, 1) < cost_of(*best, g, batch, lower, 1)) best = &c;
    return *best;
}
// X X' of few rows and long ones has few tiles: its K is cut into parts, whose sums lie where the next X will (not in use then, and large enough where the parts are worth it) and are
// joined by a launch of its own, about 2 + 0.4 a part us.  Measured, with the join: 256 x 16384 bf16 48 us without, 30 / 19 / 15 with 2 / 4 / 8 parts; 512 x 8192 26, 20 / 16 / 19;
// 512 x 8192 F32 58, 37 / 26 / 32; 256 x 1024 6.2, 8.6 with two.  (Tiles of 128 in parts were no faster for 2048 x 8192: 68, 80 / 71 with 2 / 3.)
template <bool SPLIT> static int parts_of(const Product& g, const Mat& q) {
    const TileCost& small = SPLIT ? TWO_TERMS[0] : ONE_TERM[0];
    double least = 0.9 * (SPLIT ? cost_of(best_tile(TWO_TERMS, g, q.batch, true), g, q.batch, true, 1) : cost_of(best_tile(ONE_TERM, g, q.batch, true), g, q.batch, true, 1));
    int best = 1;
    for (int parts = 2; parts <= 8; parts *= 2) {
        if (parts > g.K / PADDED || parts * tiles_of(g, 1, true, 64) * 64 * 64 * 2 > q.mp * q.np) break;
        const double t = cost_of(small, g, q.batch, true, parts) + 2.0 + 0.4 * parts;
        if (t < least) { least = t; best = parts; }
    }
    return best;
}
template <class T, int EPI, bool SPLIT> static void product_of(const Product& g, const Mat& q, const Io<T>& io, int from, int to, hipStream_t s) {
    constexpr bool LOWER = EPI == GRAM || EPI == POLY;
    if constexpr (SPLIT) {
        if (best_tile(TWO_TERMS, g, q.batch, LOWER).BT == 64) product<T, 64, EPI, true, 2>(g, q, io, from, to, s);
        else product<T, 128, EPI, true, 2>(g, q, io, from, to, s);
    } else switch (best_tile(ONE_TERM, g, q.batch, LOWER).BT) {
        case 64: product<T, 64, EPI, false, 2>(g, q, io, from, to, s); break;
        case 128: product<T, 128, EPI, false, 1>(g, q, io, from, to, s); break;
        case 192: product<T, 192, EPI, false, 1>(g, q, io, from, to, s); break;
        default: product<T, 256, EPI, false, 1>(g, q, io, from, to, s); break;
    }
}

template <class T, bool SPLIT> static void iterate(const hipadj_orthogonal* o, const Mat& q, const Io<T>& io, hipStream_t s) {
    const bool flat = io.g_r == io.cols && (!io.mom || io.m_r == io.cols);
    const int64_t rows = flat ? 1 : io.rows, cols = flat ? io.rows * io.cols : io.cols;
    auto aligned = [&](const void* p, int64_t sb, int64_t sr, int64_t per) { return (uintptr_t)p % 16 == 0 && (q.batch == 1 || sb % per == 0) && (rows == 1 || sr % per == 0); };
    const bool vec = cols % 8 == 0 && aligned(io.grad, io.g_b, io.g_r, 16 / sizeof(T)) && (!io.mom || aligned(io.mom, io.m_b, io.m_r, 4));
    ops_launch(k_norm<T>, dim3((uint32_t)q.nblocks, (uint32_t)q.batch), dim3(256), s, io, rows, cols, vec, q.partial);
    const dim3 pieces((uint32_t)(q.np / 64), (uint32_t)(q.mp / 64), (uint32_t)q.batch);
    if (q.np / 64 * (q.mp / 64) * q.batch <= 1024) ops_launch(k_start<T, SPLIT, 16>, pieces, dim3(1024), s, io, q);
    else ops_launch(k_start<T, SPLIT, 4>, pieces, dim3(256), s, io, q);
    const int64_t smm = q.mp * q.mp, smn = q.mp * q.np;
    auto rounded = [&](int step) { return !SPLIT && step >= o->steps - 2; };
    for (int step = 0; step < o->steps; ++step) {
        const double* c = o->coefficients + 3 * step;
        const int from = step & 1, to = 1 - from;
        Product g{};
        g.c0 = (float)c[0]; g.c1 = (float)c[1]; g.c2 = (float)c[2];
        g.P[0] = g.Q[0] = q.x[0]; g.P[1] = g.Q[1] = q.x[1]; g.sP = g.sQ = smn; g.K = q.np; g.M = g.N = q.mp;
        g.parts = parts_of<SPLIT>(g, q);
        if (g.parts > 1) {
            g.tiles = (int)tiles_of(g, 1, true, 64);
            product<T, 64, PARTS, SPLIT, 2>(g, q, io, from, to, s);
            product<T, 64, JOIN, SPLIT, 2>(g, q, io, from, to, s);
        } else product_of<T, GRAM, SPLIT>(g, q, io, from, to, s);
        g.P[0] = g.Q[0] = q.a[0]; g.P[1] = g.Q[1] = q.a[1]; g.sP = g.sQ = smm; g.K = q.mp;
        product_of<T, POLY, SPLIT>(g, q, io, from, to, s);
        g.P[0] = q.b[0]; g.P[1] = q.b[1]; g.sP = smm;
        g.Q[0] = q.xt[from][0]; g.Q[1] = q.xt[from][1]; g.sQ = smn; g.N = q.np;
        g.rounded = rounded(step); g.keep = !rounded(step + 1);
        if (step + 1 < o->steps) product_of<T, APPLY, SPLIT>(g, q, io, from, to, s);
        else product_of<T, LAST, SPLIT>(g, q, io, from, to, s);
    }
}

template <class T> static void run(const hipadj_orthogonal* o, const Plan& p, const void* grad, float* mom, void* out, hipStream_t s) {
    Io<T> io;
    io.grad = (const T*)grad; io.mom = mom; io.out = (T*)out; io.rows = o->rows; io.cols = o->cols;
    io.g_b = o->grad_stride[0]; io.g_r = o->grad_stride[1]; io.m_b = o->momentum_stride[0]; io.m_r = o->momentum_stride[1]; io.o_b = o->out_stride[0]; io.o_r = o->out_stride[1];
    io.beta = (float)o->beta; io.scale = (float)o->scale; io.nesterov = o->nesterov;
    io.vec = (uintptr_t)out % (4 * sizeof(T)) == 0 && io.o_r % 4 == 0 && (o->batch == 1 || io.o_b % 4 == 0);
    if (p.small) {
        Coefficients co;
        for (int i = 0; i < 3 * o->steps; ++i) co.c[i] = (float)o->coefficients[i];
        const dim3 grid((uint32_t)o->batch);
        if (p.q.n <= 32) ops_launch(k_small<T, 32>, grid, dim3(64), s, io, p.q.m, p.q.n, p.q.flip, o->steps, co);
        else if (p.q.n <= 64) ops_launch(k_small<T, 64>, grid, dim3(256), s, io, p.q.m, p.q.n, p.q.flip, o->steps, co);
        else ops_launch(k_small<T, 128>, grid, dim3(1024), s, io, p.q.m, p.q.n, p.q.flip, o->steps, co);
        return;
    }
    if (p.split) iterate<T, true>(o, p.q, io, s);
    else if constexpr (sizeof(T) == 2) iterate<T, false>(o, p.q, io, s);
}

// How far the coefficients let the iteration grow: X starts with singular values in [0, 1], a step maps a bound s to the largest |c0 x + c1 x^3 + c2 x^5| on [0, s], reached at s or where
// the derivative vanishes, and B has eigenvalues c1 y + c2 y^2, y <= s^2.  F16 holds 2^13 X up to 8 and 2^11 A, 2^11 B up to 32: an X that goes into another step, where A = X X' is formed, may
// have singular values up to 5.6 (its square 31.4), the last one up to 6.
static bool grows(const hipadj_orthogonal* o, double& s, double& big) {
    s = 1.0; big = 0.0;
    for (int k = 0; k < o->steps; ++k) {
        if (s > 5.6) return true;
        const double c0 = o->coefficients[3 * k], c1 = o->coefficients[3 * k + 1], c2 = o->coefficients[3 * k + 2];
        auto p = [&](double x) { return std::fabs(x * (c0 + x * x * (c1 + x * x * c2))); };
        auto b = [&](double y) { return std::fabs(y * (c1 + y * c2)); };
        double most = p(s), mb = b(s * s);
        const double disc = 9 * c1 * c1 - 20 * c0 * c2;
        if (disc >= 0)
            for (int sign = -1; sign <= 1; sign += 2) {
                const double d = -3 * c1 + sign * std::sqrt(disc), y = c2 != 0 ? d / (10 * c2) : (c1 != 0 ? -c0 / (3 * c1) : -1.0);
                if (y > 0 && y < s * s) most = std::max(most, p(std::sqrt(y)));
            }
        if (c2 != 0 && -c1 / (2 * c2) > 0 && -c1 / (2 * c2) < s * s) mb = std::max(mb, b(-c1 / (2 * c2)));
        big = std::max(big, mb);
        s = most;
        if (s > 6.0 || big > 24.0) return true;
    }
    return false;
}

static int check(const hipadj_orthogonal* o) {
    if (!o || o->struct_size != sizeof(hipadj_orthogonal)) return ops_fail(HIPADJ_ERR_INVALID_ARG, "hipadj_orthogonal.struct_size does not match this library");
    if (o->dtype != HIPADJ_F32 && o->dtype != HIPADJ_BF16 && o->dtype != HIPADJ_F16) return ops_fail(HIPADJ_ERR_UNSUPPORTED, "orthogonalized update: matrices are F32, BF16 or F16");
    if (o->batch < 0 || o->rows < 0 || o->cols < 0) return ops_fail(HIPADJ_ERR_INVALID_ARG, "orthogonalized update: negative size");
    if (o->steps < 1 || o->steps > MOST_STEPS || !o->coefficients) return ops_fail(HIPADJ_ERR_INVALID_ARG, "orthogonalized update: 1 to 64 steps with three coefficients each, got %d", o->steps);
    for (int i = 0; i < 3 * o->steps; ++i)
        if (!(std::fabs(o->coefficients[i]) <= 32.0)) return ops_fail(HIPADJ_ERR_INVALID_ARG, "orthogonalized update: coefficients within +-32, got %g", o->coefficients[i]);
    double s, big;
    if (grows(o, s, big)) return ops_fail(HIPADJ_ERR_UNSUPPORTED, "orthogonalized update: with these coefficients singular values can grow to %.3g (at most 5.6 before a step, 6 behind the last) and c1 A + c2 A A to %.3g (at most 24)", s, big);
    if (!std::isfinite(o->beta) || !std::isfinite(o->scale)) return ops_fail(HIPADJ_ERR_INVALID_ARG, "orthogonalized update: beta and scale must be finite");
    if (std::max(o->rows, o->cols) > 65536 || std::min(o->rows, o->cols) > 32768 || o->batch > 65535)
        return ops_fail(HIPADJ_ERR_UNSUPPORTED, "orthogonalized update: at most 65535 matrices with sides of at most 32768 and 65536");
    return HIPADJ_OK;
}

}  // namespace orth

extern "C" int hipadj_orthogonalized_update_size(const hipadj_orthogonal* o, int64_t* workspace_bytes) {
    const int rc = orth::check(o);
    if (rc != HIPADJ_OK) return rc;
    if (workspace_bytes) *workspace_bytes = orth::plan_of(o, nullptr).bytes;
    return HIPADJ_OK;
}

extern "C" int hipadj_orthogonalized_update_dev(const hipadj_orthogonal* o, const void* grad, float* momentum, void* out, void* workspace, int64_t workspace_bytes, void* stream) {
    const int rc = orth::check(o);
    if (rc != HIPADJ_OK) return rc;
    if (o->batch == 0 || o->rows == 0 || o->cols == 0) return HIPADJ_OK;
    const orth::Plan p = orth::plan_of(o, (char*)workspace);
    if (!grad || !out || (p.bytes && (!workspace || (uintptr_t)workspace % 256 || workspace_bytes < p.bytes)))
        return ops_fail(HIPADJ_ERR_INVALID_ARG, "hipadj_orthogonalized_update_dev: grad, out and a 256-byte aligned workspace of %lld bytes are required", (long long)p.bytes);
    OpsDevice dev(o->device);
    if (dev.rc != HIPADJ_OK) return dev.rc;
    hipStream_t s = (hipStream_t)stream;
    if (o->dtype == HIPADJ_F32) orth::run<float>(o, p, grad, momentum, out, s);
    else if (o->dtype == HIPADJ_BF16) orth::run<orth::bf16>(o, p, grad, momentum, out, s);
    else orth::run<orth::f16>(o, p, grad, momentum, out, s);
    return ops_launched("orthogonalized update");
}
