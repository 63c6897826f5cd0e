// hipadj_tu_recurrence.hip — translation units of the gated linear recurrence: hipcc -DHIPADJ_TU_PAIR=<rec::PAIR_*>; without it the C entry points.
#include <algorithm>
#include "hipadj_ops.hpp"
#include "hipadj_recurrence.hpp"

#if defined(HIPADJ_TU_PAIR)
namespace rec {

template <int PAIR, int V, int FORM, bool COUPLED> static void pick(const Args& a, bool adjoint, bool packed, hipStream_t s) {
    typedef Types<PAIR> Y;
    const dim3 grid((uint32_t)((int64_t)a.nchains * a.ntiles)), block(NT);
    if (adjoint) {
        if (packed) ops_launch(k_adjoint<typename Y::T, typename Y::TG, typename Y::S, V, FORM, COUPLED, true>, grid, block, s, a);
        else ops_launch(k_adjoint<typename Y::T, typename Y::TG, typename Y::S, V, FORM, COUPLED, false>, grid, block, s, a);
    } else {
        if (packed) ops_launch(k_forward<typename Y::T, typename Y::TG, typename Y::S, V, FORM, COUPLED, true>, grid, block, s, a);
        else ops_launch(k_forward<typename Y::T, typename Y::TG, typename Y::S, V, FORM, COUPLED, false>, grid, block, s, a);
    }
}
template <int PAIR, int V> static void pick_form(const Args& a, bool adjoint, int form, bool coupled, bool packed, hipStream_t s) {
    if (form == 0) { if (coupled) pick<PAIR, V, 0, true>(a, adjoint, packed, s); else pick<PAIR, V, 0, false>(a, adjoint, packed, s); }
    else if (form == 1) { if (coupled) pick<PAIR, V, 1, true>(a, adjoint, packed, s); else pick<PAIR, V, 1, false>(a, adjoint, packed, s); }
    else { if (coupled) pick<PAIR, V, 2, true>(a, adjoint, packed, s); else pick<PAIR, V, 2, false>(a, adjoint, packed, s); }
}
template <int PAIR> void launch(const Args& a, bool adjoint, bool wide, int form, bool coupled, bool packed, hipStream_t s) {
    if (wide) pick_form<PAIR, Types<PAIR>::V>(a, adjoint, form, coupled, packed, s);
    else if constexpr (Types<PAIR>::V > 1) pick_form<PAIR, 1>(a, adjoint, form, coupled, packed, s);
}
template void launch<HIPADJ_TU_PAIR>(const Args&, bool, bool, int, bool, bool, hipStream_t);

template <int PAIR, int V, int FORM> static void pick_step(const StepArgs& a, bool coupled, hipStream_t s) {
    typedef Types<PAIR> Y;
    const int ncg = (int)((a.D + NS * V - 1) / (NS * V));
    const dim3 grid((uint32_t)(a.B * ncg)), block(NS);
    if (coupled) ops_launch(k_step<typename Y::T, typename Y::TG, typename Y::S, V, FORM, true>, grid, block, s, a, ncg);
    else ops_launch(k_step<typename Y::T, typename Y::TG, typename Y::S, V, FORM, false>, grid, block, s, a, ncg);
}
template <int PAIR, int V> static void pick_step_form(const StepArgs& a, int form, bool coupled, hipStream_t s) {
    if (form == 0) pick_step<PAIR, V, 0>(a, coupled, s); else if (form == 1) pick_step<PAIR, V, 1>(a, coupled, s); else pick_step<PAIR, V, 2>(a, coupled, s);
}
template <int PAIR> void launch_step(const StepArgs& a, bool wide, int form, bool coupled, hipStream_t s) {
    if (wide) pick_step_form<PAIR, Types<PAIR>::V>(a, form, coupled, s);
    else if constexpr (Types<PAIR>::V > 1) pick_step_form<PAIR, 1>(a, form, coupled, s);
}
template void launch_step<HIPADJ_TU_PAIR>(const StepArgs&, bool, int, bool, hipStream_t);

}  // namespace rec
#else
#include <cstdio>

namespace rec {

// the words of the chains and the ticket, zeroed before the launch that uses them
static __global__ void __launch_bounds__(256) k_zero(uint64_t* w, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) w[i] = 0;
}

// no rows: what leaves is what came in
template <class S> static __global__ void __launch_bounds__(256) k_same(S* to, const S* from, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) to[i] = from ? from[i] : S(0);
}

static int pair_of(int dtype, int gate_dtype) {
    if (dtype == HIPADJ_F64 && gate_dtype == HIPADJ_F64) return PAIR_F64;
    if (dtype == HIPADJ_F32 && gate_dtype == HIPADJ_F32) return PAIR_F32;
    if (dtype == HIPADJ_BF16) return gate_dtype == HIPADJ_BF16 ? PAIR_BF16 : gate_dtype == HIPADJ_F32 ? PAIR_BF16_F32 : -1;
    if (dtype == HIPADJ_F16) return gate_dtype == HIPADJ_F16 ? PAIR_F16 : gate_dtype == HIPADJ_F32 ? PAIR_F16_F32 : -1;
    return -1;
}
static int size_of(int dtype) { return dtype == HIPADJ_F64 ? 8 : dtype == HIPADJ_F32 ? 4 : 2; }
static void run(int pair, const Args& a, bool adjoint, bool wide, int form, bool coupled, bool packed, hipStream_t s) {
    switch (pair) {
    case PAIR_F64: launch<PAIR_F64>(a, adjoint, wide, form, coupled, packed, s); break;
    case PAIR_F32: launch<PAIR_F32>(a, adjoint, wide, form, coupled, packed, s); break;
    case PAIR_BF16: launch<PAIR_BF16>(a, adjoint, wide, form, coupled, packed, s); break;
    case PAIR_BF16_F32: launch<PAIR_BF16_F32>(a, adjoint, wide, form, coupled, packed, s); break;
    case PAIR_F16: launch<PAIR_F16>(a, adjoint, wide, form, coupled, packed, s); break;
    default: launch<PAIR_F16_F32>(a, adjoint, wide, form, coupled, packed, s); break;
    }
}

// the split of a problem: it depends on the sizes alone
static int64_t tiles_of(const hipadj_recurrence* r, bool adjoint) { const int64_t rows = adjoint ? TTA : TTF; return std::max<int64_t>(1, r->length / rows + (r->length % rows != 0)); }
// Tiles of a group.  The exchange from group to group is what a few long chains wait for, and reading the group's earlier maps is what many chains pay for.  Measured with groups of 8, 16
// and 32, forward and adjoint, BF16: 1 x 65536 x 128 (one chain) 53 / 36 / 31 and 95 / 62 / 48 us; 1 x 65536 x 512 (4 chains) 71 / 67 / 70 and 134 / 114 / 118; 1 x 65536 x 2048 (16 chains)
// 206 / 207 / 213 and 357 / 363 / 372; 8 x 4096 x 2048 (128 chains) 97 / 98 / 96 and 162 / 168 / 176.  (All before maps passed exactly and the adjoint kept small decays; the chosen ones are
// 31, 50; 66, 115; 204, 358 and 107, 185 since.)
static int group_of(int64_t nchains) { return nchains <= 2 ? 32 : nchains <= 4 ? 16 : 8; }
// 64-bit words of a launch: the ticket, a map for each tile, a state for each group, by channel
static int64_t words_of(const hipadj_recurrence* r, int64_t ntiles, int V) {
    if (ntiles == 1) return 0;
    const int64_t CW = 64 * V, chains = r->batch * ((r->channels + CW - 1) / CW), GS = group_of(chains), wide = r->dtype == HIPADJ_F64;
    return 1 + chains * CW * ((wide ? WPM<double> : WPM<float>) * ntiles + (wide ? WPV<double> : WPV<float>) * ((ntiles + GS - 1) / GS));
}

constexpr int64_t MOST_THREADS = (int64_t(1) << 32) - 1;      // of a launch, in a dimension

static int check(const hipadj_recurrence* r) {
    if (!r || r->struct_size != sizeof(hipadj_recurrence)) return ops_fail(HIPADJ_ERR_INVALID_ARG, "hipadj_recurrence.struct_size does not match this library");
    if (pair_of(r->dtype, r->gate_dtype) < 0) return ops_fail(HIPADJ_ERR_UNSUPPORTED, "recurrence: x is F64, F32, BF16 or F16 and the gate of x's type, or F32 next to BF16 / F16");
    if (r->gate < HIPADJ_GATE_DECAY || r->gate > HIPADJ_GATE_SIGMOID) return ops_fail(HIPADJ_ERR_INVALID_ARG, "recurrence: gate must be a hipadj_gate, got %d", r->gate);
    if (r->batch < 0 || r->length < 0 || r->channels < 0 || r->nseq < 0) return ops_fail(HIPADJ_ERR_INVALID_ARG, "recurrence: negative size");
    if (r->nseq > 0 && (r->batch != 1 || !r->offsets)) return ops_fail(HIPADJ_ERR_INVALID_ARG, "recurrence: packed sequences (nseq > 0) need batch = 1 and offsets[nseq + 1]");
    if (r->nseq > 0 && r->offsets_bits != 32 && r->offsets_bits != 64) return ops_fail(HIPADJ_ERR_INVALID_ARG, "recurrence: offsets_bits must be 32 or 64");
    const int64_t ntiles = tiles_of(r, true);
    const int64_t chains = r->channels / 64 + (r->channels % 64 != 0);
    if (r->batch && chains && ntiles > ((int64_t(1) << 31) - 1) / chains / r->batch) return ops_fail(HIPADJ_ERR_UNSUPPORTED, "recurrence: more than 2^31 - 1 tiles");
    return HIPADJ_OK;
}

static bool fits(const void* p, const int64_t* st, int64_t bytes, int64_t V) {
    return !p || (((uintptr_t)p % (uintptr_t)(bytes * V)) == 0 && st[0] % V == 0 && st[1] % V == 0);
}

static int go(const hipadj_recurrence* r, Args& a, bool adjoint, void* workspace, int64_t workspace_bytes, void* stream) {
    const int pair = pair_of(r->dtype, r->gate_dtype);
    const int64_t xb = size_of(r->dtype), gb = size_of(r->gate_dtype), VW = xb == 2 ? 2 : 1;
    const int64_t ntiles = tiles_of(r, adjoint);
    // V neighbouring channels a lane where every row starts on a multiple of V elements; else one (odd channel counts, sliced inputs)
    const bool wide = VW == 1 || (r->channels % VW == 0 && fits(a.x, r->x_stride, xb, VW) && fits(a.gate, r->gate_stride, gb, VW) &&
                                  (adjoint ? fits(a.dh, r->dh_stride, xb, VW) && fits(a.dx, r->dx_stride, xb, VW) && fits(a.dgate, r->dgate_stride, gb, VW)
                                           : fits(a.h, r->h_stride, xb, VW)));
    const int V = wide ? (int)VW : 1;
    a.x_sb = r->x_stride[0]; a.x_st = r->x_stride[1]; a.g_sb = r->gate_stride[0]; a.g_st = r->gate_stride[1]; a.h_sb = r->h_stride[0]; a.h_st = r->h_stride[1];
    a.dh_sb = r->dh_stride[0]; a.dh_st = r->dh_stride[1]; a.dx_sb = r->dx_stride[0]; a.dx_st = r->dx_stride[1]; a.dg_sb = r->dgate_stride[0]; a.dg_st = r->dgate_stride[1];
    a.L = r->length; a.D = r->channels; a.nseq = r->nseq; a.offsets = r->offsets; a.offsets64 = r->offsets_bits == 64;
    a.ntiles = (int)ntiles; a.nckpt = (int)tiles_of(r, true); a.ncg = (int)((r->channels + 64 * V - 1) / (64 * V)); a.nchains = (int)(r->batch * a.ncg); a.GS = group_of(a.nchains);
    if ((int64_t)a.ntiles * a.nchains > MOST_THREADS / NT)
        return ops_fail(HIPADJ_ERR_UNSUPPORTED, "recurrence: %lld tiles, a launch has at most %lld workgroups: fewer batch rows at a time", (long long)a.ntiles * a.nchains, (long long)(MOST_THREADS / NT));
    const int64_t words = words_of(r, ntiles, V);
    OpsDevice dev(r->device);
    if (dev.rc != HIPADJ_OK) return dev.rc;
    if (r->length == 0) {
        const int64_t n = (r->nseq ? r->nseq : r->batch) * r->channels;
        void* to = adjoint ? a.dh0 : a.h_final;
        const void* from = adjoint ? a.dh_final : a.h0;
        const dim3 grid((uint32_t)std::min<int64_t>(1024, (n + 255) / 256)), block(256);
        if (to && r->dtype == HIPADJ_F64) ops_launch(k_same<double>, grid, block, (hipStream_t)stream, (double*)to, (const double*)from, n);
        else if (to) ops_launch(k_same<float>, grid, block, (hipStream_t)stream, (float*)to, (const float*)from, n);
        return ops_launched("recurrence");
    }
    if (words) {
        if (!workspace || (uintptr_t)workspace % 8 || workspace_bytes < 8 * words)
            return ops_fail(HIPADJ_ERR_INVALID_ARG, "recurrence: %lld rows need a workspace of %lld bytes (hipadj_recurrence_sizes), 8-byte aligned", (long long)r->length, (long long)(8 * words));
        uint64_t* w = (uint64_t*)workspace;
        const int64_t W = r->dtype == HIPADJ_F64 ? WPM<double> : WPM<float>;
        a.ticket = (uint32_t*)w; a.agg = w + 1; a.car = a.agg + (int64_t)a.nchains * a.ntiles * W * 64 * V;
        ops_launch(k_zero, dim3((uint32_t)std::min<int64_t>(1024, (words + 255) / 256)), dim3(256), (hipStream_t)stream, w, words);
    }
    run(pair, a, adjoint, wide, r->gate, r->coupled != 0, r->nseq > 0, (hipStream_t)stream);
    return ops_launched("recurrence");
}

}  // namespace rec

extern "C" int hipadj_recurrence_sizes(const hipadj_recurrence* r, int64_t* checkpoint_bytes, int64_t* workspace_bytes) {
    const int rc = rec::check(r);
    if (rc != HIPADJ_OK) return rc;
    const int64_t ntiles = rec::tiles_of(r, true);            // the adjoint's tiles are the smaller ones: its words suffice for the forward pass
    if (checkpoint_bytes) *checkpoint_bytes = r->batch * ntiles * r->channels * (r->dtype == HIPADJ_F64 ? 8 : 4);
    if (workspace_bytes) *workspace_bytes = 8 * std::max(rec::words_of(r, ntiles, 1), rec::words_of(r, ntiles, 2));
    return HIPADJ_OK;
}

extern "C" int hipadj_recurrence_forward_dev(const hipadj_recurrence* r, const void* x, const void* gate, const void* h0, void* h, void* h_final, void* checkpoints,
                                             void* workspace, int64_t workspace_bytes, void* stream) {
    const int rc = rec::check(r);
    if (rc != HIPADJ_OK) return rc;
    if (r->channels == 0 || (r->nseq == 0 && r->batch == 0)) return HIPADJ_OK;
    if (!h_final || (r->length > 0 && (!x || !gate || !h))) return ops_fail(HIPADJ_ERR_INVALID_ARG, "hipadj_recurrence_forward_dev: x, gate, h and h_final are required");
    rec::Args a{};
    a.x = x; a.gate = gate; a.h0 = h0; a.h = h; a.h_final = h_final; a.ckpt = checkpoints;
    return rec::go(r, a, false, workspace, workspace_bytes, stream);
}

extern "C" int hipadj_recurrence_adjoint_dev(const hipadj_recurrence* r, const void* x, const void* gate, const void* h0, const void* checkpoints, const void* dh, const void* dh_final,
                                             void* dx, void* dgate, void* dh0, void* workspace, int64_t workspace_bytes, void* stream) {
    const int rc = rec::check(r);
    if (rc != HIPADJ_OK) return rc;
    if (r->channels == 0 || (r->nseq == 0 && r->batch == 0)) return HIPADJ_OK;
    if (r->length > 0 && (!checkpoints || !x || !gate)) return ops_fail(HIPADJ_ERR_INVALID_ARG, "hipadj_recurrence_adjoint_dev: x, gate and the forward pass's checkpoints are required");
    rec::Args a{};
    a.x = x; a.gate = gate; a.h0 = h0; a.ckpt = const_cast<void*>(checkpoints); a.dh = dh; a.dh_final = dh_final; a.dx = dx; a.dgate = dgate; a.dh0 = dh0;
    return rec::go(r, a, true, workspace, workspace_bytes, stream);
}

extern "C" int hipadj_recurrence_step_dev(int32_t device, int32_t dtype, int32_t gate_dtype, int32_t gate_form, int32_t coupled, int64_t batch, int64_t channels, const void* x,
                                          int64_t x_stride, const void* gate, int64_t gate_stride, void* state, int64_t state_stride, int64_t nslots, const void* slots,
                                          int32_t slots_bits, void* h, int64_t h_stride, void* stream) {
    const int pair = rec::pair_of(dtype, gate_dtype);
    if (pair < 0) return ops_fail(HIPADJ_ERR_UNSUPPORTED, "recurrence step: x is F64, F32, BF16 or F16 and the gate of x's type, or F32 next to BF16 / F16");
    if (gate_form < HIPADJ_GATE_DECAY || gate_form > HIPADJ_GATE_SIGMOID) return ops_fail(HIPADJ_ERR_INVALID_ARG, "recurrence step: gate must be a hipadj_gate, got %d", gate_form);
    if (batch < 0 || channels < 0 || nslots < 0) return ops_fail(HIPADJ_ERR_INVALID_ARG, "recurrence step: negative size");
    if (batch == 0 || channels == 0) return HIPADJ_OK;
    if (!x || !gate || !h || (!state && nslots > 0)) return ops_fail(HIPADJ_ERR_INVALID_ARG, "hipadj_recurrence_step_dev: x, gate, state and h are required");
    if (slots && slots_bits != 32 && slots_bits != 64) return ops_fail(HIPADJ_ERR_INVALID_ARG, "recurrence step: slots_bits must be 32 or 64");
    if (!slots && nslots < batch) return ops_fail(HIPADJ_ERR_INVALID_ARG, "recurrence step: %lld rows without slots need as many states, got %lld", (long long)batch, (long long)nslots);
    const int64_t xb = rec::size_of(dtype), gb = rec::size_of(gate_dtype), sb = dtype == HIPADJ_F64 ? 8 : 4, VW = xb == 2 ? 2 : 1;
    auto fits = [&](const void* p, int64_t st, int64_t bytes) { return (uintptr_t)p % (uintptr_t)(bytes * VW) == 0 && st % VW == 0; };
    const bool wide = VW == 1 || (channels % VW == 0 && fits(x, x_stride, xb) && fits(gate, gate_stride, gb) && fits(h, h_stride, xb) && fits(state, state_stride, sb));
    if (batch > rec::MOST_THREADS / rec::NS / ((channels + rec::NS * (wide ? VW : 1) - 1) / (rec::NS * (wide ? VW : 1))))
        return ops_fail(HIPADJ_ERR_UNSUPPORTED, "recurrence step: %lld rows of %lld channels, a launch has at most %lld workgroups", (long long)batch, (long long)channels, (long long)(rec::MOST_THREADS / rec::NS));
    rec::StepArgs a{x, gate, slots, state, h, x_stride, gate_stride, state_stride, h_stride, batch, channels, nslots, slots_bits == 64};
    OpsDevice dev(device);
    if (dev.rc != HIPADJ_OK) return dev.rc;
    hipStream_t s = (hipStream_t)stream;
    switch (pair) {
    case rec::PAIR_F64: rec::launch_step<rec::PAIR_F64>(a, wide, gate_form, coupled != 0, s); break;
    case rec::PAIR_F32: rec::launch_step<rec::PAIR_F32>(a, wide, gate_form, coupled != 0, s); break;
    case rec::PAIR_BF16: rec::launch_step<rec::PAIR_BF16>(a, wide, gate_form, coupled != 0, s); break;
    case rec::PAIR_BF16_F32: rec::launch_step<rec::PAIR_BF16_F32>(a, wide, gate_form, coupled != 0, s); break;
    case rec::PAIR_F16: rec::launch_step<rec::PAIR_F16>(a, wide, gate_form, coupled != 0, s); break;
    default: rec::launch_step<rec::PAIR_F16_F32>(a, wide, gate_form, coupled != 0, s); break;
    }
    return ops_launched("recurrence step");
}
#endif
