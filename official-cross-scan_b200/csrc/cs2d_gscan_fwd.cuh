// Gated scan, forward.  See cs2d_gscan.cuh.
#pragma once

#include "cs2d_gscan.cuh"

namespace cs2d {

namespace gs {

template <int DT> constexpr int FTW = DT == CS2D_F32 ? 8 : 16;   // rows of a slot
constexpr int FSTAGES = 2;  // tiles of a warp that are on their way

template <int DT, int G> size_t fwd_smem() {
    return (size_t)NW * (2 * FSTAGES + 1) * Place<DT, G, FTW<DT>>::TB + 2 * NW * sizeof(MapStore<G>) + sizeof(Exchange<G>);
}

template <int DT, int G, int FORM, bool WEIGHTED, bool PACKED>
__global__ void __launch_bounds__(32 * NW, 2) gscan_fwd(const GScan P, const int wt, const int C) {
    using At = Place<DT, G, FTW<DT>>;
    using T = typename At::T;
    using M = Map<FORM != CS2D_GATE_SIGMOID, PACKED>;
    constexpr bool FULL = DT == CS2D_F32, GROWS = FORM != CS2D_GATE_SIGMOID;
    constexpr int TW = FTW<DT>, TB = At::TB, WB = (2 * FSTAGES + 1) * TB;   // bytes of a tile; of a warp's tiles: u and gate on their way, y
    extern __shared__ __align__(16) unsigned char smem[];
    MapStore<G> *agg = (MapStore<G> *)(smem + NW * WB);
    Exchange<G> *ex = (Exchange<G> *)(agg + 2 * NW);
    const int rank = C > 1 ? (int)(blockIdx.x % C) : 0;
    const At at(P, wt, (int)(blockIdx.x / C));
    const int warp = at.warp, first = warp - at.wi;
    unsigned char *ring = smem + warp * WB, *yt = ring + 2 * FSTAGES * TB;
    const int L = at.rows, tile = wt * At::ROWS, span = tile * C;
    float2 state = both(0.f);   // before the cluster's rows of this step
    if (!PACKED && P.h0) state = ld2(P.h0 + at.b * P.h0_bs + at.ch, at.one, at.two);
    if constexpr (PACKED) empty_sequences(P, at, rank * wt + at.wi, wt * C, P.h0, P.h0_bs, P.last, blockIdx.x < C && warp < wt);
    if (C > 1) exchange_init<PACKED>(ex, C);

    const int w_first = rank * tile + at.wi * At::ROWS;   // of the warp; its slots follow each other
    Walk<DT, G, TW> u(P.u, P.u_bs, P.u_ls, at, w_first, span), gate(P.gate, P.g_bs, P.g_ls, at, w_first, span), y(P.y, P.y_bs, P.y_ls, at, w_first, span);
    auto copy = [&](int w0, int stage) {
        const int n = at.there(w0, At::ROWS);
        u.fetch(ring + stage * 2 * TB, n, at, P.dim, P.io);
        gate.fetch(ring + stage * 2 * TB + TB, n, at, P.dim, P.io);
        u.next();
        gate.next();
        copies_commit();
    };
    Marks<G, TW> marks;
    if constexpr (PACKED) marks.load(P, w_first + at.sub * TW, at.li, L);
#pragma unroll
    for (int s = 0; s < FSTAGES; ++s) copy(w_first + s * span, s);
    int stage = 0;
    unsigned step = 0;
    for (int base = 0; base < (int)P.length; base += span, ++step) {
        const int w0 = base + w_first, t0 = w0 + at.sub * TW;   // the warp's and the slot's first row
        const int n = at.there(t0, TW);
        unsigned starts = 0, ends = 0;
        if constexpr (PACKED) {
            marks.masks(at.sub, starts, ends);
            marks.load(P, t0 + span, at.li, L);
        }
        copies_wait<FSTAGES - 1>();
        __syncwarp();
        const unsigned char *xu = ring + stage * 2 * TB, *xg = xu + TB;
        float2 a[TW], b[TW];
#pragma unroll
        for (int i = 0; i < TW; ++i) {
            const float2 g = at.staged(xg, i);
            float2 c;
            gate_values<FORM, FULL>(g.x, a[i].x, c.x);
            gate_values<FORM, FULL>(g.y, a[i].y, c.y);
            b[i] = at.staged(xu, i);
            if (WEIGHTED) b[i] = mul2(b[i], c);
        }
        __syncwarp();
        copy(w0 + FSTAGES * span, stage);
        stage = stage + 1 == FSTAGES ? 0 : stage + 1;
        if (n < TW) {
#pragma unroll
            for (int i = 0; i < TW; ++i)
                if (i >= n) { a[i] = both(1.f); b[i] = both(0.f); }
        }
        if constexpr (PACKED) {
            if (starts) {
#pragma unroll
                for (int i = 0; i < TW; ++i) {
                    if (!(starts >> i & 1)) continue;
                    const int s = t0 + i < L ? P.map[t0 + i].x : SEQ_OUTSIDE;
                    if (s < 0) b[i] = both(0.f);   // a row of no sequence
                    else if (P.h0) b[i] = through<GROWS>(a[i], b[i], ld2(P.h0 + s * P.h0_bs + at.ch, at.one, at.two));
                }
            }
            __syncwarp();
        }
        M m;
#pragma unroll
        for (int i = 0; i < TW; ++i) {
            m.B = fma2(a[i], m.B, b[i]);
            if (PACKED && (starts >> i & 1)) m.B = b[i];
            m.A = mul2(m.A, a[i]);
        }
        m.cut = starts != 0;
        M before;
        over_slots<G, GROWS, PACKED, true>(m, before, at.lane);
        MapStore<G> *maps = agg + (step & 1) * NW + first;   // two sets: a warp may be a tile ahead of the others' reading
        if (at.sub == At::S - 1) maps[at.wi].put(m, at.li);
        __syncthreads();
        float2 h = C > 1 ? pass_cluster<GROWS, PACKED, true>(maps, ex, step, rank, C, at, state, P.status)
                         : pass<GROWS, PACKED, true, NW>(maps, wt, at.wi, at.li, state);
        if (G < 32) h = before.apply(h);
#pragma unroll
        for (int i = 0; i < TW; ++i) {
            h = fma2(a[i], h, b[i]);
            if (PACKED && (starts >> i & 1)) h = b[i];
            at.stage(yt, i, h);
            if (PACKED && (ends >> i & 1)) st2(P.last + (int64_t)P.map[t0 + i].y * P.dim + at.ch, h, at.one, at.two);
            const int end = t0 + i + 1;
            if ((i + 1) % (TW < GS_CK ? TW : GS_CK) == 0 && P.ckpt && end % GS_CK == 0 && end < L)
                st2(P.ckpt + ((int64_t)at.b * P.nck + end / GS_CK - 1) * P.dim + at.ch, h, at.one, at.two);
        }
        __syncwarp();
        y.flush(yt, at.there(w0, At::ROWS), at, P.dim, P.io_out);
        y.next();
        __syncwarp();
    }
    if (!PACKED && rank == 0 && at.wi == 0 && at.sub == 0) st2(P.last + (int64_t)at.b * P.dim + at.ch, state, at.one, at.two);
    if (C > 1) cg::this_cluster().sync();   // nobody writes to a CTA that has gone
}

template <int DT, int G, int FORM, bool WEIGHTED> cudaError_t fwd3(GScan P, cudaStream_t st) {
    constexpr int rows = Place<DT, G, FTW<DT>>::ROWS;
    return P.map ? start<gscan_fwd<DT, G, FORM, WEIGHTED, true>>(P, G, rows, fwd_smem<DT, G>(), st) : start<gscan_fwd<DT, G, FORM, WEIGHTED, false>>(P, G, rows, fwd_smem<DT, G>(), st);
}
template <int DT, int G> cudaError_t fwd2(const GScan &P, cudaStream_t st) {
    switch (P.form * 2 + P.weighted) {
        case CS2D_GATE_SIGMOID * 2: return fwd3<DT, G, CS2D_GATE_SIGMOID, false>(P, st);
        case CS2D_GATE_SIGMOID * 2 + 1: return fwd3<DT, G, CS2D_GATE_SIGMOID, true>(P, st);
        case CS2D_GATE_LOG * 2: return fwd3<DT, G, CS2D_GATE_LOG, false>(P, st);
        case CS2D_GATE_LOG * 2 + 1: return fwd3<DT, G, CS2D_GATE_LOG, true>(P, st);
        case CS2D_GATE_DIRECT * 2: return fwd3<DT, G, CS2D_GATE_DIRECT, false>(P, st);
        default: return fwd3<DT, G, CS2D_GATE_DIRECT, true>(P, st);
    }
}
template <int DT> cudaError_t fwd(const GScan &P, cudaStream_t st) { return narrow(P) ? fwd2<DT, 8>(P, st) : fwd2<DT, 32>(P, st); }

}  // namespace gs

}  // namespace cs2d
