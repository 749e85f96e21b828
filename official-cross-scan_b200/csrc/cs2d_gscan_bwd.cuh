// Gated scan, backward.  See cs2d_gscan.cuh.
//
//   dh[t] = dy[t] + e[t+1]   e[t] = a[t] dh[t]   du = dh c (weighted) or dh   da = dh (h[t-1] - u) or dh h[t-1]   dgate = da * da/dgate
//
// e is the same kind of recurrence against the rows' order.  h[t-1] is made again from the checkpoint before the tile (4 bytes per
// channel and GS_CK rows instead of reading the rounded y), by maps that are composed between the same two barriers.
#pragma once

#include "cs2d_gscan.cuh"

namespace cs2d {

namespace gs {

template <int DT> constexpr int BTW = DT == CS2D_F32 ? 4 : 8;   // rows of a slot
constexpr int BSTAGES = 2;  // tiles of a warp that are on their way

template <int DT, int G> size_t bwd_smem() {
    return (size_t)NW * (3 * BSTAGES + 2) * Place<DT, G, BTW<DT>>::TB + 4 * NW * sizeof(MapStore<G>) + sizeof(Exchange<G>);
}

template <int DT, int G, int FORM, bool WEIGHTED, bool PACKED>
__global__ void __launch_bounds__(32 * NW, 2) gscan_bwd(const GScan P, const int wt, const int C) {
    using At = Place<DT, G, BTW<DT>>;
    using T = typename At::T;
    using M = Map<FORM != CS2D_GATE_SIGMOID, PACKED>;
    constexpr bool FULL = DT == CS2D_F32, GROWS = FORM != CS2D_GATE_SIGMOID;
    constexpr int TW = BTW<DT>, TB = At::TB, WB = (3 * BSTAGES + 2) * TB;   // bytes of a tile; of a warp's tiles: u, gate and dy on their way, du, dgate
    constexpr int BETWEEN = GS_CK / At::ROWS;   // warps from one checkpoint to the next
    static_assert(GS_CK % At::ROWS == 0 && NW % BETWEEN == 0, "a checkpoint lies before a warp's rows");
    extern __shared__ __align__(16) unsigned char smem[];
    MapStore<G> *agg = (MapStore<G> *)(smem + NW * WB), *agf = agg + 2 * NW;
    Exchange<G> *ex = (Exchange<G> *)(agf + 2 * NW);
    const int rank = C > 1 ? (int)(blockIdx.x % C) : 0;
    const At at(P, wt, (int)(blockIdx.x / C));
    const int warp = at.warp, first = warp - at.wi;
    unsigned char *ring = smem + warp * WB, *ut = ring + 3 * BSTAGES * TB, *gt = ut + TB;
    const int L = at.rows, tile = wt * At::ROWS, span = tile * C;
    float2 state = both(0.f);   // what comes from the rows behind the cluster's
    if (!PACKED && P.dlast) state = ld2(P.dlast + at.b * P.dlast_bs + at.ch, at.one, at.two);
    if constexpr (PACKED)
        if (P.dh0) empty_sequences(P, at, rank * wt + at.wi, wt * C, P.dlast, P.dlast_bs, P.dh0, false);
    if (C > 1) exchange_init<PACKED>(ex, C);

    const int last = ((int)P.length - 1) / span * span, w_last = last + rank * tile + at.wi * At::ROWS;   // of the cluster; of the warp
    Walk<DT, G, TW> u(P.u, P.u_bs, P.u_ls, at, w_last, -span), gate(P.gate, P.g_bs, P.g_ls, at, w_last, -span), dy(P.dy, P.dy_bs, P.dy_ls, at, w_last, -span);
    Walk<DT, G, TW> du(P.du, P.y_bs, P.y_ls, at, w_last, -span), dgate(P.dgate, P.y_bs, P.y_ls, at, w_last, -span);
    auto copy = [&](int w0, int stage) {
        if (w0 >= 0) {
            const int n = at.there(w0, At::ROWS);
            unsigned char *d = ring + stage * 3 * TB;
            u.fetch(d, n, at, P.dim, P.io);
            gate.fetch(d + TB, n, at, P.dim, P.io);
            dy.fetch(d + 2 * TB, n, at, P.dim, P.io);
            u.next();
            gate.next();
            dy.next();
        }
        copies_commit();
    };
    float2 hc;
    Marks<G, TW> marks;
    auto before_rows = [&](int w0) {   // the state before the warp's rows (the last checkpoint before them), and what starts and ends at the slot's
        hc = both(0.f);
        const int cb = w0 < 0 ? -1 : w0 / GS_CK;
        if (cb > 0 && cb * GS_CK < L) hc = ld2(P.ckpt + ((int64_t)at.b * P.nck + cb - 1) * P.dim + at.ch, at.one, at.two);
        if (!PACKED && cb == 0 && P.h0) hc = ld2(P.h0 + at.b * P.h0_bs + at.ch, at.one, at.two);
        if constexpr (PACKED) marks.load(P, w0 < 0 ? -TW : w0 + at.sub * TW, at.li, L);
    };
#pragma unroll
    for (int s = 0; s < BSTAGES; ++s) copy(w_last - s * span, s);
    before_rows(w_last);
    int stage = 0;
    unsigned step = 0;
    for (int w0 = w_last; w0 >= 0; w0 -= span, ++step) {   // (all warps of a cluster take as many steps)
        const int t0 = w0 + at.sub * TW;
        const int n = at.there(t0, TW);
        float2 h = hc;
        unsigned starts = 0, ends = 0;
        if constexpr (PACKED) marks.masks(at.sub, starts, ends);
        before_rows(w0 - span);
        copies_wait<BSTAGES - 1>();
        __syncwarp();
        const unsigned char *xu = ring + stage * 3 * TB, *xg = xu + TB, *xd = xg + TB;
        float2 a[TW], c[TW], x[TW], dh[TW];
#pragma unroll
        for (int i = 0; i < TW; ++i) {
            const float2 g = at.staged(xg, i);
            gate_values<FORM, FULL>(g.x, a[i].x, c[i].x);
            gate_values<FORM, FULL>(g.y, a[i].y, c[i].y);
            x[i] = at.staged(xu, i);
            dh[i] = at.staged(xd, i);
        }
        __syncwarp();
        copy(w0 - BSTAGES * span, stage);
        stage = stage + 1 == BSTAGES ? 0 : stage + 1;
        if (n < TW) {
#pragma unroll
            for (int i = 0; i < TW; ++i)
                if (i >= n) a[i] = both(1.f);   // u and dy are zero there
        }
        auto starting = [&](int i) { return t0 + i < L ? P.map[t0 + i].x : (int)SEQ_OUTSIDE; };
        // the input term of a row; of a first row with what the state before it adds
        auto input = [&](int i) {
            float2 b = x[i];
            if (WEIGHTED) b = mul2(b, c[i]);
            if (PACKED && (starts >> i & 1)) {
                const int s = starting(i);
                if (s < 0) b = both(0.f);
                else if (P.h0) b = through<GROWS>(a[i], b, ld2(P.h0 + s * P.h0_bs + at.ch, at.one, at.two));
            }
            return b;
        };
        if (PACKED && ends && P.dlast) {   // the gradient of a last state arrives with its row's
#pragma unroll
            for (int i = 0; i < TW; ++i)
                if (ends >> i & 1) dh[i] = add2(dh[i], ld2(P.dlast + P.map[t0 + i].y * P.dlast_bs + at.ch, at.one, at.two));
        }
        M f, r;
#pragma unroll
        for (int i = 0; i < TW; ++i) {
            const float2 b = input(i);
            f.B = fma2(a[i], f.B, b);
            if (PACKED && (starts >> i & 1)) f.B = b;
            f.A = mul2(f.A, a[i]);
        }
#pragma unroll
        for (int i = TW - 1; i >= 0; --i) {
            r.B = mul2(a[i], add2(dh[i], r.B));
            if (PACKED && (starts >> i & 1)) r.B = both(0.f);
        }
        if (PACKED) __syncwarp();
        r.A = f.A;
        f.cut = r.cut = starts != 0;
        M before, behind;
        over_slots<G, GROWS, PACKED, false>(r, behind, at.lane);
        over_slots<G, GROWS, PACKED, true>(f, before, at.lane);
        MapStore<G> *maps = agg + (step & 1) * NW + first, *mapf = agf + (step & 1) * NW + first;   // two sets: a warp may be a tile ahead of the others' reading
        if (at.sub == 0) maps[at.wi].put(r, at.li);
        if (BETWEEN > 1 && at.sub == At::S - 1) mapf[at.wi].put(f, at.li);
        __syncthreads();
        float2 e = C > 1 ? pass_cluster<GROWS, PACKED, false>(maps, ex, step, rank, C, at, state, P.status)
                         : pass<GROWS, PACKED, false, NW>(maps, wt, at.wi, at.li, state);
        if (BETWEEN > 1) h = pass<GROWS, PACKED, true, BETWEEN>(mapf + at.wi / BETWEEN * BETWEEN, min(BETWEEN, wt), at.wi % BETWEEN, at.li, h);
        if (G < 32) {
            e = behind.apply(e);
            h = before.apply(h);
        }
        float2 hp[TW];
#pragma unroll
        for (int i = 0; i < TW; ++i) {
            const float2 b = input(i);
            hp[i] = h;
            h = fma2(a[i], h, b);
            if (PACKED && (starts >> i & 1)) {
                const int s = starting(i);
                hp[i] = s >= 0 && P.h0 ? ld2(P.h0 + s * P.h0_bs + at.ch, at.one, at.two) : both(0.f);
                h = b;
            }
        }
#pragma unroll
        for (int i = TW - 1; i >= 0; --i) {
            const float2 d = add2(dh[i], e);
            float2 ou = WEIGHTED ? mul2(d, c[i]) : d;
            float2 og = mul2(d, WEIGHTED ? sub2(hp[i], x[i]) : hp[i]);
            if (FORM == CS2D_GATE_SIGMOID) og = mul2(og, mul2(a[i], c[i]));
            if (FORM == CS2D_GATE_LOG) og = mul2(og, a[i]);
            e = mul2(a[i], d);
            if (PACKED && (starts >> i & 1)) {
                const int s = starting(i);
                if (s < 0) ou = og = both(0.f);
                else if (P.dh0) st2(P.dh0 + (int64_t)s * P.dim + at.ch, e, at.one, at.two);
                e = both(0.f);
            }
            at.stage(ut, i, ou);
            at.stage(gt, i, og);
        }
        __syncwarp();
        const int m = at.there(w0, At::ROWS);
        du.flush(ut, m, at, P.dim, P.io_out);
        dgate.flush(gt, m, at, P.dim, P.io_out);
        du.next();
        dgate.next();
        __syncwarp();
    }
    if (!PACKED && P.dh0 && rank == 0 && at.wi == 0 && at.sub == 0) st2(P.dh0 + (int64_t)at.b * P.dim + at.ch, state, at.one, at.two);
    if (C > 1) cg::this_cluster().sync();   // nobody writes to a CTA that has gone
}

template <int DT, int G, int FORM, bool WEIGHTED> cudaError_t bwd3(GScan P, cudaStream_t st) {
    constexpr int rows = Place<DT, G, BTW<DT>>::ROWS;
    return P.map ? start<gscan_bwd<DT, G, FORM, WEIGHTED, true>>(P, G, rows, bwd_smem<DT, G>(), st) : start<gscan_bwd<DT, G, FORM, WEIGHTED, false>>(P, G, rows, bwd_smem<DT, G>(), st);
}
template <int DT, int G> cudaError_t bwd2(const GScan &P, cudaStream_t st) {
    switch (P.form * 2 + P.weighted) {
        case CS2D_GATE_SIGMOID * 2: return bwd3<DT, G, CS2D_GATE_SIGMOID, false>(P, st);
        case CS2D_GATE_SIGMOID * 2 + 1: return bwd3<DT, G, CS2D_GATE_SIGMOID, true>(P, st);
        case CS2D_GATE_LOG * 2: return bwd3<DT, G, CS2D_GATE_LOG, false>(P, st);
        case CS2D_GATE_LOG * 2 + 1: return bwd3<DT, G, CS2D_GATE_LOG, true>(P, st);
        case CS2D_GATE_DIRECT * 2: return bwd3<DT, G, CS2D_GATE_DIRECT, false>(P, st);
        default: return bwd3<DT, G, CS2D_GATE_DIRECT, true>(P, st);
    }
}
template <int DT> cudaError_t bwd(const GScan &P, cudaStream_t st) { return narrow(P) ? bwd2<DT, 8>(P, st) : bwd2<DT, 32>(P, st); }

}  // namespace gs

}  // namespace cs2d
