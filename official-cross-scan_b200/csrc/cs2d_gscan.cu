// Gated linear recurrence over tokens: h[t] = a[t] h[t-1] + b[t] per channel, forward, backward and one token.
//
// A run of rows maps the state before it to the state behind it by h -> A h + B, and such maps compose: a warp reduces its rows
// to (A, B), a CTA composes its warps' maps, and every warp then walks its rows again from the state that reaches it.  Lanes hold
// channels, so a row is one coalesced access, nothing is exchanged between lanes, and the walk itself is one fma per element in
// 32 bits.  The rows stay in registers between the two walks: every input is read once and every output written once.
#include "cs2d_seq.cuh"

namespace cs2d {

namespace {

constexpr int NT = GS_WARPS * 32;

// h -> A h + B.  A state of exactly zero meets products A that have overflowed (factors above one) and adds nothing.
__device__ __forceinline__ float through(float A, float B, float h) { return h == 0.f ? B : fmaf(A, h, B); }

// A warp's place: its rows' unit, time slot and channels.
template <int V> struct Place {
    int lane, warp, wt, wi, b, ch;
    bool on;          // the lane has channels
    __device__ __forceinline__ Place(const GScan &P, int wt_) {
        lane = threadIdx.x & 31; warp = threadIdx.x >> 5; wt = wt_;
        wi = warp % wt;
        const int64_t unit = (int64_t)blockIdx.x * (GS_WARPS / wt) + warp / wt;
        const int blk = (int)(unit % P.nblk);
        b = (int)(unit / P.nblk);
        ch = (blk * 32 + lane) * V;
        on = unit < P.units && ch < P.dim;
        if (!on) { ch = 0; b = 0; }   // addresses stay inside the tensors; nothing is read or written
    }
};

__device__ __forceinline__ int64_t offset_at(const GScan &P, int i) {
    return P.off64 ? ((const int64_t *)P.offsets)[i] : (int64_t)((const int32_t *)P.offsets)[i];
}

// Sequences without a row: their state passes through.  Also reports borders that are not ascending or leave the tensor.
template <int V>
__device__ __forceinline__ void empty_sequences(const GScan &P, const Place<V> &at, const float *in, int64_t in_s, float *out, bool report) {
    for (int s = at.wi; s < P.nseq; s += at.wt) {   // the warps of the unit share them
        const bool on = at.on;
        const int ch = at.ch;
        const int64_t lo = offset_at(P, s), hi = offset_at(P, s + 1);
        if (report && (lo < 0 || hi > P.length || hi < lo) && at.lane == 0) atomicOr(P.status, ERR_SEQ_OFFSETS);
        if (hi > lo || !on) continue;
        for (int v = 0; v < V; ++v) out[(int64_t)s * P.dim + ch + v] = in ? in[(int64_t)s * in_s + ch + v] : 0.f;
    }
}

// ---- forward -----------------------------------------------------------------------------------------------
template <int DT, int V, bool PACKED>
__global__ void __launch_bounds__(NT, 1) gscan_fwd(const GScan P, const int wt) {
    using Pk = Pack<DT, V>;
    using W = typename Pk::W;
    using T = typename Pk::T;
    constexpr bool FULL = DT == CS2D_F32;
    constexpr int TW = GS_TW;
    __shared__ float2 agg[GS_WARPS][V][32], pre[GS_WARPS][V][32];   // maps of the warps' rows; of the rows before them in the tile
    __shared__ int cut[GS_WARPS], cut_pre[GS_WARPS], cut_all[GS_WARPS];   // a sequence starts in them: the state before ends there
    __shared__ float2 whole[GS_WARPS][V][32];
    const Place<V> at(P, wt);
    const int lane = at.lane, warp = at.warp, wi = at.wi;
    const int64_t L = P.length, tile = (int64_t)wt * TW;
    const T *u = (const T *)P.u + at.b * P.u_bs + at.ch, *gate = (const T *)P.gate + at.b * P.g_bs + at.ch;
    T *y = (T *)P.y + at.b * P.y_bs + at.ch;
    float h0[V];
#pragma unroll
    for (int v = 0; v < V; ++v) h0[v] = !PACKED && P.h0 && at.on ? P.h0[at.b * P.h0_bs + at.ch + v] : 0.f;
    if constexpr (PACKED) empty_sequences(P, at, P.h0, P.h0_bs, P.last, blockIdx.x == 0 && warp < wt);

    W ru[TW], rg[TW];
    int code = 0;
    auto load = [&](int64_t t0) {
        const int n = at.on ? (int)max((int64_t)0, min(L - t0, (int64_t)TW)) : 0;
#pragma unroll
        for (int i = 0; i < TW; ++i) {
            ru[i] = i < n ? *(const W *)(u + (t0 + i) * P.u_ls) : W{};
            rg[i] = i < n ? *(const W *)(gate + (t0 + i) * P.g_ls) : W{};
        }
        if constexpr (PACKED) {
            const int64_t t = t0 + (lane & (TW - 1));
            code = SEQ_OUTSIDE;
            if (t < L) code = lane < TW ? P.map[t].x : P.map[t].y;
        }
    };
    load((int64_t)wi * TW);
    for (int64_t base = 0; base < L; base += tile) {
        const int64_t t0 = base + (int64_t)wi * TW;
        const int n = (int)max((int64_t)0, min(L - t0, (int64_t)TW));
        float a[TW][V], b[TW][V];
        unsigned starts = 0, ends = 0;
        const int now = code;
        if constexpr (PACKED) {
            starts = __ballot_sync(~0u, lane < TW && code != SEQ_NONE);
            ends = __ballot_sync(~0u, lane >= TW && code >= 0) >> TW;
        }
        auto values = [&](auto form) {
#pragma unroll
            for (int i = 0; i < TW; ++i) {
                float x[V], g[V];
                Pk::up(ru[i], x);
                Pk::up(rg[i], g);
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    float c;
                    gate_values<decltype(form)::value, FULL>(g[v], a[i][v], c);
                    b[i][v] = P.weighted ? c * x[v] : x[v];
                }
            }
        };
        switch (P.form) {
            case CS2D_GATE_SIGMOID: values(std::integral_constant<int, CS2D_GATE_SIGMOID>{}); break;
            case CS2D_GATE_LOG: values(std::integral_constant<int, CS2D_GATE_LOG>{}); break;
            default: values(std::integral_constant<int, CS2D_GATE_DIRECT>{});
        }
        load(t0 + tile);   // the next tile's rows arrive while this one is worked on
        if constexpr (PACKED) {
#pragma unroll
            for (int i = 0; i < TW; ++i) {
                if (!(starts >> i & 1)) continue;
                const int s = __shfl_sync(~0u, now, i);
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    if (s < 0) b[i][v] = 0.f;   // a row of no sequence
                    else if (P.h0 && at.on) b[i][v] = through(a[i][v], b[i][v], P.h0[s * P.h0_bs + at.ch + v]);
                }
            }
        }
        float A[V], B[V];
#pragma unroll
        for (int v = 0; v < V; ++v) { A[v] = 1.f; B[v] = 0.f; }
#pragma unroll
        for (int i = 0; i < TW; ++i) {
            const bool cuts = PACKED && (starts >> i & 1);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                if (i < n) {
                    B[v] = cuts ? b[i][v] : fmaf(a[i][v], B[v], b[i][v]);
                    A[v] *= a[i][v];
                }
            }
        }
#pragma unroll
        for (int v = 0; v < V; ++v) agg[warp][v][lane] = make_float2(A[v], B[v]);
        if (PACKED && lane == 0) cut[warp] = starts != 0;
        __syncthreads();
        if (wi == 0) {   // the maps of the rows before each warp's, then of the whole tile
            float pA[V], pB[V];
            int c = 0;
#pragma unroll
            for (int v = 0; v < V; ++v) { pA[v] = 1.f; pB[v] = 0.f; }
            for (int k = 0; k < wt; ++k) {
                const int cw = PACKED ? cut[warp + k] : 0;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float2 m = agg[warp + k][v][lane];
                    pre[warp + k][v][lane] = make_float2(pA[v], pB[v]);
                    pB[v] = cw ? m.y : through(m.x, m.y, pB[v]);
                    pA[v] *= m.x;
                }
                if (PACKED && lane == 0) cut_pre[warp + k] = c;
                c |= cw;
            }
#pragma unroll
            for (int v = 0; v < V; ++v) whole[warp][v][lane] = make_float2(pA[v], pB[v]);
            if (PACKED && lane == 0) cut_all[warp] = c;
        }
        __syncthreads();
        float h[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const float2 m = pre[warp][v][lane], all = whole[warp - wi][v][lane];
            const int cp = PACKED ? cut_pre[warp] : 0, ca = PACKED ? cut_all[warp - wi] : 0;
            h[v] = cp ? m.y : through(m.x, m.y, h0[v]);
            h0[v] = ca ? all.y : through(all.x, all.y, h0[v]);
        }
#pragma unroll
        for (int i = 0; i < TW; ++i) {
            const bool cuts = PACKED && (starts >> i & 1);
            if (i < n) {
#pragma unroll
                for (int v = 0; v < V; ++v) h[v] = cuts ? b[i][v] : fmaf(a[i][v], h[v], b[i][v]);
                if (at.on) *(W *)(y + (t0 + i) * P.y_ls) = Pk::down(h);
                if (PACKED && (ends >> i & 1)) {
                    const int s = __shfl_sync(~0u, now, TW + i);
                    if (at.on)
#pragma unroll
                        for (int v = 0; v < V; ++v) P.last[(int64_t)s * P.dim + at.ch + v] = h[v];
                }
            }
        }
        const int64_t end = t0 + TW;   // the backward's tiles begin at multiples of GS_CK
        if (P.ckpt && at.on && end % GS_CK == 0 && end < L) {
            float *ck = P.ckpt + ((int64_t)at.b * P.nck + end / GS_CK - 1) * P.dim + at.ch;
#pragma unroll
            for (int v = 0; v < V; ++v) ck[v] = h[v];
        }
        __syncthreads();   // pre and agg are written again
    }
    if (!PACKED && wi == 0 && at.on)
#pragma unroll
        for (int v = 0; v < V; ++v) P.last[(int64_t)at.b * P.dim + at.ch + v] = h0[v];
}

// ---- backward ----------------------------------------------------------------------------------------------
// e[t] = a[t] dh[t], dh[t] = dy[t] + e[t+1]: the same kind of recurrence against the rows' order, and h[t-1] again from the
// checkpoint before the tile.  Both walks compose their maps over the warps between the same two barriers.
template <int DT, int V, bool PACKED>
__global__ void __launch_bounds__(NT, 1) gscan_bwd(const GScan P, const int wt) {
    using Pk = Pack<DT, V>;
    using W = typename Pk::W;
    using T = typename Pk::T;
    constexpr bool FULL = DT == CS2D_F32;
    constexpr int TW = GS_TWB;
    __shared__ float agg[GS_WARPS][3][V][32];    // A, the forward's B, the backward's E of the warps' rows
    __shared__ float hs[GS_WARPS][V][32];        // the state before the warps' rows
    __shared__ float2 suf[GS_WARPS][V][32];      // the backward's map of the rows behind them in the tile
    __shared__ float2 whole[GS_WARPS][V][32];    // and of the tile
    __shared__ int cut[GS_WARPS], cut_suf[GS_WARPS], cut_all[GS_WARPS];
    const Place<V> at(P, wt);
    const int lane = at.lane, warp = at.warp, wi = at.wi;
    const int64_t L = P.length, tile = (int64_t)wt * TW;
    const T *u = (const T *)P.u + at.b * P.u_bs + at.ch, *gate = (const T *)P.gate + at.b * P.g_bs + at.ch;
    const T *dy = (const T *)P.dy + at.b * P.dy_bs + at.ch;
    T *du = (T *)P.du + at.b * P.y_bs + at.ch, *dgate = (T *)P.dgate + at.b * P.y_bs + at.ch;
    float e0[V];   // what comes from the rows behind the tile
#pragma unroll
    for (int v = 0; v < V; ++v) e0[v] = !PACKED && P.dlast && at.on ? P.dlast[at.b * P.dlast_bs + at.ch + v] : 0.f;
    if constexpr (PACKED)
        if (P.dh0) empty_sequences(P, at, P.dlast, P.dlast_bs, P.dh0, false);

    W ru[TW], rg[TW], rd[TW];
    float hc[V];
    int code = 0;
    auto load = [&](int64_t t0, int64_t base) {
        const int n = at.on && base >= 0 ? (int)max((int64_t)0, min(L - t0, (int64_t)TW)) : 0;
#pragma unroll
        for (int i = 0; i < TW; ++i) {
            ru[i] = i < n ? *(const W *)(u + (t0 + i) * P.u_ls) : W{};
            rg[i] = i < n ? *(const W *)(gate + (t0 + i) * P.g_ls) : W{};
            rd[i] = i < n ? *(const W *)(dy + (t0 + i) * P.dy_ls) : W{};
        }
        if (wi == 0 && at.on && base >= 0) {
#pragma unroll
            for (int v = 0; v < V; ++v)
                hc[v] = base > 0 ? P.ckpt[((int64_t)at.b * P.nck + base / GS_CK - 1) * P.dim + at.ch + v]
                                 : !PACKED && P.h0 ? P.h0[at.b * P.h0_bs + at.ch + v] : 0.f;
        }
        if constexpr (PACKED) {
            const int64_t t = t0 + (lane & (TW - 1));
            code = SEQ_OUTSIDE;
            if (base >= 0 && t < L) code = lane < TW ? P.map[t].x : P.map[t].y;
        }
    };
#pragma unroll
    for (int v = 0; v < V; ++v) hc[v] = 0.f;
    int64_t base = (L - 1) / tile * tile;
    load(base + (int64_t)wi * TW, base);
    for (; base >= 0; base -= tile) {
        const int64_t t0 = base + (int64_t)wi * TW;
        const int n = (int)max((int64_t)0, min(L - t0, (int64_t)TW));
        float a[TW][V], c[TW][V], dh[TW][V];
        W x[TW];
        unsigned starts = 0, ends = 0;
        const int now = code;
        float hnow[V];
#pragma unroll
        for (int v = 0; v < V; ++v) hnow[v] = hc[v];
        if constexpr (PACKED) {
            starts = __ballot_sync(~0u, lane < TW && code != SEQ_NONE);
            ends = __ballot_sync(~0u, lane >= TW && lane < 2 * TW && code >= 0) >> TW;
        }
        auto values = [&](auto form) {
#pragma unroll
            for (int i = 0; i < TW; ++i) {
                float g[V];
                Pk::up(rg[i], g);
                Pk::up(rd[i], dh[i]);
                x[i] = ru[i];
#pragma unroll
                for (int v = 0; v < V; ++v) gate_values<decltype(form)::value, FULL>(g[v], a[i][v], c[i][v]);
            }
        };
        switch (P.form) {
            case CS2D_GATE_SIGMOID: values(std::integral_constant<int, CS2D_GATE_SIGMOID>{}); break;
            case CS2D_GATE_LOG: values(std::integral_constant<int, CS2D_GATE_LOG>{}); break;
            default: values(std::integral_constant<int, CS2D_GATE_DIRECT>{});
        }
        load(t0 - tile, base - tile);
        if constexpr (PACKED) {
#pragma unroll
            for (int i = 0; i < TW; ++i) {
                if ((ends >> i & 1) && P.dlast) {
                    const int s = __shfl_sync(~0u, now, TW + i);
#pragma unroll
                    for (int v = 0; v < V; ++v)
                        if (at.on) dh[i][v] += P.dlast[s * P.dlast_bs + at.ch + v];
                }
            }
        }
        // the state before a first row (packed), and the input term
        auto first_state = [&](int i, int v) {
            const int s = __shfl_sync(~0u, now, i);
            return s >= 0 && P.h0 && at.on ? P.h0[s * P.h0_bs + at.ch + v] : 0.f;
        };
        auto input = [&](int i, float (&b)[V]) {
            Pk::up(x[i], b);
            if (P.weighted)
#pragma unroll
                for (int v = 0; v < V; ++v) b[v] *= c[i][v];
        };
        auto outside = [&](int i) { return __shfl_sync(~0u, now, i) == SEQ_OUTSIDE; };
        float A[V], B[V], E[V];
#pragma unroll
        for (int v = 0; v < V; ++v) { A[v] = 1.f; B[v] = 0.f; E[v] = 0.f; }
#pragma unroll
        for (int i = 0; i < TW; ++i) {
            float b[V];
            input(i, b);
            if (PACKED && (starts >> i & 1)) {
                const bool none = outside(i);
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float hf = first_state(i, v);
                    B[v] = none ? 0.f : through(a[i][v], b[v], hf);
                }
            } else if (i < n) {
#pragma unroll
                for (int v = 0; v < V; ++v) { B[v] = fmaf(a[i][v], B[v], b[v]); A[v] *= a[i][v]; }
            }
        }
#pragma unroll
        for (int i = TW - 1; i >= 0; --i) {
            if (PACKED && (starts >> i & 1)) {
#pragma unroll
                for (int v = 0; v < V; ++v) E[v] = 0.f;
            } else if (i < n) {
#pragma unroll
                for (int v = 0; v < V; ++v) E[v] = a[i][v] * (dh[i][v] + E[v]);
            }
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
            agg[warp][0][v][lane] = A[v]; agg[warp][1][v][lane] = B[v]; agg[warp][2][v][lane] = E[v];
        }
        if (PACKED && lane == 0) cut[warp] = starts != 0;
        __syncthreads();
        if (wi == 0) {   // states before the warps' rows
            float h[V];
#pragma unroll
            for (int v = 0; v < V; ++v) h[v] = hnow[v];
            for (int k = 0; k < wt; ++k) {
                const int cw = PACKED ? cut[warp + k] : 0;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    hs[warp + k][v][lane] = h[v];
                    const float mB = agg[warp + k][1][v][lane];
                    h[v] = cw ? mB : through(agg[warp + k][0][v][lane], mB, h[v]);
                }
            }
        }
        if (wi == wt - 1) {   // maps of the rows behind them, then of the whole tile
            float pA[V], pE[V];
            int cc = 0;
#pragma unroll
            for (int v = 0; v < V; ++v) { pA[v] = 1.f; pE[v] = 0.f; }
            for (int k = warp; k > warp - wt; --k) {
                const int cw = PACKED ? cut[k] : 0;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    suf[k][v][lane] = make_float2(pA[v], pE[v]);
                    const float mA = agg[k][0][v][lane], mE = agg[k][2][v][lane];
                    pE[v] = cw ? mE : through(mA, mE, pE[v]);
                    pA[v] *= mA;
                }
                if (PACKED && lane == 0) cut_suf[k] = cc;
                cc |= cw;
            }
#pragma unroll
            for (int v = 0; v < V; ++v) whole[warp][v][lane] = make_float2(pA[v], pE[v]);
            if (PACKED && lane == 0) cut_all[warp] = cc;
        }
        __syncthreads();
        float h[V], e[V], hp[TW][V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const float2 m = suf[warp][v][lane], all = whole[warp - wi + wt - 1][v][lane];
            const int cs = PACKED ? cut_suf[warp] : 0, ca = PACKED ? cut_all[warp - wi + wt - 1] : 0;
            h[v] = hs[warp][v][lane];
            e[v] = cs ? m.y : through(m.x, m.y, e0[v]);
            e0[v] = ca ? all.y : through(all.x, all.y, e0[v]);
        }
#pragma unroll
        for (int i = 0; i < TW; ++i) {
            float b[V];
            input(i, b);
            const bool cuts = PACKED && (starts >> i & 1), none = cuts && outside(i);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                if (cuts) h[v] = first_state(i, v);
                hp[i][v] = h[v];
                h[v] = none ? 0.f : cuts ? through(a[i][v], b[v], h[v]) : fmaf(a[i][v], h[v], b[v]);
            }
        }
#pragma unroll
        for (int i = TW - 1; i >= 0; --i) {
            if (i >= n) continue;
            const bool cuts = PACKED && (starts >> i & 1);
            const int s = cuts ? __shfl_sync(~0u, now, i) : SEQ_NONE;
            float xv[V], ou[V], og[V];
            Pk::up(x[i], xv);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float d = dh[i][v] + e[v];
                const float slope = P.form == CS2D_GATE_SIGMOID ? a[i][v] * c[i][v] : P.form == CS2D_GATE_LOG ? a[i][v] : 1.f;
                ou[v] = P.weighted ? d * c[i][v] : d;
                og[v] = d * (P.weighted ? hp[i][v] - xv[v] : hp[i][v]) * slope;
                e[v] = a[i][v] * d;
                if (s == SEQ_OUTSIDE) ou[v] = og[v] = 0.f;
                if (s >= 0 && P.dh0 && at.on) P.dh0[(int64_t)s * P.dim + at.ch + v] = e[v];
                if (cuts) e[v] = 0.f;
            }
            if (at.on) {
                *(W *)(du + (t0 + i) * P.y_ls) = Pk::down(ou);
                *(W *)(dgate + (t0 + i) * P.y_ls) = Pk::down(og);
            }
        }
        __syncthreads();
    }
    if (!PACKED && P.dh0 && wi == 0 && at.on)
#pragma unroll
        for (int v = 0; v < V; ++v) P.dh0[(int64_t)at.b * P.dim + at.ch + v] = e0[v];
}

// ---- one token ---------------------------------------------------------------------------------------------
template <int DT>
__global__ void __launch_bounds__(256) gscan_step(const GScan P) {
    using T = typename Elem<DT>::T;
    constexpr bool FULL = DT == CS2D_F32;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)P.batch * P.dim) return;
    const int64_t b = i / P.dim, ch = i % P.dim;
    const float g = Elem<DT>::up(((const T *)P.gate)[b * P.g_bs + ch]), x = Elem<DT>::up(((const T *)P.u)[b * P.u_bs + ch]);
    float *h = P.h + b * P.h_bs + ch;
    float a, c;
    if (P.form == CS2D_GATE_SIGMOID) gate_values<CS2D_GATE_SIGMOID, FULL>(g, a, c);
    else if (P.form == CS2D_GATE_LOG) gate_values<CS2D_GATE_LOG, FULL>(g, a, c);
    else gate_values<CS2D_GATE_DIRECT, FULL>(g, a, c);
    const float v = fmaf(a, *h, P.weighted ? c * x : x);
    *h = v;
    ((T *)P.y)[b * P.y_bs + ch] = Elem<DT>::down(v);
}

// ---- packed sequences: which sequence starts and ends at a row -------------------------------------------------
__global__ void __launch_bounds__(256) gscan_map(const GScan P) {
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (t >= P.length) return;
    int lo = 0, hi = P.nseq + 1;   // the last border at or before the row; of equal ones the last: the sequences before it are empty
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (offset_at(P, mid) <= t) lo = mid; else hi = mid;
    }
    const int64_t first = offset_at(P, lo);
    int2 m = make_int2(SEQ_NONE, SEQ_NONE);
    if (first > t || lo == P.nseq) m.x = SEQ_OUTSIDE;
    else {
        if (first == t) m.x = lo;
        if (offset_at(P, lo + 1) == t + 1) m.y = lo;
    }
    P.map[t] = m;
}

// Warps of a CTA along the rows: as many as the rows need, the others take further units.
int warps_along(int64_t length, int rows) {
    int wt = 1;
    while (wt < GS_WARPS && (int64_t)wt * rows < length) wt <<= 1;
    return wt;
}

template <int DT, int V> cudaError_t fwd(const GScan &P, cudaStream_t st) {
    const int wt = warps_along(P.length, GS_TW);
    const int64_t grid = (P.units + GS_WARPS / wt - 1) / (GS_WARPS / wt);
    if (P.map) gscan_fwd<DT, V, true><<<(unsigned)grid, NT, 0, st>>>(P, wt);
    else gscan_fwd<DT, V, false><<<(unsigned)grid, NT, 0, st>>>(P, wt);
    return cudaGetLastError();
}
template <int DT, int V> cudaError_t bwd(const GScan &P, cudaStream_t st) {
    const int wt = warps_along(P.length, GS_TWB);
    const int64_t grid = (P.units + GS_WARPS / wt - 1) / (GS_WARPS / wt);
    if (P.map) gscan_bwd<DT, V, true><<<(unsigned)grid, NT, 0, st>>>(P, wt);
    else gscan_bwd<DT, V, false><<<(unsigned)grid, NT, 0, st>>>(P, wt);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_gscan_map(const GScan &P, cudaStream_t st) {
    gscan_map<<<(unsigned)((P.length + 255) / 256), 256, 0, st>>>(P);
    return cudaGetLastError();
}
cudaError_t launch_gscan_fwd(const GScan &P, int dt, bool words, cudaStream_t st) {
    switch (dt) {
        case CS2D_F32: return fwd<CS2D_F32, 1>(P, st);
        case CS2D_F16: return words ? fwd<CS2D_F16, 2>(P, st) : fwd<CS2D_F16, 1>(P, st);
        default: return words ? fwd<CS2D_BF16, 2>(P, st) : fwd<CS2D_BF16, 1>(P, st);
    }
}
cudaError_t launch_gscan_bwd(const GScan &P, int dt, bool words, cudaStream_t st) {
    switch (dt) {
        case CS2D_F32: return bwd<CS2D_F32, 1>(P, st);
        case CS2D_F16: return words ? bwd<CS2D_F16, 2>(P, st) : bwd<CS2D_F16, 1>(P, st);
        default: return words ? bwd<CS2D_BF16, 2>(P, st) : bwd<CS2D_BF16, 1>(P, st);
    }
}
cudaError_t launch_gscan_step(const GScan &P, int dt, cudaStream_t st) {
    const unsigned grid = (unsigned)(((int64_t)P.batch * P.dim + 255) / 256);
    switch (dt) {
        case CS2D_F32: gscan_step<CS2D_F32><<<grid, 256, 0, st>>>(P); break;
        case CS2D_F16: gscan_step<CS2D_F16><<<grid, 256, 0, st>>>(P); break;
        default: gscan_step<CS2D_BF16><<<grid, 256, 0, st>>>(P);
    }
    return cudaGetLastError();
}

}  // namespace cs2d
