// Gated linear recurrence over tokens, h[t] = a[t] h[t-1] + b[t] per channel: what the forward and the backward kernel share.
//
// A run of rows maps the state before it to the state behind it by h -> A h + B, and such maps compose.  A warp reduces its rows
// to (A, B), the warps of a CTA compose their maps, the CTAs of a cluster theirs, and every warp then walks its rows again from the state
// that reaches it.  A warp copies its own rows to shared memory some tiles ahead (16 bytes per lane and copy), keeps the factors in
// registers between the two walks, and writes each result once: every input is read once and every output written once.  A lane holds two
// channels, which one packed instruction serves.  Nothing depends on the order in which CTAs run.
//
// Units are 64 channels wide (rows of 128 bytes of a 16-bit type) or, where those would not fill the GPU, 16 (a warp then holds four slots of rows).
// Eight warps to a CTA, two CTAs to an SM: one computes while the other waits at its barrier (one CTA of 16 warps: 10 % slower).
// What bounds it is the issue of instructions, not memory: 28 per element and warp lane in the forward, 54 in the backward (B8 L4096 D768, sigmoid
// gate, ncu), 51 % of the issue slots used, the rest waits for MUFU results, shared memory and the barrier.  Measured (bf16, sigmoid, kernels
// alone): B16 L16384 D512 forward 184 us, 67 % of the HBM copy rate, backward 358 us, 57 % (direct gate, not weighted: 162 us, 76 %, and 315 us, 65 %);
// B8 L4096 D768 53 + 96 us (192 CTAs on 296 places); B1 L67200 D384 70 + 115 us.
#pragma once

#include <cooperative_groups.h>

#include <atomic>
#include <cstring>

#include "cs2d_seq.cuh"

namespace cs2d {

namespace gs {

namespace cg = cooperative_groups;

constexpr int MAXC = 16;       // CTAs of a cluster, at most
constexpr int NW = 8;          // warps of a CTA

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 sub2(float2 a, float2 b) { return __ffma2_rn(b, make_float2(-1.f, -1.f), a); }
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// h -> A h + B.  GROWS: factors may be above one; a state of exactly zero meets products A that have overflowed and adds nothing.
template <bool GROWS> __device__ __forceinline__ float2 through(float2 A, float2 B, float2 h) {
    const float2 r = fma2(A, h, B);
    return GROWS ? make_float2(h.x == 0.f ? B.x : r.x, h.y == 0.f ? B.y : r.y) : r;
}

// ---- a lane's two channels -----------------------------------------------------------------------------------
template <int DT> struct Two;
template <> struct Two<CS2D_F32> {
    using W = float2;
    static __device__ __forceinline__ float2 up(W w) { return w; }
    static __device__ __forceinline__ W down(float2 x) { return x; }
};
template <> struct Two<CS2D_F16> {
    using W = __half2;
    static __device__ __forceinline__ float2 up(W w) { return __half22float2(w); }
    static __device__ __forceinline__ W down(float2 x) { return __float22half2_rn(x); }
};
template <> struct Two<CS2D_BF16> {
    using W = unsigned;   // a bf16 is the upper half of the fp32 of the same value
    static __device__ __forceinline__ float2 up(W w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
    static __device__ __forceinline__ W down(float2 x) {
        const __nv_bfloat162 v = __float22bfloat162_rn(x);
        W w;
        memcpy(&w, &v, 4);
        return w;
    }
};
__device__ __forceinline__ float2 ld2(const float *p, bool one, bool two) { return make_float2(one ? p[0] : 0.f, two ? p[1] : 0.f); }
__device__ __forceinline__ void st2(float *p, float2 v, bool one, bool two) {
    if (one) p[0] = v.x;
    if (two) p[1] = v.y;
}

// ---- places --------------------------------------------------------------------------------------------------
// A slot: G lanes with two channels each, TW rows.  A warp holds 32 / G slots one behind the other, of one unit of 2 G channels; warps follow
// each other along the rows.  Where the rows do not fill the CTA's warps (wt of them along the rows), the others take further units.
template <int DT, int G, int TW> struct Place {
    using T = typename Elem<DT>::T;
    static constexpr int CB = 2 * G, S = 32 / G, ROWS = S * TW;   // channels of a unit; slots and rows of a warp
    static constexpr int RB = CB * sizeof(T);                     // bytes of a staged row
    static constexpr int SB = TW * RB + (S > 1 ? RB : 0);         // of a slot: the slots of a warp lie in different banks
    static constexpr int TB = S * SB;                             // of a warp's tile
    int lane, warp, li, sub, wi, b, c0, ch;
    bool one, two;    // which of the lane's channels exist
    int rows;         // of the unit; 0: no such unit
    bool full;        // all channels of the unit exist
    __device__ __forceinline__ Place(const GScan &P, int wt, int cluster_id) {
        lane = threadIdx.x & 31;
        li = lane % G;
        sub = lane / G;
        warp = __shfl_sync(~0u, threadIdx.x >> 5, 0);
        wi = warp % wt;
        const int64_t unit = (int64_t)cluster_id * (NW / wt) + warp / wt;
        const bool here = unit < P.units;
        b = here ? (int)(unit / P.nblk) : 0;
        c0 = here ? (int)(unit % P.nblk) * CB : 0;
        ch = c0 + 2 * li;
        one = here && ch < P.dim;
        two = here && ch + 1 < P.dim;
        if (!one) ch = c0;   // addresses stay inside the tensors
        rows = here ? (int)P.length : 0;
        full = c0 + CB <= P.dim;
    }
    // rows of the warp's (the slot's) that are there, from row r
    __device__ __forceinline__ int there(int r, int most) const { return max(0, min(rows - r, most)); }
    // where the lane's word of its slot's row i lies
    __device__ __forceinline__ const unsigned char *in(const unsigned char *tile) const { return tile + sub * SB + li * 2 * sizeof(T); }
    __device__ __forceinline__ float2 staged(const unsigned char *tile, int i) const {
        return Two<DT>::up(*(const typename Two<DT>::W *)(in(tile) + i * RB));
    }
    __device__ __forceinline__ void stage(unsigned char *tile, int i, float2 v) const {
        *(typename Two<DT>::W *)(const_cast<unsigned char *>(in(tile)) + i * RB) = Two<DT>::down(v);
    }
};

__device__ __forceinline__ int64_t offset_at(const GScan &P, int i) {
    return P.off64 ? ((const int64_t *)P.offsets)[i] : (int64_t)((const int32_t *)P.offsets)[i];
}
// Packed sequences: where in a slot's rows sequences start and end, as bits.  Loaded a tile ahead.
template <int G, int TW> struct Marks {
    static constexpr int K = (TW + G - 1) / G, N = TW < G ? TW : G;   // rows of a lane; lanes with rows
    int2 m[K];
    __device__ __forceinline__ void load(const GScan &P, int t0, int li, int L) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int t = t0 + k * G + li % N;
            m[k] = t >= 0 && t < L ? P.map[t] : make_int2(SEQ_OUTSIDE, SEQ_NONE);
        }
    }
    __device__ __forceinline__ void masks(int sub, unsigned &starts, unsigned &ends) const {
        starts = ends = 0;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            starts |= ((__ballot_sync(~0u, m[k].x != SEQ_NONE) >> (sub * G)) & ((1u << N) - 1)) << (k * G);
            ends |= ((__ballot_sync(~0u, m[k].y >= 0) >> (sub * G)) & ((1u << N) - 1)) << (k * G);
        }
    }
};
// Sequences without a row: their state passes through.  The warps of the unit share them (first, of how many).  Also reports borders
// that are not ascending or leave the tensor.
template <class Place> __device__ __forceinline__ void empty_sequences(const GScan &P, const Place &at, int first, int stride, const float *in, int64_t in_s, float *out, bool report) {
    for (int s = first; s < P.nseq; s += stride) {
        const int64_t lo = offset_at(P, s), hi = offset_at(P, s + 1);
        if (report && (lo < 0 || hi > P.length || hi < lo) && at.lane == 0) atomicOr(P.status, ERR_SEQ_OFFSETS);
        if (hi <= lo && at.sub == 0) st2(out + (int64_t)s * P.dim + at.ch, in ? ld2(in + (int64_t)s * in_s + at.ch, at.one, at.two) : both(0.f), at.one, at.two);
    }
}

// ---- rows to shared memory -------------------------------------------------------------------------------------
template <int BYTES> __device__ __forceinline__ void copy_async(void *dst, const void *src, bool ok) {   // !ok: zeros
    const unsigned d = (unsigned)__cvta_generic_to_shared(dst);
    const int n = ok ? BYTES : 0;
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(src), "r"(n) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(d), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

template <int BYTES> __device__ __forceinline__ void copy_async(void *dst, const void *src) {
    const unsigned d = (unsigned)__cvta_generic_to_shared(dst);
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(d), "l"(src) : "memory");
}

// A tensor as a warp walks it: `at` is the address of the first channel of its unit in the first row of its next tile.
template <int DT, int G, int TW> struct Walk {
    using L = Place<DT, G, TW>;
    using T = typename L::T;
    static constexpr int ES = sizeof(T);
    char *at;
    int64_t step, row;   // bytes: from tile to tile, from row to row
    __device__ __forceinline__ Walk(const void *base, int64_t bs, int64_t ls, const L &p, int first, int64_t rows_per_step)
        : at((char *)base + (p.b * bs + first * ls + p.c0) * (int64_t)ES), step(rows_per_step * ls * ES), row(ls * ES) {}
    // Pieces of B bytes: a warp moves RPI rows at a time, in N instructions where a row has more than 32 pieces.
    template <int B> struct Pieces {
        static constexpr int CPR = L::RB / B, N = CPR > 32 ? CPR / 32 : 1, RPI = CPR > 32 ? 1 : 32 / CPR;
        static_assert(RPI % TW == 0 || TW % RPI == 0, "an instruction's rows are whole slots or part of one");
        static __device__ __forceinline__ int of(int lane) { return CPR > 32 ? lane : lane % CPR; }
        static __device__ __forceinline__ int row(int lane) { return CPR > 32 ? 0 : lane / CPR; }
        static __device__ __forceinline__ int place(int j) { return RPI >= TW ? j * (RPI / TW) * L::SB : j * RPI / TW * L::SB + j * RPI % TW * L::RB; }
        static __device__ __forceinline__ int lane_place(int lane) { return row(lane) / TW * L::SB + row(lane) % TW * L::RB + of(lane) * B; }
    };
    template <int B> __device__ __forceinline__ void fetch_pieces(unsigned char *dst, int n, const L &p, int dim) const {
        using Q = Pieces<B>;
        const char *s = at + Q::row(p.lane) * row + Q::of(p.lane) * B;
        unsigned char *d = dst + Q::lane_place(p.lane);
        const int64_t rows = Q::RPI * row;
        if (n == L::ROWS && p.full) {
#pragma unroll
            for (int j = 0; j < L::ROWS / Q::RPI; ++j) {
#pragma unroll
                for (int h = 0; h < Q::N; ++h) copy_async<B>(d + Q::place(j) + h * 32 * B, s + h * 32 * B);
                s += rows;
            }
        } else {   // what is not there comes as zeros
            const int left = n - Q::row(p.lane), c = p.c0 + Q::of(p.lane) * B / ES;
#pragma unroll
            for (int j = 0; j < L::ROWS / Q::RPI; ++j) {
#pragma unroll
                for (int h = 0; h < Q::N; ++h) {
                    const bool ok = j * Q::RPI < left && c + h * 32 * B / ES < dim;
                    copy_async<B>(d + Q::place(j) + h * 32 * B, ok ? s + h * 32 * B : at, ok);
                }
                s += rows;
            }
        }
    }
    template <int B> __device__ __forceinline__ void flush_pieces(const unsigned char *tile, int n, const L &p, int dim) const {
        using Q = Pieces<B>;
        using W = typename WordOf<B>::W;
        char *d = at + Q::row(p.lane) * row + Q::of(p.lane) * B;
        const unsigned char *s = tile + Q::lane_place(p.lane);
        const int64_t rows = Q::RPI * row;
        const int left = n - Q::row(p.lane), c = p.c0 + Q::of(p.lane) * B / ES;
#pragma unroll
        for (int j = 0; j < L::ROWS / Q::RPI; ++j) {
#pragma unroll
            for (int h = 0; h < Q::N; ++h)
                if (j * Q::RPI < left && c + h * 32 * B / ES < dim) *(W *)(d + h * 32 * B) = *(const W *)(s + Q::place(j) + h * 32 * B);
            d += rows;
        }
    }
    // The n rows that are there to shared memory.
    __device__ __forceinline__ void fetch(unsigned char *dst, int n, const L &p, int dim, int how) const {
        if (how == GS_CHUNKS) fetch_pieces<16>(dst, n, p, dim);
        else if (how == GS_WORDS) fetch_pieces<4>(dst, n, p, dim);
        else if constexpr (ES == 2) {
            T *d = (T *)(dst + p.sub * L::SB) + p.li * 2;
            const char *s = at + p.sub * TW * row + (p.ch - p.c0) * ES;
#pragma unroll 4
            for (int i = 0; i < TW; ++i) {
                const bool ok = p.sub * TW + i < n;
                d[i * L::CB] = ok && p.one ? ((const T *)(s + i * row))[0] : Elem<DT>::down(0.f);
                d[i * L::CB + 1] = ok && p.two ? ((const T *)(s + i * row))[1] : Elem<DT>::down(0.f);
            }
        }
    }
    // The first n rows of a staged tile to the tensor.
    __device__ __forceinline__ void flush(const unsigned char *tile, int n, const L &p, int dim, int how) const {
        if (how == GS_CHUNKS) flush_pieces<16>(tile, n, p, dim);
        else if (how == GS_WORDS) flush_pieces<4>(tile, n, p, dim);
        else if constexpr (ES == 2) {
#pragma unroll 1
            for (int j = p.lane; j < L::ROWS * L::CB; j += 32) {
                const int r = j / L::CB, c = j % L::CB;
                if (r < n && p.c0 + c < dim) ((T *)(at + r * row))[c] = ((const T *)(tile + r / TW * L::SB + r % TW * L::RB))[c];
            }
        }
    }
    __device__ __forceinline__ void next() { at += step; }
};

// ---- maps ------------------------------------------------------------------------------------------------------
// The map of a run of rows; cut: a sequence starts inside, so the state before the run does not reach its end.
template <bool GROWS, bool PACKED> struct Map {
    float2 A, B;
    int cut;
    __device__ __forceinline__ Map() : A(both(1.f)), B(both(0.f)), cut(0) {}
    __device__ __forceinline__ float2 apply(float2 h) const {
        const float2 r = through<GROWS>(A, B, h);
        return PACKED && cut ? B : r;
    }
    __device__ __forceinline__ void after(const Map &m) {   // this run behind m's
        B = apply(m.B);
        A = mul2(A, m.A);
        cut |= m.cut;
    }
};
template <int G> struct MapStore {   // one per lane of a slot
    float4 ab[G];
    int cut, pad[3];
    template <bool GROWS, bool PACKED> __device__ __forceinline__ void put(const Map<GROWS, PACKED> &m, int li) {
        ab[li] = make_float4(m.A.x, m.A.y, m.B.x, m.B.y);
        if (PACKED && li == 0) cut = m.cut;
    }
    template <bool GROWS, bool PACKED> __device__ __forceinline__ Map<GROWS, PACKED> get(int li) const {
        Map<GROWS, PACKED> m;
        const float4 t = ab[li];
        m.A = make_float2(t.x, t.y);
        m.B = make_float2(t.z, t.w);
        if (PACKED) m.cut = cut;
        return m;
    }
};
// Over the slots of a warp: m becomes the map of all of them in the last one (UP; else the first), `before` that of the slots before (behind) each.
template <int G, bool GROWS, bool PACKED, bool UP> __device__ __forceinline__ void over_slots(Map<GROWS, PACKED> &m, Map<GROWS, PACKED> &before, int lane) {
    if constexpr (G < 32) {
        auto shifted = [&](int d) {
            Map<GROWS, PACKED> o;
            auto s = [&](auto v) { return UP ? __shfl_up_sync(~0u, v, d) : __shfl_down_sync(~0u, v, d); };
            o.A = make_float2(s(m.A.x), s(m.A.y));
            o.B = make_float2(s(m.B.x), s(m.B.y));
            if (PACKED) o.cut = s(m.cut);
            return o;
        };
#pragma unroll
        for (int d = G; d < 32; d <<= 1) {
            const Map<GROWS, PACKED> o = shifted(d);
            if (UP ? lane >= d : lane + d < 32) m.after(o);
        }
        const Map<GROWS, PACKED> o = shifted(G);
        if (UP ? lane >= G : lane + G < 32) before = o;
    }
}

// What reaches run k of the n <= N runs whose maps these are, from `state` before (UP) or behind them all; `state` moves past them.
template <bool GROWS, bool PACKED, bool UP, int N, int G> __device__ __forceinline__ float2 pass(const MapStore<G> *maps, int n, int k, int li, float2 &state) {
    float2 reach = state;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const int w = UP ? j : N - 1 - j;
        if (w == k) reach = state;
        if (w < n) state = maps[w].template get<GROWS, PACKED>(li).apply(state);
    }
    return reach;
}

// ---- from CTA to CTA -------------------------------------------------------------------------------------------
// Every CTA of a cluster sends the map of its tile to all of them (itself too) by stores that count their bytes on the receiver's barrier, and
// waits for its own barrier alone.  Two places: who sends for step s + 2 has all maps of step s + 1, which their CTAs sent behind a barrier that
// all of their warps met after reading those of step s.
template <int G> struct Exchange {
    MapStore<G> slot[2][MAXC];
    uint64_t full[2], pad[2];
};
constexpr int WAIT_POLLS = 1 << 20;
__device__ __forceinline__ unsigned shared_address(const void *p) { return (unsigned)__cvta_generic_to_shared(p); }
template <bool PACKED, int G> __device__ __forceinline__ void expect(Exchange<G> *x, int place, int C) {   // one thread
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(shared_address(&x->full[place])), "r"(C * (G * 16 + (PACKED ? 4 : 0))) : "memory");
}
template <bool PACKED, int G> __device__ __forceinline__ void exchange_init(Exchange<G> *x, int C) {
    if (threadIdx.x == 0) {
        for (int k = 0; k < 2; ++k) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(shared_address(&x->full[k])) : "memory");
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        for (int k = 0; k < 2; ++k) expect<PACKED>(x, k, C);
    }
    cg::this_cluster().sync();   // every CTA runs and has its barriers before another one writes there
}
__device__ __forceinline__ unsigned in_cta(unsigned address, int rank) {
    unsigned r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(address), "r"(rank));
    return r;
}
template <bool GROWS, bool PACKED, bool UP, int G, class Place>
__device__ __forceinline__ float2 pass_cluster(const MapStore<G> *maps, Exchange<G> *x, unsigned step, int rank, int C, const Place &at, float2 &state,
                                               int *status) {
    const int place = step & 1;
    for (int r = at.warp; r < C; r += NW) {   // warp r sends to CTA r (and r + 8)
        Map<GROWS, PACKED> m;
#pragma unroll
        for (int k = 0; k < NW; ++k) {
            Map<GROWS, PACKED> q = maps[UP ? k : NW - 1 - k].template get<GROWS, PACKED>(at.li);
            q.after(m);
            m = q;
        }
        const unsigned full = in_cta(shared_address(&x->full[place]), r);
        if (at.lane < G)
            asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(
                             in_cta(shared_address(&x->slot[place][rank].ab[at.li]), r)),
                         "r"(__float_as_uint(m.A.x)), "r"(__float_as_uint(m.A.y)), "r"(__float_as_uint(m.B.x)), "r"(__float_as_uint(m.B.y)), "r"(full)
                         : "memory");
        if (PACKED && at.lane == 0)
            asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];" ::"r"(
                             in_cta(shared_address(&x->slot[place][rank].cut), r)),
                         "r"(m.cut), "r"(full)
                         : "memory");
    }
    const unsigned phase = (step >> 1) & 1;
    int left = WAIT_POLLS;
    for (;;) {
        unsigned ok;
        asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
                     : "=r"(ok) : "r"(shared_address(&x->full[place])), "r"(phase) : "memory");
        if (ok) break;
        if (--left == 0) {   // goes on, so that everybody runs to the end
            atomicOr(status, ERR_WORKER_TIMEOUT);
            break;
        }
    }
    if (threadIdx.x == 0) expect<PACKED>(x, place, C);
    float2 own = state;
#pragma unroll 4
    for (int k = 0; k < C; ++k) {
        const int r = UP ? k : C - 1 - k;
        if (r == rank) own = state;
        state = x->slot[place][r].template get<GROWS, PACKED>(at.li).apply(state);
    }
    return pass<GROWS, PACKED, UP, NW>(maps, NW, at.wi, at.li, own);
}

// ---- launches ----------------------------------------------------------------------------------------------------
struct Split { int wt, C; int64_t grid; };   // warps along the rows; CTAs of a cluster

inline void configure(cudaLaunchConfig_t &cfg, cudaLaunchAttribute *attr, int64_t grid, int C, size_t smem, cudaStream_t st) {
    cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(32 * NW);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    if (C == 1) return;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
}
// Launches KERNEL with its rows split as they should be; rows: of a warp's tile.
template <auto KERNEL> cudaError_t start(GScan &P, int G, int rows, size_t smem, cudaStream_t st) {
    // Per device and cluster size: clusters that fit the GPU at a time.  The entry of size one is written last: the others are there.  Threads that
    // come at the same time write the same numbers.
    static std::atomic<int> at_once[64][MAXC + 1] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || dev < 0 || dev >= 64) return e != cudaSuccess ? e : cudaErrorInvalidDevice;
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr[1];
    if (!at_once[dev][1].load(std::memory_order_acquire)) {
        if ((e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem)) != cudaSuccess) return e;
        if ((e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeNonPortableClusterSizeAllowed, 1)) != cudaSuccess) return e;
        for (int C = MAXC; C >= 1; --C) {
            configure(cfg, attr, C, C, smem, st);
            int n = 1;
            if (C > 1 && cudaOccupancyMaxActiveClusters(&n, KERNEL, &cfg) != cudaSuccess) n = 0;
            at_once[dev][C].store(n, std::memory_order_release);
        }
        cudaGetLastError();   // (a size that the device does not have)
    }
    Split s{1, 1, 0};
    P.nblk = (P.dim + 2 * G - 1) / (2 * G);
    P.units = (int64_t)P.batch * P.nblk;
    while (s.wt < NW && (int64_t)s.wt * rows < P.length) s.wt <<= 1;   // the others take further units
    const int64_t tile = (int64_t)s.wt * rows, tiles = (P.length + tile - 1) / tile, per = NW / s.wt, ctas = (P.units + per - 1) / per;
    // The largest cluster of which all fit the GPU at once: a second round would take as long as the first (24 units: 26 clusters of 10
    // fit, B1 L67200 D384 70 + 114 us; 21 of 12, 88 + 148 us; 33 of 8, 76 + 129 us).
    for (int C = (int)(tiles < MAXC ? tiles : MAXC); C > 1 && s.C == 1; --C)
        if (at_once[dev][C].load(std::memory_order_relaxed) >= ctas) s.C = C;
    s.grid = ctas * s.C;
    configure(cfg, attr, s.grid, s.C, smem, st);
    return cudaLaunchKernelEx(&cfg, KERNEL, (const GScan)P, (const int)s.wt, (const int)s.C);
}
// Units of 16 channels instead of 64 where there are few wide ones: rows of 32 bytes instead of 128 take more instructions per element, but there are
// four times as many units for clusters of at most 16 CTAs.  Wide against narrow, forward + backward in us (bf16, sigmoid): 6 wide units of 67200 rows
// 86 + 166, 70 + 115; 12 of 16384 37 + 66, 39 + 55; 96 of 4096 53 + 96, 55 + 96; 128 of 16384 184 + 358, 231 + 428.  From 24 to 95 units it depends
// on the rows: of 512, 64 units 12 + 14, 10 + 14; of 4096, 48 units 31 + 47, 37 + 61; of 16384, 80 units 131 + 247, 180 + 346 (fp32, 48 units of
// 4096: 47 + 79, 53 + 88).  So the border of 96 is the better one for short rows and not for long ones.
inline bool narrow(const GScan &P) { return P.batch * (int64_t)((P.dim + 63) / 64) < 96 && P.length > 128; }

}  // namespace gs

}  // namespace cs2d
