// Layer norm: how rows are laid over lanes, launches, the sum over slots; rows too wide for registers.  See cs2d_norm.cuh.
#include "cs2d_norm.cuh"

namespace cs2d {

namespace {

using nm::param;

// ---- rows of more channels than a CTA holds in registers: a warp per row, which reads it again for every step ---------
constexpr int NW = 8;   // warps of a CTA

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    return v;
}
template <int DT> __global__ void __launch_bounds__(NW * 32) wide_fwd(const Norm P) {
    using T = typename Elem<DT>::T;
    const int lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * NW + (threadIdx.x >> 5);
    if (row >= P.rows) return;
    const int64_t o = row / P.inner, i = row % P.inner;
    const T *x = (const T *)P.x + o * P.x_os + i * P.x_is;
    const T *z = P.gate ? (const T *)P.gate + o * P.g_os + i * P.g_is : nullptr;
    T *y = (T *)P.y + row * P.dim;
    float s = 0.f, q = 0.f;
    for (int d = lane; d < P.dim; d += 32) s += Elem<DT>::up(x[d * P.x_cs]);
    const float mean = warp_sum(s) / P.dim;
    for (int d = lane; d < P.dim; d += 32) {
        const float m = Elem<DT>::up(x[d * P.x_cs]) - mean;
        q = fmaf(m, m, q);
    }
    const float rstd = rsqrtf(warp_sum(q) / P.dim + P.eps);
    if (P.stats && lane == 0) ((float2 *)P.stats)[row] = make_float2(mean, rstd);
    for (int d = lane; d < P.dim; d += 32) {
        float n = fmaf((Elem<DT>::up(x[d * P.x_cs]) - mean) * rstd, param(P.weight, P.wtype, d, 1.f), param(P.bias, P.wtype, d, 0.f));
        if (z) {
            const float zv = Elem<DT>::up(z[d]);
            n *= zv * sigmoid<DT == CS2D_F32>(zv);
        }
        y[d] = Elem<DT>::down(n);
    }
}

template <int DT> __global__ void __launch_bounds__(NW * 32) wide_bwd(const Norm P) {
    using T = typename Elem<DT>::T;
    constexpr bool FULL = DT == CS2D_F32;
    const int lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * NW + (threadIdx.x >> 5);
    if (row >= P.rows) return;
    const int64_t o = row / P.inner, i = row % P.inner;
    const T *x = (const T *)P.x + o * P.x_os + i * P.x_is, *dy = (const T *)P.dy + o * P.dy_os + i * P.dy_is;
    const T *z = P.gate ? (const T *)P.gate + o * P.g_os + i * P.g_is : nullptr;
    T *dx = (T *)P.dx + o * P.dx_os + i * P.dx_is;
    const float2 st = ((const float2 *)P.stats)[row];
    float s1 = 0.f, s2 = 0.f;
    for (int d = lane; d < P.dim; d += 32) {
        const float xh = (Elem<DT>::up(x[d * P.x_cs]) - st.x) * st.y, w = param(P.weight, P.wtype, d, 1.f);
        float g = Elem<DT>::up(dy[d]);
        if (z) {
            const float zv = Elem<DT>::up(z[d]), sg = sigmoid<FULL>(zv), n = fmaf(xh, w, param(P.bias, P.wtype, d, 0.f));
            ((T *)P.dgate)[row * P.dim + d] = Elem<DT>::down(g * n * (sg + zv * sg * (1.f - sg)));
            g *= zv * sg;
        }
        s1 = fmaf(g, w, s1);
        s2 = fmaf(g * w, xh, s2);
    }
    s1 = warp_sum(s1) / P.dim;
    s2 = warp_sum(s2) / P.dim;
    for (int d = lane; d < P.dim; d += 32) {
        const float xh = (Elem<DT>::up(x[d * P.x_cs]) - st.x) * st.y;
        float g = Elem<DT>::up(dy[d]);
        if (z) {
            const float zv = Elem<DT>::up(z[d]);
            g *= zv * sigmoid<FULL>(zv);
        }
        dx[d * P.dx_cs] = Elem<DT>::down(st.y * (g * param(P.weight, P.wtype, d, 1.f) - s1 - xh * s2));
    }
}

// the parameters' gradients: rows in `parts` runs, a thread per channel
template <int DT> __global__ void __launch_bounds__(NW * 32) wide_part(const Norm P) {
    using T = typename Elem<DT>::T;
    const int d = blockIdx.x * NW * 32 + threadIdx.x;
    if (d >= P.dim) return;
    float w = 0.f, b = 0.f;
    for (int64_t row = blockIdx.y; row < P.rows; row += P.parts) {
        const int64_t o = row / P.inner, i = row % P.inner;
        const float2 st = ((const float2 *)P.stats)[row];
        float g = Elem<DT>::up(((const T *)P.dy)[o * P.dy_os + i * P.dy_is + d]);
        if (P.gate) {
            const float zv = Elem<DT>::up(((const T *)P.gate)[o * P.g_os + i * P.g_is + d]);
            g *= zv * sigmoid<DT == CS2D_F32>(zv);
        }
        b += g;
        w = fmaf(g, (Elem<DT>::up(((const T *)P.x)[o * P.x_os + i * P.x_is + d * P.x_cs]) - st.x) * st.y, w);
    }
    P.part[(int64_t)blockIdx.y * 2 * P.dim + d] = w;
    P.part[((int64_t)blockIdx.y * 2 + 1) * P.dim + d] = b;
}
// ---- the parameters' gradients from their slots ------------------------------------------------------------------
__device__ __forceinline__ void put(void *p, int dt, int i, float v) {
    if (!p) return;
    if (dt == CS2D_F32) ((float *)p)[i] = v;
    else if (dt == CS2D_F16) ((__half *)p)[i] = __float2half_rn(v);
    else ((__nv_bfloat16 *)p)[i] = __float2bfloat16_rn(v);
}
// 32 channels of one sum, the parts in a fixed order: warp w adds parts w, w + 32, ...
__global__ void __launch_bounds__(1024) norm_join(const Norm P) {
    __shared__ float s[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, i = blockIdx.x * 32 + lane;
    float v = 0.f;
    if (i < 2 * P.dim) {
#pragma unroll 8
        for (int k = warp; k < P.parts; k += 32) v += P.part[(int64_t)k * 2 * P.dim + i];
    }
    s[warp][lane] = v;
    __syncthreads();
    v = s[lane][warp];   // warp w: channel w of the block
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    const int c = blockIdx.x * 32 + warp;
    if (lane || c >= 2 * P.dim) return;
    if (c < P.dim) put(P.dweight, P.wtype, c, v);
    else put(P.dbias, P.wtype, c - P.dim, v);
}

// Lanes of a row and vectors of a lane: the fewest places for the row's vectors, of equal ones the fewest lanes (fewer shuffles).
bool lanes_of(int dim, int v, int dt, bool bwd, bool heavy, int *T, int *nv) {
    static const int two[] = {1, 2, 0}, three[] = {1, 2, 3, 0}, f32[] = {1, 2, 3, 6, 0}, pairs[] = {2, 4, 6, 0}, single[] = {4, 6, 8, 12, 0};
    const int *set = v == 1 ? single : v == 2 ? pairs : bwd ? (heavy ? two : three) : dt == CS2D_F32 ? f32 : three;
    const int nvec = dim / v;
    int best = 0;
    for (int t = 1; t <= nm::NT; t <<= 1)
        for (const int *s = set; *s; ++s) {
            if (t * *s < nvec) continue;
            if (!best || t * *s < best) { best = t * *s; *T = t; *nv = *s; }
            break;
        }
    return best != 0;
}
bool on(int bytes, const void *p, int64_t a, int64_t b, int es) { return reinterpret_cast<uintptr_t>(p) % bytes == 0 && a * es % bytes == 0 && b * es % bytes == 0; }
bool on16(const void *p, int64_t a, int64_t b, int es) { return on(16, p, a, b, es); }

struct Plan { nm::Layout l; int v, nv; size_t smem; bool wide; };
constexpr int kSMs = 148;

Plan plan(const Norm &P, int dt, bool bwd) {
    Plan r{};
    const int es = dt == CS2D_F32 ? 4 : 2, V = 16 / es;
    const bool image = P.x_cs != 1;
    // vectors of 16 bytes, pairs of 16-bit elements, single elements
    const auto fits = [&](int v) {
        const int n = v * es;
        bool ok = P.dim % v == 0 && on(n, P.y, 0, 0, es) && (!P.gate || on(n, P.gate, P.g_os, P.g_is, es)) && (v == 2 || (on16(P.weight, 0, 0, 1) && on16(P.bias, 0, 0, 1)));
        if (v == 2 && P.wtype != CS2D_F32) ok = ok && on(4, P.weight, 0, 0, 1) && on(4, P.bias, 0, 0, 1);
        if (!image) ok = ok && on(n, P.x, P.x_os, P.x_is, es);
        if (bwd) ok = ok && on(n, P.dy, P.dy_os, P.dy_is, es) && on(n, P.dgate, 0, 0, es) && (image || on(n, P.dx, P.dx_os, P.dx_is, es));
        return ok;
    };
    r.v = fits(V) ? V : es == 2 && fits(2) ? 2 : 1;
    r.wide = !lanes_of(P.dim, r.v, dt, bwd, P.gate || image, &r.l.T, &r.nv);
    // images whose gradient is not one, and the other way round, take the wide kernels too
    if (bwd && image != (P.dx_cs != 1)) r.wide = true;
    if (r.wide) return r;
    const int e = r.v * r.nv, per = bwd ? (r.v == 1 ? 2 : e <= 8 ? 4 : e <= 12 ? 3 : 2) : 6, groups = nm::NT / r.l.T;
    r.l.image = image;
    if (image) {
        const int64_t row = (int64_t)P.dim * es;
        r.l.pitch = (int)(es == 2 ? (row + 63) / 128 * 128 + 64 : (row + 127) / 128 * 128 + 16);
        r.l.whole = P.inner * es % 16 == 0 && on16(P.x, P.x_os, P.x_cs, es) && (!bwd || on16(P.dx, P.dx_os, P.dx_cs, es));
        r.l.P = es == 2 ? 64 : 32;   // 128 bytes of a channel; fewer where there would be few tiles, or where two CTAs would not fit an SM
        while (r.l.P > (r.l.whole && es == 2 ? 32 : 16) && (P.inner + r.l.P - 1) / r.l.P * (P.rows / P.inner) < 2 * kSMs) r.l.P >>= 1;
        while (r.l.P > 8 && r.l.P * (int64_t)r.l.pitch > (bwd ? 56 : 72) * 1024) r.l.P >>= 1;
        if (r.l.P * (int64_t)r.l.pitch > (bwd ? 120 : 220) * 1024) r.wide = true;
        r.smem = (size_t)r.l.P * r.l.pitch;
    } else {   // some rows per group and tile, as long as there are tiles for all CTAs
        int k = 8;
        while (k > 1 && P.rows < (int64_t)groups * k * kSMs * per) k >>= 1;
        r.l.P = groups * k;
    }
    r.l.tiles = (P.inner + r.l.P - 1) / r.l.P;
    r.l.tiles_all = P.rows / P.inner * r.l.tiles;
    r.l.grid = (int)(r.l.tiles_all < kSMs * per ? r.l.tiles_all : kSMs * per);
    return r;
}

template <int DT> cudaError_t wide(const Norm &P, bool bwd, cudaStream_t st) {
    const unsigned grid = (unsigned)((P.rows + NW - 1) / NW);
    if (!bwd) {
        wide_fwd<DT><<<grid, NW * 32, 0, st>>>(P);
        return cudaGetLastError();
    }
    wide_bwd<DT><<<grid, NW * 32, 0, st>>>(P);
    if (P.part) wide_part<DT><<<dim3((P.dim + NW * 32 - 1) / (NW * 32), P.parts), NW * 32, 0, st>>>(P);
    return cudaGetLastError();
}
cudaError_t wide(const Norm &P, int dt, bool bwd, cudaStream_t st) {
    return dt == CS2D_F32 ? wide<CS2D_F32>(P, bwd, st) : dt == CS2D_F16 ? wide<CS2D_F16>(P, bwd, st) : wide<CS2D_BF16>(P, bwd, st);
}

}  // namespace

// Slots of the parameters' gradients: at most as many as CTAs of any of the kernels.
int norm_parts(const Norm &P, int) { return (int)(P.rows < 4 * kSMs ? P.rows : 4 * kSMs); }

cudaError_t launch_norm_fwd(const Norm &P, int dt, cudaStream_t st) {
    const Plan r = plan(P, dt, false);
    if (r.wide) return wide(P, dt, false, st);
    return (dt == CS2D_F32 ? nm::fwd_f32 : dt == CS2D_F16 ? nm::fwd_f16 : nm::fwd_bf16)(P, r.l, r.v, r.nv, r.smem, st);
}
cudaError_t launch_norm_bwd(const Norm &P_, int dt, cudaStream_t st, int *launches) {
    Norm P = P_;
    if (!P.dweight && !P.dbias) P.part = nullptr;
    const Plan r = plan(P, dt, true);
    if (!r.wide) P.parts = r.l.grid;
    *launches = !P.part ? 1 : r.wide ? 3 : 2;
    const cudaError_t e = r.wide ? wide(P, dt, true, st) : (dt == CS2D_F32 ? nm::bwd_f32 : dt == CS2D_F16 ? nm::bwd_f16 : nm::bwd_bf16)(P, r.l, r.v, r.nv, r.smem, st);
    if (e != cudaSuccess || !P.part) return e;
    norm_join<<<(2 * P.dim + 31) / 32, 1024, 0, st>>>(P);
    return cudaGetLastError();
}

}  // namespace cs2d
