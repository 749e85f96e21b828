// Layer norm over the channels of a row, with an optional SiLU gate behind it:
//   xh = (x - mean) / sqrt(var + eps)    n = xh w + b    y = n silu(z)
//   dn = dy silu(z)   t = dn w   dx = (t - mean(t) - xh mean(t xh)) / sqrt(var + eps)   dz = dy n silu'(z)
//   dw = sum over rows of dn xh   db = sum over rows of dn
// Sums and statistics in 32 bits; the variance is that of the centred values.
#include "cs2d_seq.cuh"

namespace cs2d {

namespace {

constexpr int NW = 8;   // warps of a CTA

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    return v;
}
__device__ __forceinline__ float param(const void *p, int dt, int i, float none) {
    if (!p) return none;
    return dt == CS2D_F32 ? ((const float *)p)[i] : dt == CS2D_F16 ? __half2float(((const __half *)p)[i]) : __bfloat162float(((const __nv_bfloat16 *)p)[i]);
}

template <int DT> __global__ void __launch_bounds__(NW * 32) norm_fwd(const Norm P) {
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

template <int DT> __global__ void __launch_bounds__(NW * 32) norm_bwd(const Norm P) {
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
template <int DT> __global__ void __launch_bounds__(NW * 32) norm_part(const Norm P) {
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
__device__ __forceinline__ void put(void *p, int dt, int i, float v) {
    if (!p) return;
    if (dt == CS2D_F32) ((float *)p)[i] = v;
    else if (dt == CS2D_F16) ((__half *)p)[i] = __float2half_rn(v);
    else ((__nv_bfloat16 *)p)[i] = __float2bfloat16_rn(v);
}
// 32 channels of one sum, the parts in a fixed order
__global__ void __launch_bounds__(NW * 32) norm_join(const Norm P) {
    __shared__ float s[NW][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, i = blockIdx.x * 32 + lane;
    float v = 0.f;
    if (i < 2 * P.dim)
        for (int k = warp; k < P.parts; k += NW) v += P.part[(int64_t)k * 2 * P.dim + i];
    s[warp][lane] = v;
    __syncthreads();
    if (warp || i >= 2 * P.dim) return;
    for (int k = 1; k < NW; ++k) v += s[k][lane];
    if (i < P.dim) put(P.dweight, P.wtype, i, v);
    else put(P.dbias, P.wtype, i - P.dim, v);
}

template <int DT> cudaError_t bwd(const Norm &P, cudaStream_t st) {
    norm_bwd<DT><<<(unsigned)((P.rows + NW - 1) / NW), NW * 32, 0, st>>>(P);
    if (!P.dweight && !P.dbias) return cudaGetLastError();
    norm_part<DT><<<dim3((P.dim + NW * 32 - 1) / (NW * 32), P.parts), NW * 32, 0, st>>>(P);
    norm_join<<<(2 * P.dim + 31) / 32, NW * 32, 0, st>>>(P);
    return cudaGetLastError();
}

}  // namespace

int norm_parts(const Norm &P, int) { return (int)(P.rows < 512 ? (P.rows < 1 ? 1 : P.rows) : 512); }

cudaError_t launch_norm_fwd(const Norm &P, int dt, cudaStream_t st) {
    const unsigned grid = (unsigned)((P.rows + NW - 1) / NW);
    switch (dt) {
        case CS2D_F32: norm_fwd<CS2D_F32><<<grid, NW * 32, 0, st>>>(P); break;
        case CS2D_F16: norm_fwd<CS2D_F16><<<grid, NW * 32, 0, st>>>(P); break;
        default: norm_fwd<CS2D_BF16><<<grid, NW * 32, 0, st>>>(P);
    }
    return cudaGetLastError();
}
cudaError_t launch_norm_bwd(const Norm &P, int dt, cudaStream_t st) {
    switch (dt) {
        case CS2D_F32: return bwd<CS2D_F32>(P, st);
        case CS2D_F16: return bwd<CS2D_F16>(P, st);
        default: return bwd<CS2D_BF16>(P, st);
    }
}

}  // namespace cs2d
