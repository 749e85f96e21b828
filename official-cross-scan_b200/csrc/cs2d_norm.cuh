// Layer norm over the channels of a row, with an optional SiLU gate behind it:
//   xh = (x - mean) / sqrt(var + eps)    n = xh w + b    y = n silu(z)
//   dn = dy silu(z)   t = dn w   dx = (t - mean(t) - xh mean(t xh)) / sqrt(var + eps)   dz = dy n silu'(z)
//   dw = sum over rows of dn xh   db = sum over rows of dn
// Sums and statistics in 32 bits; the variance is that of the centred values.
//
// A group of T lanes (up to the whole CTA) holds a row in registers, E channels per lane, and reads every input once.  The backward keeps the
// sums of dw and db of its rows in registers too; CTAs leave them in slots, which a second kernel adds in a fixed order.
// Channel-major images pass through shared memory: a tile of P positions and all channels is read along the positions, transposed on the way
// in (16-bit types: by stmatrix), and its rows are worked on like those of tokens; the backward puts dx in the place of x and stores the tile the
// way it came.
#pragma once

#include <cstring>

#include "cs2d_seq.cuh"

namespace cs2d {

namespace nm {

constexpr int NT = 256;       // threads of a CTA
constexpr int NWARP = NT / 32;
constexpr int MAXE = 24;      // channels of a lane

struct Layout {
    int T, P, pitch;          // lanes of a row; positions of a tile and bytes between its rows in shared memory (images)
    bool whole;               // tiles are read in 16-byte chunks
    int64_t tiles;            // per outer index
    int grid;
};

__device__ __forceinline__ float param(const void *p, int dt, int i, float none) {
    if (!p) return none;
    return dt == CS2D_F32 ? ((const float *)p)[i] : dt == CS2D_F16 ? __half2float(((const __half *)p)[i]) : __bfloat162float(((const __nv_bfloat16 *)p)[i]);
}

// V consecutive parameters from channel d
template <int V> __device__ __forceinline__ void params(float (&v)[V], const void *p, int dt, int d, float none) {
    if (V > 1 && p && dt == CS2D_F32) {
#pragma unroll
        for (int k = 0; k < V; k += 4) {
            const float4 t = *(const float4 *)((const float *)p + d + k);
            v[k] = t.x; v[k + 1] = t.y; v[k + 2] = t.z; v[k + 3] = t.w;
        }
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = param(p, dt, d + k, none);
    }
}

// Sums of two values over the T lanes of a row.  More than a warp: through shared memory, a named barrier per row group; two sets of
// slots, so that the next sum may begin while others still read.
struct Reduce {
    float2 (*slots)[NWARP];
    int T, parity;
    __device__ __forceinline__ float2 operator()(float a, float b) {
        const int in_warp = T < 32 ? T : 32;
        for (int o = in_warp >> 1; o; o >>= 1) {
            a += __shfl_xor_sync(~0u, a, o);
            b += __shfl_xor_sync(~0u, b, o);
        }
        if (T <= 32) return make_float2(a, b);
        const int warp = threadIdx.x >> 5, R = T / 32, first = warp / R * R;
        if ((threadIdx.x & 31) == 0) slots[parity][warp] = make_float2(a, b);
        asm volatile("bar.sync %0, %1;" ::"r"(1 + warp / R), "r"(T) : "memory");
        float2 s = slots[parity][first];
        for (int k = 1; k < R; ++k) {
            s.x += slots[parity][first + k].x;
            s.y += slots[parity][first + k].y;
        }
        parity ^= 1;
        return s;
    }
};

// ---- tiles of images -------------------------------------------------------------------------------------------
// Row p of a tile starts at p * pitch; its 16-byte chunk c lies in the place of chunk c ^ swizzle(p).  pitch is 64 more than a multiple of 128
// (16-bit types), 16 more (fp32): the rows that an instruction touches fall into different banks.
template <int ES> __device__ __forceinline__ int swizzle(int p) { return ES == 2 ? (p >> 3) & 3 : (p >> 2) & 7; }
template <int ES> __device__ __forceinline__ unsigned char *chunk(unsigned char *tile, int pitch, int p, int c) { return tile + p * pitch + ((c ^ swizzle<ES>(p)) << 4); }
template <int ES> __device__ __forceinline__ unsigned char *element(unsigned char *tile, int pitch, int p, int d) {
    return chunk<ES>(tile, pitch, p, d / (16 / ES)) + d % (16 / ES) * ES;
}
// IN: image -> tile, else tile -> image.  img: channel 0, first position; cs: elements between channels; n positions are there.
template <int DT, bool IN> __device__ __forceinline__ void move_tile(unsigned char *tile, const Layout &l, typename Elem<DT>::T *img, int64_t cs, int dim, int n) {
    using T = typename Elem<DT>::T;
    constexpr int ES = sizeof(T);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (ES == 2 && l.whole && l.P == 32) {
        // a warp takes 8 channels x 32 positions: lane t has 8 positions of channel t / 4.  Word k of the lanes is an 8 x 8 matrix whose column
        // c is position 8 (c / 2) + 2 k + c % 2; its transpose is eight 16-byte chunks, one per position.
        const int m = lane >> 3, c = lane & 7, p = 8 * (c >> 1) + 2 * m + (c & 1), q = 8 * (lane & 3);
#pragma unroll 4
        for (int d0 = warp * 8; d0 < dim; d0 += NWARP * 8) {
            const int d = d0 + (lane >> 2);
            const bool ok = d < dim && q < n;
            T *g = img + d * cs + q;
            const unsigned s = (unsigned)__cvta_generic_to_shared(chunk<ES>(tile, l.pitch, p, d0 >> 3));
            uint4 v = make_uint4(0, 0, 0, 0);
            if constexpr (IN) {
                if (ok) v = *(const uint4 *)g;
                asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(s), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
            } else {
                asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(s) : "memory");
                if (ok) *(uint4 *)g = v;
            }
        }
    } else if (ES == 4 && l.whole) {
        const int per = l.P / 4;   // chunks of a channel
#pragma unroll 4
        for (int i = threadIdx.x; i < dim * per; i += NT) {
            const int d = i / per, q = i % per * 4;
            if (q >= n) continue;
            T *g = img + d * cs + q;
            if constexpr (IN) {
                const float4 v = *(const float4 *)g;
                *(float *)element<ES>(tile, l.pitch, q, d) = v.x;
                *(float *)element<ES>(tile, l.pitch, q + 1, d) = v.y;
                *(float *)element<ES>(tile, l.pitch, q + 2, d) = v.z;
                *(float *)element<ES>(tile, l.pitch, q + 3, d) = v.w;
            } else {
                float4 v;
                v.x = *(const float *)element<ES>(tile, l.pitch, q, d);
                v.y = *(const float *)element<ES>(tile, l.pitch, q + 1, d);
                v.z = *(const float *)element<ES>(tile, l.pitch, q + 2, d);
                v.w = *(const float *)element<ES>(tile, l.pitch, q + 3, d);
                *(float4 *)g = v;
            }
        }
    } else {
#pragma unroll 8
        for (int i = threadIdx.x; i < dim * l.P; i += NT) {
            const int d = i / l.P, p = i % l.P;
            if (p >= n) continue;
            T *e = (T *)element<ES>(tile, l.pitch, p, d), *g = img + d * cs + p;
            if constexpr (IN) *e = *g;
            else *g = *e;
        }
    }
}

// ---- rows ------------------------------------------------------------------------------------------------------
// A lane's channels of a row: NV vectors of V, vector j of lane l being number j T + l of the row.
template <int DT, int V, int NV> struct Row {
    using P = Pack<DT, V>;
    using W = typename P::W;
    static __device__ __forceinline__ void load(W (&w)[NV], const typename Elem<DT>::T *row, int l, int T, int nvec, bool on) {
#pragma unroll
        for (int j = 0; j < NV; ++j) w[j] = on && j * T + l < nvec ? *(const W *)(row + (int64_t)(j * T + l) * V) : W{};
    }
};

template <int DT, int V, int NV, bool GATED, bool IMAGE>
__global__ void __launch_bounds__(NT, 2) norm_fwd(const Norm P, const Layout lay) {
    using R = Row<DT, V, NV>;
    using W = typename R::W;
    using T = typename Elem<DT>::T;
    constexpr bool FULL = DT == CS2D_F32;
    extern __shared__ __align__(16) unsigned char tile[];
    __shared__ float2 slots[2][NWARP];
    Reduce sum{slots, lay.T, 0};
    const int TL = lay.T, l = threadIdx.x % TL, g = threadIdx.x / TL, groups = NT / TL, nvec = P.dim / V;
    const float inv = 1.f / P.dim;
    auto work = [&](int64_t row, const T *x, int p, bool on) {
        W xw[NV], zw[GATED ? NV : 1];
        const int64_t o = on ? row / P.inner : 0, i = on ? row % P.inner : 0;
        if constexpr (IMAGE) {
#pragma unroll
            for (int j = 0; j < NV; ++j)
                xw[j] = on && j * TL + l < nvec ? *(const W *)element<sizeof(T)>(tile, lay.pitch, p, (j * TL + l) * V) : W{};
        } else {
            R::load(xw, x + o * P.x_os + i * P.x_is, l, TL, nvec, on);
        }
        if constexpr (GATED) R::load(zw, (const T *)P.gate + o * P.g_os + i * P.g_is, l, TL, nvec, on);
        float s = 0.f, q = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float v[V];
            R::P::up(xw[j], v);
#pragma unroll
            for (int k = 0; k < V; ++k) s += v[k];
        }
        const float mean = sum(s, 0.f).x * inv;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float v[V];
            R::P::up(xw[j], v);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float m = j * TL + l < nvec ? v[k] - mean : 0.f;
                q = fmaf(m, m, q);
            }
        }
        const float rstd = rsqrtf(sum(q, 0.f).x * inv + P.eps);
        if (!on) return;
        if (P.stats && l == 0) ((float2 *)P.stats)[row] = make_float2(mean, rstd);
        T *y = (T *)P.y + row * P.dim;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int vec = j * TL + l;
            if (vec >= nvec) continue;
            float v[V], w[V], b[V], z[V];
            R::P::up(xw[j], v);
            params<V>(w, P.weight, P.wtype, vec * V, 1.f);
            params<V>(b, P.bias, P.wtype, vec * V, 0.f);
            if constexpr (GATED) R::P::up(zw[j], z);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                v[k] = fmaf((v[k] - mean) * rstd, w[k], b[k]);
                if (GATED) v[k] *= z[k] * sigmoid<FULL>(z[k]);
            }
            *(W *)(y + (int64_t)vec * V) = R::P::down(v);
        }
    };
    if constexpr (IMAGE) {
        const int64_t all = P.rows / P.inner * lay.tiles;
        for (int64_t t = blockIdx.x; t < all; t += gridDim.x) {
            const int64_t o = t / lay.tiles, p0 = t % lay.tiles * lay.P;
            const int n = (int)min((int64_t)lay.P, P.inner - p0);
            move_tile<DT, true>(tile, lay, (T *)P.x + o * P.x_os + p0, P.x_cs, P.dim, n);
            __syncthreads();
            for (int p = g; p < (n + groups - 1) / groups * groups; p += groups) work(o * P.inner + p0 + p, nullptr, p, p < n);
            __syncthreads();
        }
    } else {
        for (int64_t r = (int64_t)blockIdx.x * groups; r < P.rows; r += (int64_t)gridDim.x * groups) work(r + g, (const T *)P.x, 0, r + g < P.rows);
    }
}

template <int DT, int V, int NV, bool GATED, bool IMAGE>
__global__ void __launch_bounds__(NT, 2) norm_bwd(const Norm P, const Layout lay) {
    using R = Row<DT, V, NV>;
    using W = typename R::W;
    using T = typename Elem<DT>::T;
    constexpr bool FULL = DT == CS2D_F32;
    extern __shared__ __align__(16) unsigned char tile[];
    __shared__ float2 slots[2][NWARP];
    Reduce sum{slots, lay.T, 0};
    const int TL = lay.T, l = threadIdx.x % TL, g = threadIdx.x / TL, groups = NT / TL, nvec = P.dim / V;
    const float inv = 1.f / P.dim;
    float dw[NV][V], db[NV][V];
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int k = 0; k < V; ++k) dw[j][k] = db[j][k] = 0.f;
    auto work = [&](int64_t row, int p, bool on) {
        W xw[NV], dw_[NV], zw[GATED ? NV : 1];
        const int64_t o = on ? row / P.inner : 0, i = on ? row % P.inner : 0;
        if constexpr (IMAGE) {
#pragma unroll
            for (int j = 0; j < NV; ++j)
                xw[j] = on && j * TL + l < nvec ? *(const W *)element<sizeof(T)>(tile, lay.pitch, p, (j * TL + l) * V) : W{};
        } else {
            R::load(xw, (const T *)P.x + o * P.x_os + i * P.x_is, l, TL, nvec, on);
        }
        R::load(dw_, (const T *)P.dy + o * P.dy_os + i * P.dy_is, l, TL, nvec, on);
        if constexpr (GATED) R::load(zw, (const T *)P.gate + o * P.g_os + i * P.g_is, l, TL, nvec, on);
        const float2 st = on ? ((const float2 *)P.stats)[row] : make_float2(0.f, 0.f);
        float xh[NV][V], t[NV][V], s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int vec = j * TL + l;
            const bool here = on && vec < nvec;
            float w[V], b[V], z[V], dz[V];
            R::P::up(xw[j], xh[j]);
            R::P::up(dw_[j], t[j]);
            if constexpr (GATED) R::P::up(zw[j], z);
            params<V>(w, here ? P.weight : nullptr, P.wtype, vec * V, 1.f);
            if constexpr (GATED) params<V>(b, here ? P.bias : nullptr, P.wtype, vec * V, 0.f);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float h = here ? (xh[j][k] - st.x) * st.y : 0.f;
                float d = t[j][k];
                if constexpr (GATED) {
                    const float sg = sigmoid<FULL>(z[k]), silu = z[k] * sg, n = fmaf(h, w[k], b[k]);
                    dz[k] = d * n * fmaf(silu, 1.f - sg, sg);
                    d *= silu;
                }
                db[j][k] += d;
                dw[j][k] = fmaf(d, h, dw[j][k]);
                d *= w[k];
                s1 += d;
                s2 = fmaf(d, h, s2);
                xh[j][k] = h;
                t[j][k] = d;
            }
            if constexpr (GATED)
                if (here) *(W *)((T *)P.dgate + row * P.dim + (int64_t)vec * V) = R::P::down(dz);
        }
        const float2 s = sum(s1, s2);
        s1 = s.x * inv;
        s2 = s.y * inv;
        if (!on) return;
        T *dx = (T *)P.dx + o * P.dx_os + i * P.dx_is;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int vec = j * TL + l;
            if (vec >= nvec) continue;
            float v[V];
#pragma unroll
            for (int k = 0; k < V; ++k) v[k] = st.y * (t[j][k] - s1 - xh[j][k] * s2);
            if constexpr (IMAGE) *(W *)element<sizeof(T)>(tile, lay.pitch, p, vec * V) = R::P::down(v);
            else *(W *)(dx + (int64_t)vec * V) = R::P::down(v);
        }
    };
    if constexpr (IMAGE) {
        const int64_t all = P.rows / P.inner * lay.tiles;
        for (int64_t t = blockIdx.x; t < all; t += gridDim.x) {
            const int64_t o = t / lay.tiles, p0 = t % lay.tiles * lay.P;
            const int n = (int)min((int64_t)lay.P, P.inner - p0);
            move_tile<DT, true>(tile, lay, (T *)P.x + o * P.x_os + p0, P.x_cs, P.dim, n);
            __syncthreads();
            for (int p = g; p < (n + groups - 1) / groups * groups; p += groups) work(o * P.inner + p0 + p, p, p < n);
            __syncthreads();
            move_tile<DT, false>(tile, lay, (T *)P.dx + o * P.dx_os + p0, P.dx_cs, P.dim, n);
            __syncthreads();
        }
    } else {
        for (int64_t r = (int64_t)blockIdx.x * groups; r < P.rows; r += (int64_t)gridDim.x * groups) work(r + g, 0, r + g < P.rows);
    }
    if (!P.part) return;
    // the CTA's sums: over the rows of a warp by shuffles, over the groups one after the other
    for (int off = TL; off < 32; off <<= 1) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                dw[j][k] += __shfl_xor_sync(~0u, dw[j][k], off);
                db[j][k] += __shfl_xor_sync(~0u, db[j][k], off);
            }
    }
    const int per = TL < 32 ? 32 : TL, turns = NT / per;   // threads of a turn
    float *acc = (float *)tile;
    for (int turn = 0; turn < turns; ++turn) {
        __syncthreads();
        if ((int)threadIdx.x / per != turn || (int)threadIdx.x % per >= TL) continue;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int vec = j * TL + l;
            if (vec >= nvec) continue;
#pragma unroll
            for (int k = 0; k < V; ++k) {
                float *aw = acc + vec * V + k, *ab = aw + P.dim;
                *aw = turn ? *aw + dw[j][k] : dw[j][k];
                *ab = turn ? *ab + db[j][k] : db[j][k];
            }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * P.dim; i += NT) P.part[(int64_t)blockIdx.x * 2 * P.dim + i] = acc[i];
}

// ---- launches ----------------------------------------------------------------------------------------------------
template <class K> cudaError_t start(K *kernel, const Norm &P, const Layout &l, size_t smem, cudaStream_t st) {
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
    }
    kernel<<<l.grid, NT, smem, st>>>(P, l);
    return cudaGetLastError();
}
template <bool BWD, int DT, int V, int NV> cudaError_t go(const Norm &P, const Layout &l, size_t smem, cudaStream_t st) {
    const bool image = l.P > 0;
    if constexpr (BWD) {
        if (P.gate) return image ? start(norm_bwd<DT, V, NV, true, true>, P, l, smem, st) : start(norm_bwd<DT, V, NV, true, false>, P, l, smem, st);
        return image ? start(norm_bwd<DT, V, NV, false, true>, P, l, smem, st) : start(norm_bwd<DT, V, NV, false, false>, P, l, smem, st);
    } else {
        if (P.gate) return image ? start(norm_fwd<DT, V, NV, true, true>, P, l, smem, st) : start(norm_fwd<DT, V, NV, true, false>, P, l, smem, st);
        return image ? start(norm_fwd<DT, V, NV, false, true>, P, l, smem, st) : start(norm_fwd<DT, V, NV, false, false>, P, l, smem, st);
    }
}
template <bool BWD, int DT> cudaError_t launch(const Norm &P, const Layout &l, int v, int nv, size_t smem, cudaStream_t st) {
    constexpr int V = DT == CS2D_F32 ? 4 : 8;
    if (v == V) switch (nv) {
            case 1: return go<BWD, DT, V, 1>(P, l, smem, st);
            case 2: return go<BWD, DT, V, 2>(P, l, smem, st);
            case 3: return go<BWD, DT, V, 3>(P, l, smem, st);
            case 6: if constexpr (DT == CS2D_F32) return go<BWD, DT, V, 6>(P, l, smem, st);
        }
    else switch (nv) {
            case 4: return go<BWD, DT, 1, 4>(P, l, smem, st);
            case 12: return go<BWD, DT, 1, 12>(P, l, smem, st);
            case 24: return go<BWD, DT, 1, 24>(P, l, smem, st);
        }
    return cudaErrorInvalidValue;
}
cudaError_t fwd_f32(const Norm &P, const Layout &l, int v, int nv, size_t smem, cudaStream_t st);
cudaError_t fwd_f16(const Norm &P, const Layout &l, int v, int nv, size_t smem, cudaStream_t st);
cudaError_t fwd_bf16(const Norm &P, const Layout &l, int v, int nv, size_t smem, cudaStream_t st);
cudaError_t bwd_f32(const Norm &P, const Layout &l, int v, int nv, size_t smem, cudaStream_t st);
cudaError_t bwd_f16(const Norm &P, const Layout &l, int v, int nv, size_t smem, cudaStream_t st);
cudaError_t bwd_bf16(const Norm &P, const Layout &l, int v, int nv, size_t smem, cudaStream_t st);

}  // namespace nm

}  // namespace cs2d
