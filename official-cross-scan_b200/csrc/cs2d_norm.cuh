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
//
// A lane holds up to 24 channels: what a row costs beside its channels (addresses, shuffles) is paid once for all of them, and 192 * 2^k channels leave
// no lane idle.  The backward with a gate and that of images hold 16, since the sums of dw and db take as many registers again (fp32 B25088 D768 gated:
// 123 us with 8 fp32 channels per lane, 143 with 12).  What bounds it is latency at 15 to 29 warps per SM (128 to 64 registers; ncu) and the
// instructions per row.  Measured: 100352 x 192 bf16 forward 25 us (48 % of the HBM copy rate), backward 41 (43 %); 25088 x 768 fp32 gated 57 (62 %)
// and 123 (48 %); B16 D384 128x128 bf16 gated image 145 (63 %) and 328 (47 %).
#pragma once

#include <atomic>
#include <cstring>

#include "cs2d_seq.cuh"

namespace cs2d {

namespace nm {

constexpr int NT = 256;       // threads of a CTA
constexpr int NWARP = NT / 32;

struct Layout {
    int T, P, pitch;             // lanes of a row; rows of a tile; images: bytes between them in shared memory
    bool image, whole;           // whole: tiles are read in 16-byte chunks
    int64_t tiles, tiles_all;    // of an outer index; in all
    int grid;
};

__device__ __forceinline__ float param(const void *p, int dt, int i, float none) {
    if (!p) return none;
    return dt == CS2D_F32 ? ((const float *)p)[i] : dt == CS2D_F16 ? __half2float(((const __half *)p)[i]) : __bfloat162float(((const __nv_bfloat16 *)p)[i]);
}

// Pairs of fp32 values, which one packed instruction serves
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
template <int DT> __device__ __forceinline__ float2 pair_up(unsigned w) {
    if constexpr (DT == CS2D_BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    __half2 h;
    memcpy(&h, &w, 4);
    return __half22float2(h);
}
template <int DT> __device__ __forceinline__ unsigned pair_down(float2 v) {
    unsigned w;
    if constexpr (DT == CS2D_BF16) {
        const __nv_bfloat162 t = __float22bfloat162_rn(v);
        memcpy(&w, &t, 4);
    } else {
        const __half2 t = __float22half2_rn(v);
        memcpy(&w, &t, 4);
    }
    return w;
}

// A lane's channels of a row: NV vectors of V elements, vector j of lane l being number j T + l of the row; H pairs of values.
template <int DT, int V, int NV> struct Row {
    using T = typename Elem<DT>::T;
    using W = typename WordOf<sizeof(T) * V>::W;
    static constexpr int H = NV * V / 2;
    static __device__ __forceinline__ void up(const W (&w)[NV], float2 (&v)[H]) {
        if constexpr (V == 1) {
#pragma unroll
            for (int h = 0; h < H; ++h) {
                T a, b;
                memcpy(&a, &w[2 * h], sizeof(T));
                memcpy(&b, &w[2 * h + 1], sizeof(T));
                v[h] = make_float2(Elem<DT>::up(a), Elem<DT>::up(b));
            }
        } else if constexpr (DT == CS2D_F32) {
#pragma unroll
            for (int j = 0; j < NV; ++j) memcpy(&v[j * 2], &w[j], 16);
        } else {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                unsigned t[V / 2];
                memcpy(t, &w[j], 2 * V);
#pragma unroll
                for (int k = 0; k < V / 2; ++k) v[j * (V / 2) + k] = pair_up<DT>(t[k]);
            }
        }
    }
    // vector j of the values
    static __device__ __forceinline__ W down(const float2 (&v)[H], int j) {
        W w;
        if constexpr (V == 1) {
            const T t = Elem<DT>::down(j & 1 ? v[j / 2].y : v[j / 2].x);
            memcpy(&w, &t, sizeof(T));
        } else if constexpr (DT == CS2D_F32) {
            memcpy(&w, &v[j * 2], 16);
        } else {
            unsigned t[V / 2];
#pragma unroll
            for (int k = 0; k < V / 2; ++k) t[k] = pair_down<DT>(v[j * (V / 2) + k]);
            memcpy(&w, t, 2 * V);
        }
        return w;
    }
    static __device__ __forceinline__ void load(W (&w)[NV], const T *row, int l, int TL, int nvec, bool on) {
#pragma unroll
        for (int j = 0; j < NV; ++j) w[j] = on && j * TL + l < nvec ? *(const W *)(row + (j * TL + l) * V) : W{};
    }
    // weight or bias
    static __device__ __forceinline__ void params(float2 (&v)[H], const void *p, int dt, int l, int TL, int nvec, float none) {
        if (!p) {
#pragma unroll
            for (int h = 0; h < H; ++h) v[h] = both(none);
        } else if (dt == CS2D_F32) {
            constexpr int F = V < 4 ? 1 : 4;   // floats of an access
            float t[NV * V];
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int k = 0; k < V; k += F) {
                    using G = typename WordOf<4 * F>::W;
                    const G g = j * TL + l < nvec ? *(const G *)((const float *)p + (j * TL + l) * V + k) : G{};
                    memcpy(&t[j * V + k], &g, sizeof(g));
                }
#pragma unroll
            for (int h = 0; h < H; ++h) v[h] = make_float2(t[2 * h], t[2 * h + 1]);
        } else {
            W w[NV];
            load(w, (const T *)p, l, TL, nvec, true);
            up(w, v);
        }
    }
};

// Sums of two values over the T lanes of a row.  More than a warp: through shared memory, a named barrier per row group; two sets of
// slots, so that the next sum may begin while others still read.
struct Reduce {
    float2 (*slots)[NWARP];
    int T, parity;
    template <bool TWO> __device__ __forceinline__ float2 of(float a, float b) {
        const int in_warp = T < 32 ? T : 32;
        for (int o = in_warp >> 1; o; o >>= 1) {
            a += __shfl_xor_sync(~0u, a, o);
            if (TWO) b += __shfl_xor_sync(~0u, b, o);
        }
        if (T <= 32) return make_float2(a, b);
        const int warp = threadIdx.x >> 5, R = T / 32, first = warp / R * R;
        if ((threadIdx.x & 31) == 0) slots[parity][warp] = make_float2(a, b);
        asm volatile("bar.sync %0, %1;" ::"r"(1 + warp / R), "r"(T) : "memory");
        float2 s = slots[parity][first];
        for (int k = 1; k < R; ++k) {
            s.x += slots[parity][first + k].x;
            if (TWO) s.y += slots[parity][first + k].y;
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
// U accesses at a time, reads before writes (two single elements count as one): the forward takes 6, the backward, whose sums are in registers
// meanwhile, 4 on the way in and, where no latency is waited for, 1 on the way out (B16 D384 128x128 bf16: 328 us; 4 and 4: 400, 1 and 1: 387).
template <int DT, bool IN, int U> __device__ __forceinline__ void move_tile(unsigned char *tile, const Layout &l, typename Elem<DT>::T *img, int64_t cs, int dim, int n) {
    using T = typename Elem<DT>::T;
    constexpr int ES = sizeof(T);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (ES == 2 && l.whole && l.P % 32 == 0) {
        // a warp takes 8 channels x 32 positions: lane t has 8 positions of channel t / 4.  Word k of the lanes is an 8 x 8 matrix whose column
        // c is position 8 (c / 2) + 2 k + c % 2; its transpose is eight 16-byte chunks, one per position.
        const int m = lane >> 3, c = lane & 7, pm = 8 * (c >> 1) + 2 * m + (c & 1), qm = 8 * (lane & 3);
        const int sh = l.P == 64, all = ((dim + 7) / 8) << sh;   // 128 bytes of a channel by two warps that follow each other
        for (int w0 = warp; w0 < all; w0 += NWARP * U) {
            uint4 v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int w = w0 + u * NWARP, b32 = (w & sh) * 32, d = (w >> sh) * 8 + (lane >> 2);
                const bool ok = w < all && d < dim && qm + b32 < n;
                if (IN) v[u] = ok ? *(const uint4 *)(img + d * cs + qm + b32) : make_uint4(0, 0, 0, 0);
                else if (w < all)
                    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(v[u].x), "=r"(v[u].y), "=r"(v[u].z), "=r"(v[u].w)
                                 : "r"((unsigned)__cvta_generic_to_shared(chunk<ES>(tile, l.pitch, pm + b32, w >> sh))) : "memory");
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int w = w0 + u * NWARP, b32 = (w & sh) * 32, d = (w >> sh) * 8 + (lane >> 2);
                if (w >= all) continue;
                if (IN)
                    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(
                                     (unsigned)__cvta_generic_to_shared(chunk<ES>(tile, l.pitch, pm + b32, w >> sh))),
                                 "r"(v[u].x), "r"(v[u].y), "r"(v[u].z), "r"(v[u].w) : "memory");
                else if (d < dim && qm + b32 < n) *(uint4 *)(img + d * cs + qm + b32) = v[u];
            }
        }
    } else if (ES == 4 && l.whole) {
        const int sh = __ffs(l.P) - 3, all = dim << sh;   // chunks of a channel: P / 4
        for (int i0 = threadIdx.x; i0 < all; i0 += NT * U) {
            float4 v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + u * NT, d = i >> sh, q = (i & ((1 << sh) - 1)) * 4;
                const bool ok = i < all && q < n;
                if (IN) v[u] = ok ? *(const float4 *)(img + d * cs + q) : make_float4(0.f, 0.f, 0.f, 0.f);
                else if (ok) {
                    v[u].x = *(const float *)element<ES>(tile, l.pitch, q, d);
                    v[u].y = *(const float *)element<ES>(tile, l.pitch, q + 1, d);
                    v[u].z = *(const float *)element<ES>(tile, l.pitch, q + 2, d);
                    v[u].w = *(const float *)element<ES>(tile, l.pitch, q + 3, d);
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + u * NT, d = i >> sh, q = (i & ((1 << sh) - 1)) * 4;
                if (i >= all || q >= n) continue;
                if (IN) {
                    *(float *)element<ES>(tile, l.pitch, q, d) = v[u].x;
                    *(float *)element<ES>(tile, l.pitch, q + 1, d) = v[u].y;
                    *(float *)element<ES>(tile, l.pitch, q + 2, d) = v[u].z;
                    *(float *)element<ES>(tile, l.pitch, q + 3, d) = v[u].w;
                } else {
                    *(float4 *)(img + d * cs + q) = v[u];
                }
            }
        }
    } else {
        constexpr int N = 2 * U;
        const int sh = __ffs(l.P) - 1, all = dim << sh;
        for (int i0 = threadIdx.x; i0 < all; i0 += NT * N) {
            T v[N];
#pragma unroll
            for (int u = 0; u < N; ++u) {
                const int i = i0 + u * NT, d = i >> sh, p = i & (l.P - 1);
                if (i < all && p < n) v[u] = IN ? img[d * cs + p] : *(const T *)element<ES>(tile, l.pitch, p, d);
            }
#pragma unroll
            for (int u = 0; u < N; ++u) {
                const int i = i0 + u * NT, d = i >> sh, p = i & (l.P - 1);
                if (i >= all || p >= n) continue;
                if (IN) *(T *)element<ES>(tile, l.pitch, p, d) = v[u];
                else img[d * cs + p] = v[u];
            }
        }
    }
}

// ---- kernels ---------------------------------------------------------------------------------------------------
// CTAs go through tiles of P rows of an outer index.
struct Tile {
    int64_t o, i, row;   // outer index, first row of it, first row of all
    int n;               // rows that are there
    __device__ __forceinline__ Tile(const Norm &P, const Layout &l, int64_t t) {
        o = l.tiles_all == l.tiles ? 0 : (unsigned)t / (unsigned)l.tiles;
        i = (t - o * l.tiles) * l.P;
        row = o * P.inner + i;
        n = (int)min((int64_t)l.P, P.inner - i);
    }
};

// CTAs that an SM is to hold: the lane's values, a parameter's and the gate's, and 25 registers more
template <int DT, int V, int NV, bool GATED> constexpr int FWD_CTAS = NV * V <= 8 && V > 1 ? 6 : NV * V < 16 ? 4 : GATED && (DT == CS2D_F32 || V == 1) ? 2 : 3;

template <int DT, int V, int NV, bool GATED, bool IMAGE>
__global__ void __launch_bounds__(NT, (FWD_CTAS<DT, V, NV, GATED>)) norm_fwd(const Norm P, const Layout lay) {
    using R = Row<DT, V, NV>;
    using W = typename R::W;
    using T = typename R::T;
    constexpr bool FULL = DT == CS2D_F32;
    constexpr int H = R::H;
    extern __shared__ __align__(16) unsigned char tile[];
    __shared__ float2 slots[2][NWARP];
    Reduce sum{slots, lay.T, 0};
    const int TL = lay.T, l = threadIdx.x % TL, g = threadIdx.x / TL, groups = NT / TL, nvec = P.dim / V;
    const float inv = 1.f / P.dim;
    const int64_t x_step = groups * P.x_is, z_step = groups * P.g_is;
    for (int64_t t = blockIdx.x; t < lay.tiles_all; t += gridDim.x) {
        const Tile tl(P, lay, t);
        if constexpr (IMAGE) {
            move_tile<DT, true, 6>(tile, lay, (T *)P.x + tl.o * P.x_os + tl.i, P.x_cs, P.dim, tl.n);
            __syncthreads();
        }
        const T *xp = (const T *)P.x + tl.o * P.x_os + (tl.i + g) * P.x_is, *zp = (const T *)P.gate + tl.o * P.g_os + (tl.i + g) * P.g_is;
        for (int p0 = 0; p0 < tl.n; p0 += groups) {
            const int p = p0 + g;
            const bool on = p < tl.n;
            W xw[NV], zw[GATED ? NV : 1];
            if constexpr (IMAGE) {
#pragma unroll
                for (int j = 0; j < NV; ++j)
                    xw[j] = on && j * TL + l < nvec ? *(const W *)element<sizeof(T)>(tile, lay.pitch, p, (j * TL + l) * V) : W{};
            } else {
                R::load(xw, xp, l, TL, nvec, on);
                xp += x_step;
            }
            if constexpr (GATED) {
                R::load(zw, zp, l, TL, nvec, on);
                zp += z_step;
            }
            float2 x[H], s = both(0.f);
            R::up(xw, x);
#pragma unroll
            for (int h = 0; h < H; ++h) s = add2(s, x[h]);
            const float mean = sum.of<false>(s.x + s.y, 0.f).x * inv;
            s = both(0.f);
#pragma unroll
            for (int j = 0; j < NV; ++j) {   // what lies behind the last channel stays out of the variance
                const bool here = j * TL + l < nvec;
                if constexpr (V == 1) {
                    float &v = j & 1 ? x[j / 2].y : x[j / 2].x;
                    v = here ? v - mean : 0.f;
                    s.x = fmaf(v, v, s.x);
                } else {
#pragma unroll
                    for (int k = 0; k < V / 2; ++k) {
                        float2 &v = x[j * V / 2 + k];
                        v = add2(v, both(-mean));
                        if (here) s = fma2(v, v, s);
                    }
                }
            }
            const float rstd = rsqrtf(sum.of<false>(s.x + s.y, 0.f).x * inv + P.eps);
            if (!on) continue;
            if (P.stats && l == 0) ((float2 *)P.stats)[tl.row + p] = make_float2(mean, rstd);
            float2 w[H];
            R::params(w, P.weight, P.wtype, l, TL, nvec, 1.f);
#pragma unroll
            for (int h = 0; h < H; ++h) x[h] = mul2(x[h], mul2(w[h], both(rstd)));
            R::params(w, P.bias, P.wtype, l, TL, nvec, 0.f);
#pragma unroll
            for (int h = 0; h < H; ++h) x[h] = add2(x[h], w[h]);
            if constexpr (GATED) {
                R::up(zw, w);
#pragma unroll
                for (int h = 0; h < H; ++h) x[h] = mul2(x[h], mul2(w[h], make_float2(sigmoid<FULL>(w[h].x), sigmoid<FULL>(w[h].y))));
            }
            T *y = (T *)P.y + (tl.row + p) * P.dim;
#pragma unroll
            for (int j = 0; j < NV; ++j)
                if (j * TL + l < nvec) *(W *)(y + (j * TL + l) * V) = R::down(x, j);
        }
        if constexpr (IMAGE) __syncthreads();
    }
}

template <int DT, int V, int NV, bool GATED> constexpr int BWD_CTAS = V == 1 ? 2 : NV * V <= 8 ? 4 : NV * V <= 12 ? 3 : 2;   // single elements take registers for their addresses
// Rows are copied to shared memory one row ahead: every lane copies the vectors that it will read itself, so nobody waits for others.
template <int BYTES> __device__ __forceinline__ void copy_async(void *dst, const void *src) {
    const unsigned d = (unsigned)__cvta_generic_to_shared(dst);
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(d), "l"(src), "n"(BYTES) : "memory");
}
template <int DT, int V> constexpr int VEC_BYTES = V * (DT == CS2D_F32 ? 4 : 2);   // of an access; single 16-bit elements are not copied ahead
template <int DT, int V, int NV, bool GATED, bool IMAGE> constexpr int STAGE_BYTES = VEC_BYTES<DT, V> < 4 ? 0 : NT * (VEC_BYTES<DT, V> * NV * (1 + GATED + !IMAGE) + 8);   // one row ahead, per CTA

template <int DT, int V, int NV, bool GATED, bool IMAGE>
__global__ void __launch_bounds__(NT, (BWD_CTAS<DT, V, NV, GATED>)) norm_bwd(const Norm P, const Layout lay) {
    using R = Row<DT, V, NV>;
    using W = typename R::W;
    using T = typename R::T;
    constexpr bool FULL = DT == CS2D_F32, AHEAD = VEC_BYTES<DT, V> >= 4;
    constexpr int H = R::H, VB = VEC_BYTES<DT, V>, STAGE = STAGE_BYTES<DT, V, NV, GATED, IMAGE>;
    extern __shared__ __align__(16) unsigned char smem[];
    unsigned char *tile = smem + 2 * STAGE;
    __shared__ float2 slots[2][NWARP];
    Reduce sum{slots, lay.T, 0};
    const int TL = lay.T, l = threadIdx.x % TL, g = threadIdx.x / TL, groups = NT / TL, nvec = P.dim / V;
    const float inv = 1.f / P.dim;
    const int64_t x_step = groups * P.x_is, z_step = groups * P.g_is, d_step = groups * P.dy_is;
    // the lane's vectors in a stage: stats, dy, z, x
    auto vec_at = [&](int stage, int k, int j) { return (W *)(smem + stage * STAGE + NT * 8 + ((k * NV + j) * NT + threadIdx.x) * VB); };
    auto stat_at = [&](int stage) { return (float2 *)(smem + stage * STAGE + threadIdx.x * 8); };
    // the row that is copied next
    const T *xp = nullptr, *dp = nullptr, *zp = nullptr;
    const float2 *sp = nullptr;
    int p_next = 0, n_next = 0;
    int64_t t_next = blockIdx.x;
    auto enter = [&]() {   // the first row of tile t_next
        p_next = n_next = 0;
        if (t_next >= lay.tiles_all) return;
        const Tile tl(P, lay, t_next);
        n_next = tl.n;
        xp = (const T *)P.x + tl.o * P.x_os + (tl.i + g) * P.x_is + l * V;
        dp = (const T *)P.dy + tl.o * P.dy_os + (tl.i + g) * P.dy_is + l * V;
        zp = (const T *)P.gate + tl.o * P.g_os + (tl.i + g) * P.g_is + l * V;
        sp = (const float2 *)P.stats + tl.row + g;
        t_next += gridDim.x;
    };
    auto ahead = [&](int stage) {
        if constexpr (AHEAD) if (p_next + g < n_next) {
            copy_async<8>(stat_at(stage), sp);
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                if (j * TL + l >= nvec) continue;
                copy_async<VB>(vec_at(stage, 0, j), dp + j * TL * V);
                if (GATED) copy_async<VB>(vec_at(stage, 1, j), zp + j * TL * V);
                if (!IMAGE) copy_async<VB>(vec_at(stage, 1 + GATED, j), xp + j * TL * V);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        p_next += groups;
        sp += groups;
        dp += d_step;
        if (GATED) zp += z_step;
        if (!IMAGE) xp += x_step;
        if (p_next >= n_next) enter();
    };
    float2 dw[H], db[H];
#pragma unroll
    for (int h = 0; h < H; ++h) dw[h] = db[h] = both(0.f);
    int stage = 0;
    if (AHEAD) {
        enter();
        ahead(0);
    }
    for (int64_t t = blockIdx.x; t < lay.tiles_all; t += gridDim.x) {
        const Tile tl(P, lay, t);
        if constexpr (IMAGE) {
            move_tile<DT, true, 4>(tile, lay, (T *)P.x + tl.o * P.x_os + tl.i, P.x_cs, P.dim, tl.n);
            __syncthreads();
        }
        T *zo = (T *)P.dgate + (tl.row + g) * P.dim + l * V, *xo = (T *)P.dx + tl.o * P.dx_os + (tl.i + g) * P.dx_is + l * V;
        for (int p0 = 0; p0 < tl.n; p0 += groups, zo += groups * (int64_t)P.dim, xo += groups * P.dx_is) {
            const int p = p0 + g;
            const bool on = p < tl.n;
            if (AHEAD) {
                ahead(stage ^ 1);
                asm volatile("cp.async.wait_group 1;" ::: "memory");
            }
            auto fetch = [&](W (&w)[NV], int k, const T *row) {
                if constexpr (AHEAD) {
#pragma unroll
                    for (int j = 0; j < NV; ++j) w[j] = on && j * TL + l < nvec ? *vec_at(stage, k, j) : W{};
                } else {
                    R::load(w, row, l, TL, nvec, on);
                }
            };
            W xw[NV], ww[NV];
            if constexpr (IMAGE) {
#pragma unroll
                for (int j = 0; j < NV; ++j)
                    xw[j] = on && j * TL + l < nvec ? *(const W *)element<sizeof(T)>(tile, lay.pitch, p, (j * TL + l) * V) : W{};
            } else {
                fetch(xw, 1 + GATED, (const T *)P.x + tl.o * P.x_os + (tl.i + p) * P.x_is);
            }
            const float2 st = !on ? both(0.f) : AHEAD ? *stat_at(stage) : ((const float2 *)P.stats)[tl.row + p];
            float2 h[H], d[H], w[H];
            R::up(xw, h);
#pragma unroll
            for (int k = 0; k < H; ++k) h[k] = mul2(add2(h[k], both(-st.x)), both(st.y));
            fetch(ww, 0, (const T *)P.dy + tl.o * P.dy_os + (tl.i + p) * P.dy_is);
            R::up(ww, d);
            R::params(w, P.weight, P.wtype, l, TL, nvec, 1.f);
            if constexpr (GATED) {
                float2 z[H], b[H];
                fetch(ww, 1, (const T *)P.gate + tl.o * P.g_os + (tl.i + p) * P.g_is);
                R::up(ww, z);
                R::params(b, P.bias, P.wtype, l, TL, nvec, 0.f);
#pragma unroll
                for (int k = 0; k < H; ++k) {
                    const float2 sg = make_float2(sigmoid<FULL>(z[k].x), sigmoid<FULL>(z[k].y)), silu = mul2(z[k], sg);
                    const float2 slope = fma2(silu, add2(both(1.f), make_float2(-sg.x, -sg.y)), sg);
                    z[k] = mul2(mul2(d[k], fma2(h[k], w[k], b[k])), slope);
                    d[k] = mul2(d[k], silu);
                }
                if (on) {
#pragma unroll
                    for (int j = 0; j < NV; ++j)
                        if (j * TL + l < nvec) *(W *)(zo + j * TL * V) = R::down(z, j);
                }
            }
            // (rows and channels that are not there have dy = 0)
            float2 s1 = both(0.f), s2 = both(0.f);
#pragma unroll
            for (int k = 0; k < H; ++k) {
                db[k] = add2(db[k], d[k]);
                dw[k] = fma2(d[k], h[k], dw[k]);
                d[k] = mul2(d[k], w[k]);
                s1 = add2(s1, d[k]);
                s2 = fma2(d[k], h[k], s2);
            }
            const float2 s = sum.of<true>(s1.x + s1.y, s2.x + s2.y);
            stage ^= 1;
            if (!on) continue;
            const float2 rs = both(st.y), c1 = both(-st.y * s.x * inv), c2 = both(-st.y * s.y * inv);
#pragma unroll
            for (int k = 0; k < H; ++k) d[k] = fma2(h[k], c2, fma2(d[k], rs, c1));
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int vec = j * TL + l;
                if (vec >= nvec) continue;
                if constexpr (IMAGE) *(W *)element<sizeof(T)>(tile, lay.pitch, p, vec * V) = R::down(d, j);
                else *(W *)(xo + j * TL * V) = R::down(d, j);
            }
        }
        if constexpr (IMAGE) {
            __syncthreads();
            move_tile<DT, false, 1>(tile, lay, (T *)P.dx + tl.o * P.dx_os + tl.i, P.dx_cs, P.dim, tl.n);
            __syncthreads();
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (!P.part) return;
    // the CTA's sums: over the rows of a warp by shuffles, over the groups one after the other
    for (int off = TL; off < 32; off <<= 1) {
#pragma unroll
        for (int h = 0; h < H; ++h) {
            dw[h] = add2(dw[h], make_float2(__shfl_xor_sync(~0u, dw[h].x, off), __shfl_xor_sync(~0u, dw[h].y, off)));
            db[h] = add2(db[h], make_float2(__shfl_xor_sync(~0u, db[h].x, off), __shfl_xor_sync(~0u, db[h].y, off)));
        }
    }
    const int per = TL < 32 ? 32 : TL, turns = NT / per;   // threads of a turn
    float *acc = (float *)smem;
    for (int turn = 0; turn < turns; ++turn) {
        __syncthreads();
        if ((int)threadIdx.x / per != turn || (int)threadIdx.x % per >= TL) continue;
#pragma unroll
        for (int e = 0; e < NV * V; ++e) {
            const int vec = e / V * TL + l;
            if (vec >= nvec) continue;
            float *aw = acc + vec * V + e % V, *ab = aw + P.dim;
            const float vw = e & 1 ? dw[e / 2].y : dw[e / 2].x, vb = e & 1 ? db[e / 2].y : db[e / 2].x;
            *aw = turn ? *aw + vw : vw;
            *ab = turn ? *ab + vb : vb;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * P.dim; i += NT) P.part[(int64_t)blockIdx.x * 2 * P.dim + i] = acc[i];
}

// ---- launches ----------------------------------------------------------------------------------------------------
template <auto KERNEL> cudaError_t start(const Norm &P, const Layout &l, size_t smem, cudaStream_t st) {
    static std::atomic<bool> done[64] = {};   // per device; threads that come at the same time set the same attribute
    const size_t acc = (size_t)8 * P.dim;   // the backward's sums, in the place of all else
    if (P.dy && smem < acc) smem = acc;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || dev < 0 || dev >= 64) return e != cudaSuccess ? e : cudaErrorInvalidDevice;
    if (!done[dev]) {
        if ((e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, 226 * 1024)) != cudaSuccess) return e;
        done[dev] = true;
    }
    KERNEL<<<l.grid, NT, smem, st>>>(P, l);
    return cudaGetLastError();
}
template <bool BWD, int DT, int V, int NV> cudaError_t go(const Norm &P, const Layout &l, size_t smem, cudaStream_t st) {
    const bool image = l.image;
    if constexpr (BWD) {
        if (P.gate) return image ? start<norm_bwd<DT, V, NV, true, true>>(P, l, smem + 2 * STAGE_BYTES<DT, V, NV, true, true>, st)
                                 : start<norm_bwd<DT, V, NV, true, false>>(P, l, smem + 2 * STAGE_BYTES<DT, V, NV, true, false>, st);
        return image ? start<norm_bwd<DT, V, NV, false, true>>(P, l, smem + 2 * STAGE_BYTES<DT, V, NV, false, true>, st)
                     : start<norm_bwd<DT, V, NV, false, false>>(P, l, smem + 2 * STAGE_BYTES<DT, V, NV, false, false>, st);
    } else {
        if (P.gate) return image ? start<norm_fwd<DT, V, NV, true, true>>(P, l, smem, st) : start<norm_fwd<DT, V, NV, true, false>>(P, l, smem, st);
        return image ? start<norm_fwd<DT, V, NV, false, true>>(P, l, smem, st) : start<norm_fwd<DT, V, NV, false, false>>(P, l, smem, st);
    }
}
template <bool BWD, int DT> cudaError_t launch(const Norm &P, const Layout &l, int v, int nv, size_t smem, cudaStream_t st) {
    constexpr int V = DT == CS2D_F32 ? 4 : 8;
    if (v == V) switch (nv) {
            case 1: return go<BWD, DT, V, 1>(P, l, smem, st);
            case 2: return go<BWD, DT, V, 2>(P, l, smem, st);
            case 3: if constexpr (BWD) return P.gate || l.image ? cudaErrorInvalidValue : start<norm_bwd<DT, V, 3, false, false>>(P, l, smem + 2 * STAGE_BYTES<DT, V, 3, false, false>, st);
                    else return go<BWD, DT, V, 3>(P, l, smem, st);
            case 6: if constexpr (DT == CS2D_F32 && !BWD) return go<BWD, DT, V, 6>(P, l, smem, st);
        }
    else if (v == 2) switch (nv) {
            case 2: if constexpr (DT != CS2D_F32) return go<BWD, DT, 2, 2>(P, l, smem, st);
            case 4: if constexpr (DT != CS2D_F32) return go<BWD, DT, 2, 4>(P, l, smem, st);
            case 6: if constexpr (DT != CS2D_F32) return go<BWD, DT, 2, 6>(P, l, smem, st);
        }
    else switch (nv) {
            case 4: return go<BWD, DT, 1, 4>(P, l, smem, st);
            case 6: return go<BWD, DT, 1, 6>(P, l, smem, st);
            case 8: return go<BWD, DT, 1, 8>(P, l, smem, st);
            case 12: return go<BWD, DT, 1, 12>(P, l, smem, st);
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
