// Operators over tokens: arguments of the kernels, element types, the gate's functions.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <cstring>

#include "../../include/cs2d.h"
#include "cs2d_status.h"

namespace cs2d {

// ---- gated scan ------------------------------------------------------------------------------------------
// Units of work: a batch row and a block of channels.  Rows are tokens.
struct GScan {
    int batch, dim, nblk, nseq, form, weighted, off64;
    int64_t units, length, nck;
    const void *u, *gate, *dy, *offsets;
    const float *h0, *dlast;
    void *y, *du, *dgate;
    float *last, *dh0, *ckpt, *h;   // ckpt: [batch][nck][dim], the state before rows GS_CK, 2 GS_CK, ...; h: the step's state
    int2 *map;                      // packed: per row the sequence that starts there and the one that ends there (SEQ_NONE, SEQ_OUTSIDE)
    int64_t u_bs, u_ls, g_bs, g_ls, dy_bs, dy_ls, y_bs, y_ls, h0_bs, h_bs, dlast_bs;
    int io, io_out;                 // how rows are read and written: GS_CHUNKS, GS_WORDS, GS_ELEMENTS
    int *status;
};
enum { SEQ_NONE = -1, SEQ_OUTSIDE = -2 };
enum { GS_CHUNKS = 0, GS_WORDS = 1, GS_ELEMENTS = 2 };   // 16 bytes, 4 bytes, one 16-bit channel at a time

constexpr int GS_CK = 32;       // rows between two checkpoints: a multiple of the rows of a warp in the backward

cudaError_t launch_gscan_map(const GScan &P, cudaStream_t st);
cudaError_t launch_gscan_fwd(const GScan &P, int dt, cudaStream_t st);
cudaError_t launch_gscan_bwd(const GScan &P, int dt, cudaStream_t st);
cudaError_t launch_gscan_step(const GScan &P, int dt, cudaStream_t st);

// ---- layer norm --------------------------------------------------------------------------------------------
// x of (outer, inner, dim): row = outer * inner + i; the channel stride of x and dx is 1 (tokens) or the position stride is (image).
struct Norm {
    int dim, wtype;              // wtype: cs2d_dtype of weight and bias
    int64_t rows, inner;
    const void *x, *gate, *dy, *weight, *bias;
    void *y, *dx, *dgate, *dweight, *dbias;
    float *stats;                // [rows][2]: mean, 1 / standard deviation
    float *part;                 // backward: [parts][2][dim]
    int parts;
    int64_t x_os, x_is, x_cs, g_os, g_is, dy_os, dy_is, dx_os, dx_is, dx_cs;
    float eps;
};
int norm_parts(const Norm &P, int dt);
cudaError_t launch_norm_fwd(const Norm &P, int dt, cudaStream_t st);
cudaError_t launch_norm_bwd(const Norm &P, int dt, cudaStream_t st, int *launches);

// ---- element types ---------------------------------------------------------------------------------------
template <int DT> struct Elem;
template <> struct Elem<CS2D_F32> {
    using T = float;
    static __device__ __forceinline__ float up(T v) { return v; }
    static __device__ __forceinline__ T down(float v) { return v; }
};
template <> struct Elem<CS2D_F16> {
    using T = __half;
    static __device__ __forceinline__ float up(T v) { return __half2float(v); }
    static __device__ __forceinline__ T down(float v) { return __float2half_rn(v); }
};
template <> struct Elem<CS2D_BF16> {
    using T = __nv_bfloat16;
    static __device__ __forceinline__ float up(T v) { return __bfloat162float(v); }
    static __device__ __forceinline__ T down(float v) { return __float2bfloat16_rn(v); }
};

// The word that so many bytes are loaded and stored as
template <int BYTES> struct WordOf;
template <> struct WordOf<2> { using W = uint16_t; };
template <> struct WordOf<4> { using W = uint32_t; };
template <> struct WordOf<8> { using W = uint2; };
template <> struct WordOf<16> { using W = uint4; };

// ---- the gate: its factor a and c = 1 - a, each to a few units of its own last place ---------------------------
// FULL: for fp32 inputs; 16-bit ones take the hardware's exponential and reciprocal (denormals flushed).
__device__ __forceinline__ float ex2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <bool FULL> __device__ __forceinline__ float exp_of(float x) { return FULL ? expf(x) : ex2_fast(x * 1.4426950408889634f); }
template <bool FULL> __device__ __forceinline__ float over(float x, float y) { return FULL ? x / y : x * rcp_fast(y); }

// a = 1 / (1 + exp(-g)).  The smaller of a and c is computed, the larger one is one less it: both keep their own digits, and a
// product of thousands of factors next to one does not drift (an approximate reciprocal next to one would).
template <bool FULL> __device__ __forceinline__ void gate_sigmoid(float g, float &a, float &c) {
    const float t = exp_of<FULL>(-fabsf(g));
    const float small = over<FULL>(t, 1.f + t), large = 1.f - small;
    a = g > 0.f ? large : small;
    c = g > 0.f ? small : large;
}
// a = exp(g), c = -expm1(g).  Near zero the Taylor series of expm1 (next term below 2e-8 of it for |g| <= 0.35) gives both.
template <bool FULL> __device__ __forceinline__ void gate_log(float g, float &a, float &c) {
    float p = 1.f / 5040.f;
    p = fmaf(p, g, 1.f / 720.f);
    p = fmaf(p, g, 1.f / 120.f);
    p = fmaf(p, g, 1.f / 24.f);
    p = fmaf(p, g, 1.f / 6.f);
    p = fmaf(p, g, 0.5f);
    const float m = fmaf(p * g, g, g), e = exp_of<FULL>(g);
    const bool near = fabsf(g) <= 0.35f;
    a = near ? 1.f + m : e;
    c = near ? -m : 1.f - e;
}
template <int FORM, bool FULL> __device__ __forceinline__ void gate_values(float g, float &a, float &c) {
    if constexpr (FORM == CS2D_GATE_SIGMOID) gate_sigmoid<FULL>(g, a, c);
    else if constexpr (FORM == CS2D_GATE_LOG) gate_log<FULL>(g, a, c);
    else { a = g; c = 1.f - g; }
}
template <bool FULL> __device__ __forceinline__ float sigmoid(float z) {
    const float t = exp_of<FULL>(-fabsf(z)), small = over<FULL>(t, 1.f + t);
    return z > 0.f ? 1.f - small : small;
}

}  // namespace cs2d
