// Gated scan: the kernels' launches by type; the step of one token; the row map of packed sequences.
#include "cs2d_gscan.cuh"

namespace cs2d {

namespace gs {

cudaError_t fwd_f32(const GScan &P, cudaStream_t st);
cudaError_t fwd_f16(const GScan &P, cudaStream_t st);
cudaError_t fwd_bf16(const GScan &P, cudaStream_t st);
cudaError_t bwd_f32(const GScan &P, cudaStream_t st);
cudaError_t bwd_f16(const GScan &P, cudaStream_t st);
cudaError_t bwd_bf16(const GScan &P, cudaStream_t st);

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

}  // namespace gs

cudaError_t launch_gscan_map(const GScan &P, cudaStream_t st) {
    gs::gscan_map<<<(unsigned)((P.length + 255) / 256), 256, 0, st>>>(P);
    return cudaGetLastError();
}
cudaError_t launch_gscan_fwd(const GScan &P, int dt, cudaStream_t st) {
    switch (dt) {
        case CS2D_F32: return gs::fwd_f32(P, st);
        case CS2D_F16: return gs::fwd_f16(P, st);
        default: return gs::fwd_bf16(P, st);
    }
}
cudaError_t launch_gscan_bwd(const GScan &P, int dt, cudaStream_t st) {
    switch (dt) {
        case CS2D_F32: return gs::bwd_f32(P, st);
        case CS2D_F16: return gs::bwd_f16(P, st);
        default: return gs::bwd_bf16(P, st);
    }
}
cudaError_t launch_gscan_step(const GScan &P, int dt, cudaStream_t st) {
    const unsigned grid = (unsigned)(((int64_t)P.batch * P.dim + 255) / 256);
    switch (dt) {
        case CS2D_F32: gs::gscan_step<CS2D_F32><<<grid, 256, 0, st>>>(P); break;
        case CS2D_F16: gs::gscan_step<CS2D_F16><<<grid, 256, 0, st>>>(P); break;
        default: gs::gscan_step<CS2D_BF16><<<grid, 256, 0, st>>>(P);
    }
    return cudaGetLastError();
}

}  // namespace cs2d
