#include "cs2d_norm.cuh"

namespace cs2d { namespace nm { cudaError_t bwd_f32(const Norm &P, const Layout &l, int v, int nv, size_t smem, cudaStream_t st) { return launch<true, CS2D_F32>(P, l, v, nv, smem, st); } } }
