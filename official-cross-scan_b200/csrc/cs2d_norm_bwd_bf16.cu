#include "cs2d_norm.cuh"

namespace cs2d { namespace nm { cudaError_t bwd_bf16(const Norm &P, const Layout &l, int v, int nv, size_t smem, cudaStream_t st) { return launch<true, CS2D_BF16>(P, l, v, nv, smem, st); } } }
