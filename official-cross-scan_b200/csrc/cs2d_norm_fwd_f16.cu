#include "cs2d_norm.cuh"

namespace cs2d { namespace nm { cudaError_t fwd_f16(const Norm &P, const Layout &l, int v, int nv, size_t smem, cudaStream_t st) { return launch<false, CS2D_F16>(P, l, v, nv, smem, st); } } }
