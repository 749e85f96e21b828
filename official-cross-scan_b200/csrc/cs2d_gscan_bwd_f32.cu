#include "cs2d_gscan_bwd.cuh"

namespace cs2d { namespace gs { cudaError_t bwd_f32(const GScan &P, cudaStream_t st) { return bwd<CS2D_F32>(P, st); } } }
