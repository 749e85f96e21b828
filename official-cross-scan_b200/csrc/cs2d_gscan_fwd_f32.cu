#include "cs2d_gscan_fwd.cuh"

namespace cs2d { namespace gs { cudaError_t fwd_f32(const GScan &P, cudaStream_t st) { return fwd<CS2D_F32>(P, st); } } }
