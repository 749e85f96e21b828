#include "cs2d_gscan_bwd.cuh"

namespace cs2d { namespace gs { cudaError_t bwd_f16(const GScan &P, cudaStream_t st) { return bwd<CS2D_F16>(P, st); } } }
