#include "cs2d_gscan_fwd.cuh"

namespace cs2d { namespace gs { cudaError_t fwd_bf16(const GScan &P, cudaStream_t st) { return fwd<CS2D_BF16>(P, st); } } }
