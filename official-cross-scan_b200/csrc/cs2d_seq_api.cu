// extern "C" boundary of the operators over tokens: validation, launch geometry, errors.
#include <initializer_list>

#include "cs2d_host.h"
#include "cs2d_seq.cuh"

namespace cs2d {

static int validate(const cs2d_gscan *p, bool step) {
    if (!p) return fail(CS2D_ERR_INVALID, "problem is NULL");
    if (p->batch <= 0 || p->dim <= 0 || (!step && p->length <= 0)) return fail(CS2D_ERR_INVALID, "all sizes must be positive");
    if (p->io_dtype < CS2D_F32 || p->io_dtype > CS2D_BF16) return fail(CS2D_ERR_INVALID, "input type must be float32, float16 or bfloat16");
    if (p->form < CS2D_GATE_SIGMOID || p->form > CS2D_GATE_DIRECT) return fail(CS2D_ERR_INVALID, "unknown form of the gate: %d", p->form);
    if (!p->u || !p->gate) return fail(CS2D_ERR_INVALID, "u and gate must be given");
    if (step) return CS2D_OK;
    // (the kernels count channels, tokens and sequences in 32 bits, up to a unit's, a cluster's or a search interval's end behind the last one)
    if (p->length > (1 << 30)) return fail(CS2D_ERR_UNSUPPORTED, "more than 2^30 tokens in a row");
    if (p->dim > (1 << 30)) return fail(CS2D_ERR_UNSUPPORTED, "more than 2^30 channels");
    if (p->offsets && p->batch != 1) return fail(CS2D_ERR_INVALID, "with offsets the batch is 1");
    if (p->offsets && p->n_seq < 0) return fail(CS2D_ERR_INVALID, "n_seq must not be negative");
    if (p->offsets && p->n_seq >= (1 << 30)) return fail(CS2D_ERR_UNSUPPORTED, "2^30 sequences or more");
    return CS2D_OK;
}
// Every row starts on a multiple of `bytes`, and so does what is behind its last channel.
static bool aligned(int bytes, int es, int dim, std::initializer_list<const void *> ptrs, std::initializer_list<int64_t> strides) {
    for (const void *p : ptrs)
        if (reinterpret_cast<uintptr_t>(p) % bytes) return false;
    for (int64_t s : strides)
        if (s * es % bytes) return false;
    return dim * (int64_t)es % bytes == 0;
}
static int how_moved(int es, int dim, std::initializer_list<const void *> ptrs, std::initializer_list<int64_t> strides) {
    return aligned(16, es, dim, ptrs, strides) ? GS_CHUNKS : aligned(4, es, dim, ptrs, strides) ? GS_WORDS : GS_ELEMENTS;
}
static size_t map_bytes(const cs2d_gscan *p) { return p->offsets ? ((size_t)p->length * 8 + 15) / 16 * 16 : 0; }
static int64_t checkpoints(const cs2d_gscan *p) { return (p->length - 1) / GS_CK; }
static int fill(GScan &d, const cs2d_gscan *p, void *saved) {
    d = GScan{};
    d.batch = p->batch; d.dim = p->dim; d.form = p->form; d.weighted = p->weighted != 0; d.length = p->length;
    d.nseq = p->offsets ? p->n_seq : 0; d.offsets = p->offsets; d.off64 = p->offsets64;
    if ((int64_t)p->batch * ((p->dim + 15) / 16) > INT32_MAX) return fail(CS2D_ERR_UNSUPPORTED, "batch times channels is too large");
    d.u = p->u; d.u_bs = p->u_bs; d.u_ls = p->u_ls;
    d.gate = p->gate; d.g_bs = p->gate_bs; d.g_ls = p->gate_ls;
    d.h0 = p->h0; d.h0_bs = p->h0_bs;
    d.nck = checkpoints(p);
    d.map = p->offsets ? (int2 *)saved : nullptr;
    d.ckpt = (float *)((char *)saved + map_bytes(p));
    d.status = status_ptr();
    if (!d.status) return fail(CS2D_ERR_CUDA, "the status word of the device is not available");
    return CS2D_OK;
}
static int launched(cudaError_t e, int n) {
    if (e != cudaSuccess) {
        cudaGetLastError();   // reported here: the next launch that asks for the last error finds none
        return fail(CS2D_ERR_CUDA, "launch failed: %s", cudaGetErrorString(e));
    }
    count_launches(n);
    return CS2D_OK;
}

static int validate(const cs2d_norm *p) {
    if (!p) return fail(CS2D_ERR_INVALID, "problem is NULL");
    if (p->dim <= 0 || p->outer <= 0 || p->inner <= 0) return fail(CS2D_ERR_INVALID, "all sizes must be positive");
    if (p->io_dtype < CS2D_F32 || p->io_dtype > CS2D_BF16) return fail(CS2D_ERR_INVALID, "input type must be float32, float16 or bfloat16");
    if (p->param_dtype != CS2D_F32 && p->param_dtype != p->io_dtype)
        return fail(CS2D_ERR_INVALID, "weight and bias must be float32 or of the input type");
    if (p->dim > (1 << 29)) return fail(CS2D_ERR_UNSUPPORTED, "more than 2^29 channels");   // 2 dim and what a warp's step leads to fit 32 bits
    if (!p->x) return fail(CS2D_ERR_INVALID, "x must be given");
    if (p->x_cs != 1 && p->x_is != 1) return fail(CS2D_ERR_INVALID, "x must have stride 1 along its channels or its rows");
    if (p->outer > ((int64_t)1 << 31) / p->inner) return fail(CS2D_ERR_UNSUPPORTED, "more than 2^31 rows");
    return CS2D_OK;
}
static Norm fill(const cs2d_norm *p) {
    Norm d{};
    d.dim = p->dim; d.wtype = p->param_dtype; d.rows = p->outer * p->inner; d.inner = p->inner; d.eps = p->eps;
    d.x = p->x; d.x_os = p->x_os; d.x_is = p->x_is; d.x_cs = p->x_cs;
    d.gate = p->gate; d.g_os = p->g_os; d.g_is = p->g_is;
    d.weight = p->weight; d.bias = p->bias;
    // One run of rows: the outer index goes on where the inner one ends, or is the only one (whose stride then is that of the rows).
    if (p->inner == 1 && (d.x_cs == 1 || d.x_os == 1)) {
        d.inner = d.rows;
        d.x_is = d.x_os;
        d.g_is = d.g_os;
    } else if (d.x_os == d.inner * d.x_is && (!d.gate || d.g_os == d.inner * d.g_is)) {
        d.inner = d.rows;
    }
    d.parts = norm_parts(d, p->io_dtype);
    return d;
}

}  // namespace cs2d

using namespace cs2d;

extern "C" {

size_t cs2d_gscan_saved_bytes(const cs2d_gscan *p, int keep) {
    if (validate(p, false)) return 0;
    const size_t n = map_bytes(p) + (keep ? (size_t)p->batch * checkpoints(p) * p->dim * 4 : 0);
    return n < 16 ? 16 : (n + 15) / 16 * 16;
}

int cs2d_gscan_fwd(const cs2d_gscan *p, void *y, int64_t y_bs, int64_t y_ls, float *h_last, void *saved, int keep, void *stream) {
    if (const int rc = validate(p, false)) return rc;
    if (!y || !saved || (!h_last && !(p->offsets && p->n_seq == 0))) return fail(CS2D_ERR_INVALID, "y, h_last and saved must be given");
    if (reinterpret_cast<uintptr_t>(saved) % 16) return fail(CS2D_ERR_INVALID, "saved must be 16-byte aligned");
    GScan d;
    if (const int rc = fill(d, p, saved)) return rc;
    const int es = p->io_dtype == CS2D_F32 ? 4 : 2;
    d.io = how_moved(es, p->dim, {p->u, p->gate}, {p->u_bs, p->u_ls, p->gate_bs, p->gate_ls});
    d.io_out = how_moved(es, p->dim, {y}, {y_bs, y_ls});
    d.y = y; d.y_bs = y_bs; d.y_ls = y_ls; d.last = h_last;
    if (!keep) d.ckpt = nullptr;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (d.map)
        if (const int rc = launched(launch_gscan_map(d, st), 1)) return rc;
    return launched(launch_gscan_fwd(d, p->io_dtype, st), 1);
}

int cs2d_gscan_bwd(const cs2d_gscan *p, const void *dy, int64_t dy_bs, int64_t dy_ls, const float *dh_last, int64_t dh_last_bs,
                   const void *saved, void *du, void *dgate, float *dh0, void *stream) {
    if (const int rc = validate(p, false)) return rc;
    if (!dy || !saved || !du || !dgate) return fail(CS2D_ERR_INVALID, "dy, saved, du and dgate must be given");
    if (reinterpret_cast<uintptr_t>(saved) % 16) return fail(CS2D_ERR_INVALID, "saved must be 16-byte aligned");
    GScan d;
    if (const int rc = fill(d, p, const_cast<void *>(saved))) return rc;
    const int es = p->io_dtype == CS2D_F32 ? 4 : 2;
    d.io = how_moved(es, p->dim, {p->u, p->gate, dy}, {p->u_bs, p->u_ls, p->gate_bs, p->gate_ls, dy_bs, dy_ls});
    d.io_out = how_moved(es, p->dim, {du, dgate}, {p->length * p->dim, p->dim});
    d.dy = dy; d.dy_bs = dy_bs; d.dy_ls = dy_ls; d.dlast = dh_last; d.dlast_bs = dh_last_bs;
    d.du = du; d.dgate = dgate; d.y_bs = p->length * p->dim; d.y_ls = p->dim; d.dh0 = dh0;
    return launched(launch_gscan_bwd(d, p->io_dtype, static_cast<cudaStream_t>(stream)), 1);
}

int cs2d_gscan_step(const cs2d_gscan *p, void *y, int64_t y_bs, float *h, int64_t h_bs, void *stream) {
    if (const int rc = validate(p, true)) return rc;
    if (!y || !h) return fail(CS2D_ERR_INVALID, "y and h must be given");
    if ((int64_t)p->batch * p->dim > ((int64_t)1 << 38)) return fail(CS2D_ERR_UNSUPPORTED, "batch times channels is too large");
    GScan d{};
    d.batch = p->batch; d.dim = p->dim; d.form = p->form; d.weighted = p->weighted != 0;
    d.u = p->u; d.u_bs = p->u_bs; d.gate = p->gate; d.g_bs = p->gate_bs; d.y = y; d.y_bs = y_bs; d.h = h; d.h_bs = h_bs;
    return launched(launch_gscan_step(d, p->io_dtype, static_cast<cudaStream_t>(stream)), 1);
}

int cs2d_norm_fwd(const cs2d_norm *p, void *y, float *stats, void *stream) {
    if (const int rc = validate(p)) return rc;
    if (!y) return fail(CS2D_ERR_INVALID, "y must be given");
    if (reinterpret_cast<uintptr_t>(stats) % 8) return fail(CS2D_ERR_INVALID, "stats must be 8-byte aligned");
    Norm d = fill(p);
    d.y = y; d.stats = stats;
    return launched(launch_norm_fwd(d, p->io_dtype, static_cast<cudaStream_t>(stream)), 1);
}

size_t cs2d_norm_bwd_scratch_bytes(const cs2d_norm *p) {
    if (validate(p)) return 0;
    return ((size_t)fill(p).parts * 2 * p->dim * 4 + 15) / 16 * 16;
}

int cs2d_norm_bwd(const cs2d_norm *p, const void *dy, int64_t dy_os, int64_t dy_is, const float *stats, void *scratch, void *dx,
                  int64_t dx_os, int64_t dx_is, int64_t dx_cs, void *dgate, void *dweight, void *dbias, void *stream) {
    if (const int rc = validate(p)) return rc;
    if (!dy || !stats || !dx || !scratch || (p->gate && !dgate)) return fail(CS2D_ERR_INVALID, "dy, stats, scratch, dx and the gate's gradient must be given");
    if (reinterpret_cast<uintptr_t>(stats) % 8 || reinterpret_cast<uintptr_t>(scratch) % 16) return fail(CS2D_ERR_INVALID, "stats must be 8-byte, scratch 16-byte aligned");
    if (dx_cs != 1 && dx_is != 1) return fail(CS2D_ERR_INVALID, "dx must have stride 1 along its channels or its rows");
    Norm d = fill(p);
    d.dy = dy; d.dy_os = dy_os; d.dy_is = dy_is; d.stats = const_cast<float *>(stats); d.part = (float *)scratch;
    d.dx = dx; d.dx_os = dx_os; d.dx_is = dx_is; d.dx_cs = dx_cs;
    if (p->inner == 1 && d.inner != 1 && (dx_cs == 1 || dx_os == 1)) {
        d.dy_is = dy_os;
        d.dx_is = dx_os;
    } else if (d.inner != p->inner && (dy_os != p->inner * dy_is || dx_os != p->inner * dx_is)) {
        d.inner = p->inner;
    }
    d.dgate = dgate; d.dweight = dweight; d.dbias = dbias;
    int n = 0;
    const cudaError_t e = launch_norm_bwd(d, p->io_dtype, static_cast<cudaStream_t>(stream), &n);
    return launched(e, n);
}

}  // extern "C"
