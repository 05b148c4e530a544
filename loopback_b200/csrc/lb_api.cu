// C-ABI layer: argument checks, tile-shape selection, TMA descriptors, launches. See include/loopback_b200.h.
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <mutex>
#include <string>

#include <cudaTypedefs.h>

#include "../../include/loopback_b200.h"
#include "lb_common.cuh"
#include "lb_kernels.h"

// one error word per device: the first bounded wait of any kernel that runs out records its code here
__device__ int g_lb_device_error = 0;

namespace {

constexpr int kMaxGrid = 304;                 // rows of the query-gradient scratch (>= 2 CTAs per SM on 148 SMs)
constexpr size_t kMaxSmem = 227 * 1024;

thread_local std::string t_err;

int fail(int code, const char *fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    t_err = buf;
    return code;
}

int cuda_fail(cudaError_t e, const char *what) {
    return fail(LB_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

struct Options {
    int fwd_stages = 0, bwd_stages = 0, fwd_fr = 0, grid_cap = 0, fwd_warps = 0, bwd_warps = 0, bwd_wpt = 0,
        tma_per_chunk = 0, write_tt = 0, write_mt = 0, fwd_sps = 0, write_tile = 0, write_stages = 0, wait_cycles = 0, test_skip_item = 0,
        ffn_tile = 0, ffn_splits = 0, block_frags = 0, ffn_small = 0;
} g_opt;

struct DeviceInfo {
    int sms = 0;
    int cc_major = 0;
    int *err_word = nullptr;
    bool ok = false;
};

int device_info(DeviceInfo *out) {
    static std::mutex mu;
    static DeviceInfo cache[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
    if (dev < 0 || dev >= 64) return fail(LB_ERR_CUDA, "device ordinal %d out of range", dev);
    // tensor maps are encoded through the driver, which wants a context bound to the calling thread; a thread that has made
    // no runtime call yet (autograd's, at its first backward) has none
    static thread_local int bound = -1;
    if (bound != dev) {
        if ((e = cudaSetDevice(dev)) != cudaSuccess) return cuda_fail(e, "cudaSetDevice");
        bound = dev;
    }
    std::lock_guard<std::mutex> lk(mu);
    if (!cache[dev].ok) {
        DeviceInfo di;
        if ((e = cudaDeviceGetAttribute(&di.sms, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess)
            return cuda_fail(e, "cudaDeviceGetAttribute(sm count)");
        if ((e = cudaDeviceGetAttribute(&di.cc_major, cudaDevAttrComputeCapabilityMajor, dev)) != cudaSuccess)
            return cuda_fail(e, "cudaDeviceGetAttribute(cc major)");
        if (di.cc_major != 10)
            return fail(LB_ERR_CUDA, "device %d has compute capability %d.x; this library is built for sm_100a only",
                        dev, di.cc_major);
        if ((e = cudaGetSymbolAddress(reinterpret_cast<void **>(&di.err_word), g_lb_device_error)) != cudaSuccess)
            return cuda_fail(e, "cudaGetSymbolAddress(device error word)");
        di.ok = true;
        cache[dev] = di;
    }
    *out = cache[dev];
    return LB_OK;
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    });
    return fn;
}

// A tiled descriptor over [outer][n_tok][d] (outer == 0: no outer dimension).
//   box_chunks == 0: dimensions (d, n_tok[, outer]), box = 512 bytes x box_tok tokens: one chunk of every token;
//   box_chunks  > 0: the row is split into whole 512-byte chunks, dimensions (chunk width, chunks, n_tok[, outer]),
//                    box = 512 bytes x box_chunks chunks x box_tok tokens: a whole tile in one copy, token-major.
//                    Needs d to be a multiple of the chunk width.
int make_map(CUtensorMap *m, const void *base, int dtype, long long n_tok, int d, int outer, int box_tok,
             int box_chunks, int box_outer = 1) {
    auto fn = encode_fn();
    if (!fn) return fail(LB_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
    const int elem = dtype == LB_DTYPE_BF16 ? 2 : 4;
    const cuuint64_t bw = lb::kChunkBytes / elem;
    cuuint64_t dims[4];
    cuuint64_t strides[3];
    cuuint32_t box[4];
    cuuint32_t estr[4] = {1, 1, 1, 1};
    cuuint32_t rank = 0;
    if (box_chunks > 0) {
        dims[0] = bw; dims[1] = (cuuint64_t)d / bw; dims[2] = (cuuint64_t)n_tok;
        strides[0] = lb::kChunkBytes; strides[1] = (cuuint64_t)d * elem;
        box[0] = (cuuint32_t)bw; box[1] = (cuuint32_t)box_chunks; box[2] = (cuuint32_t)box_tok;
        rank = 3;
    } else {
        dims[0] = (cuuint64_t)d; dims[1] = (cuuint64_t)n_tok;
        strides[0] = (cuuint64_t)d * elem;
        box[0] = (cuuint32_t)bw; box[1] = (cuuint32_t)box_tok;
        rank = 2;
    }
    if (outer > 0) {
        dims[rank] = (cuuint64_t)outer;
        strides[rank - 1] = (cuuint64_t)d * elem * (cuuint64_t)n_tok;
        box[rank] = (cuuint32_t)box_outer;
        ++rank;
    }
    CUresult r = fn(m, dtype == LB_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32,
                    rank, const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(LB_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
    return LB_OK;
}

// h / x of the tensor-core write: 2-D, boxes of box_tok rows x 64 bf16 columns, 128-byte swizzle
int make_map_sw128(CUtensorMap *m, const void *base, long long n_tok, int d, int box_tok) {
    auto fn = encode_fn();
    if (!fn) return fail(LB_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
    cuuint64_t dims[2] = {(cuuint64_t)d, (cuuint64_t)n_tok};
    cuuint64_t strides[1] = {(cuuint64_t)d * 2};
    cuuint32_t box[2] = {64, (cuuint32_t)box_tok};
    cuuint32_t estr[2] = {1, 1};
    CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void *>(base), dims, strides, box, estr,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(LB_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
    return LB_OK;
}

long long wait_limit() { return g_opt.wait_cycles > 0 ? (long long)g_opt.wait_cycles : lb::kWaitCycles; }

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int check_common(long long n_tok, int d, int dtype) {
    if (dtype != LB_DTYPE_BF16 && dtype != LB_DTYPE_F32) return fail(LB_ERR_ARG, "dtype %d is neither LB_DTYPE_F32 nor LB_DTYPE_BF16", dtype);
    if (n_tok < 0 || d <= 0) return fail(LB_ERR_ARG, "n_tok=%lld, d=%d: sizes must be positive", n_tok, d);
    if (n_tok >= (1LL << 31)) return fail(LB_ERR_UNSUPPORTED, "n_tok=%lld does not fit the 32-bit TMA coordinates", n_tok);
    const long long row = (long long)d * (dtype == LB_DTYPE_BF16 ? 2 : 4);
    if (row % 16 != 0) return fail(LB_ERR_ALIGN, "row size %lld bytes (d=%d) is not a multiple of 16", row, d);
    if (row > 32 * lb::kChunkBytes) return fail(LB_ERR_UNSUPPORTED, "row size %lld bytes exceeds the supported 16384", row);
    return LB_OK;
}

int chunks_of(int d, int dtype) {
    const int row = d * (dtype == LB_DTYPE_BF16 ? 2 : 4);
    return (row + lb::kChunkBytes - 1) / lb::kChunkBytes;
}

}  // namespace

// sets the calling thread's error message from another translation unit of this library (not exported)
extern "C" int lb_fail_message(int code, const char *msg) { return fail(code, "%s", msg); }

#pragma GCC visibility push(default)
extern "C" {

int lb_version(void) { return LB_VERSION; }

const char *lb_last_error_string(void) { return t_err.c_str(); }

int lb_device_error(int clear) {
    int v = 0;
    cudaError_t e = cudaDeviceSynchronize();
    if (e != cudaSuccess) return cuda_fail(e, "cudaDeviceSynchronize");
    e = cudaMemcpyFromSymbol(&v, g_lb_device_error, sizeof(int));
    if (e != cudaSuccess) return cuda_fail(e, "cudaMemcpyFromSymbol(device error word)");
    if (clear && v != 0) {
        int z = 0;
        e = cudaMemcpyToSymbol(g_lb_device_error, &z, sizeof(int));
        if (e != cudaSuccess) return cuda_fail(e, "cudaMemcpyToSymbol(device error word)");
    }
    if (v != 0) fail(LB_ERR_DEVICE, "a kernel gave up a bounded wait (code %d)", v);
    return v;
}

int lb_set_option(const char *name, int value) {
    if (!name) return fail(LB_ERR_ARG, "option name is NULL");
    if (!strcmp(name, "reset_all")) g_opt = Options();
    else if (!strcmp(name, "fwd_stages")) g_opt.fwd_stages = value;
    else if (!strcmp(name, "bwd_stages")) g_opt.bwd_stages = value;
    else if (!strcmp(name, "fwd_fr")) g_opt.fwd_fr = value;
    else if (!strcmp(name, "grid_cap")) g_opt.grid_cap = value;
    else if (!strcmp(name, "fwd_warps")) g_opt.fwd_warps = value;
    else if (!strcmp(name, "bwd_warps")) g_opt.bwd_warps = value;
    else if (!strcmp(name, "bwd_wpt")) g_opt.bwd_wpt = value;
    else if (!strcmp(name, "tma_per_chunk")) g_opt.tma_per_chunk = value;
    else if (!strcmp(name, "write_tt")) g_opt.write_tt = value;
    else if (!strcmp(name, "write_mt")) g_opt.write_mt = value;
    else if (!strcmp(name, "fwd_sps")) g_opt.fwd_sps = value;
    else if (!strcmp(name, "write_tile")) g_opt.write_tile = value;
    else if (!strcmp(name, "write_stages")) g_opt.write_stages = value;
    else if (!strcmp(name, "wait_cycles")) g_opt.wait_cycles = value;
    else if (!strcmp(name, "ffn_tile")) g_opt.ffn_tile = value;
    else if (!strcmp(name, "ffn_splits")) g_opt.ffn_splits = value;
    else if (!strcmp(name, "ffn_small")) g_opt.ffn_small = value;
    else if (!strcmp(name, "block_frags")) g_opt.block_frags = value;
    else if (!strcmp(name, "test_skip_item")) g_opt.test_skip_item = value;
    else return fail(LB_ERR_ARG, "unknown option '%s'", name);
    return LB_OK;
}

int lb_write(const void *h, const void *x, void *V, float *R, const float *Q, float *DOTS, int64_t n_tok, int d, int N,
             int NQ, int s, float eps, int dtype, void *stream) {
    int rc = check_common(n_tok, d, dtype);
    if (rc) return rc;
    if (!h || !x || !V) return fail(LB_ERR_ARG, "lb_write: h, x and V must be non-NULL");
    if (N <= 0 || s < 0 || s >= N) return fail(LB_ERR_ARG, "lb_write: step %d outside [0, %d)", s, N);
    if (!R) Q = nullptr;                       // without R only V[s] is written: Q is ignored
    if (Q && (!DOTS || NQ < 0 || NQ > N)) return fail(LB_ERR_ARG, "lb_write: scores need DOTS and 0 <= NQ <= N");
    if (!aligned16(h) || !aligned16(x) || !aligned16(V) || (Q && !aligned16(Q)))
        return fail(LB_ERR_ALIGN, "lb_write: h, x, V and Q must be 16-byte aligned");
    DeviceInfo di;
    if ((rc = device_info(&di))) return rc;
    const long long elem = dtype == LB_DTYPE_BF16 ? 2 : 4;
    lb::WriteParams p;
    p.h = h; p.x = x;
    p.v = static_cast<char *>(V) + (long long)s * n_tok * d * elem;
    p.r = R ? R + (long long)s * n_tok : nullptr;
    p.Q = (Q && R) ? Q : nullptr;
    p.j0 = s > 0 ? s - 1 : 0;
    p.nq = p.Q ? NQ - p.j0 : 0;
    if (p.nq <= 0) { p.nq = 0; p.Q = nullptr; }
    p.dots_s = DOTS ? DOTS + (long long)s * n_tok : nullptr;
    p.dots_qstride = (long long)N * n_tok;
    p.n_tok = n_tok; p.d = d; p.eps = eps; p.write_tt = g_opt.write_tt == 1 || g_opt.write_tt == 2 ? g_opt.write_tt : 0;
    // bf16 rows in training-sized batches (every SM gets at least 32 tokens): the persistent tensor-core kernel
    const int nt = lb::write_mma_ntiles(p.nq);
    if (dtype == LB_DTYPE_BF16 && d >= 64 && nt >= 0 && n_tok > 0 &&
        (g_opt.write_tt == 3 || (g_opt.write_tt == 0 && n_tok >= 32LL * di.sms))) {
        const long long blocks32 = (n_tok + 31) / 32;
        const long long rounds = (blocks32 + 8LL * di.sms - 1) / (8LL * di.sms);
        const long long per = (blocks32 + di.sms * rounds - 1) / (di.sms * rounds);        // 1..8
        lb::WriteMmaParams mp;
        static_cast<lb::WriteParams &>(mp) = p;
        mp.tile_tok = (int)per * 32;
        if (g_opt.write_tile >= 32 && g_opt.write_tile <= 256 && g_opt.write_tile % 32 == 0) mp.tile_tok = g_opt.write_tile;
        mp.chunks = (d + 63) / 64;
        mp.n_tiles = (n_tok + mp.tile_tok - 1) / mp.tile_tok;
        mp.err_word = di.err_word;
        mp.wait_cycles = wait_limit();
        mp.stages = g_opt.write_stages >= 2 && g_opt.write_stages <= 8 ? g_opt.write_stages : 4;
        while (mp.stages > 2 && lb::write_mma_smem_bytes(nt, mp.tile_tok, mp.stages) > 227 * 1024) --mp.stages;
        CUtensorMap tmH, tmX;
        if ((rc = make_map_sw128(&tmH, h, n_tok, d, mp.tile_tok))) return rc;
        if ((rc = make_map_sw128(&tmX, x, n_tok, d, mp.tile_tok))) return rc;
        const int grid = (int)(mp.n_tiles < di.sms ? mp.n_tiles : di.sms);
        cudaError_t e = lb::launch_write_mma(tmH, tmX, mp, nt, g_opt.write_mt == 1 ? 1 : 2, grid, static_cast<cudaStream_t>(stream));
        return e == cudaSuccess ? LB_OK : cuda_fail(e, "lb_write launch");
    }
    cudaError_t e = lb::launch_write(dtype, p, di.sms, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? LB_OK : cuda_fail(e, "lb_write launch");
}

int lb_write_bwd_dx(const void *g, void *dx, int64_t n_elem, int dtype, void *stream) {
    if (dtype != LB_DTYPE_BF16 && dtype != LB_DTYPE_F32) return fail(LB_ERR_ARG, "bad dtype %d", dtype);
    if (!g || !dx || n_elem < 0) return fail(LB_ERR_ARG, "lb_write_bwd_dx: NULL pointer or negative size");
    if (!aligned16(g) || !aligned16(dx) || (n_elem * (dtype == LB_DTYPE_BF16 ? 2 : 4)) % 16)
        return fail(LB_ERR_ALIGN, "lb_write_bwd_dx: pointers and byte size must be multiples of 16");
    DeviceInfo di;
    int rc = device_info(&di);
    if (rc) return rc;
    cudaError_t e = lb::launch_neg(dtype, g, dx, n_elem, di.sms, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? LB_OK : cuda_fail(e, "lb_write_bwd_dx launch");
}

int lb_rstd_fwd(const void *x, float *r, int64_t n_tok, int d, float eps, int dtype, void *stream) {
    int rc = check_common(n_tok, d, dtype);
    if (rc) return rc;
    if (!x || !r) return fail(LB_ERR_ARG, "lb_rstd_fwd: NULL pointer");
    if (!aligned16(x)) return fail(LB_ERR_ALIGN, "lb_rstd_fwd: x must be 16-byte aligned");
    DeviceInfo di;
    if ((rc = device_info(&di))) return rc;
    cudaError_t e = lb::launch_rstd_fwd(dtype, x, r, n_tok, d, eps, di.sms, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? LB_OK : cuda_fail(e, "lb_rstd_fwd launch");
}

static int rstd_bwd_common(const void *x, const float *r, const float *gr, void *gx, int64_t n_tok, int d, int dtype,
                           int mode, void *stream) {
    int rc = check_common(n_tok, d, dtype);
    if (rc) return rc;
    if (!x || !r || !gr || !gx) return fail(LB_ERR_ARG, "lb_rstd_bwd: NULL pointer");
    if (!aligned16(x) || !aligned16(gx)) return fail(LB_ERR_ALIGN, "lb_rstd_bwd: x and gx must be 16-byte aligned");
    DeviceInfo di;
    if ((rc = device_info(&di))) return rc;
    cudaError_t e = lb::launch_rstd_bwd(dtype, x, r, gr, gx, n_tok, d, mode, di.sms, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? LB_OK : cuda_fail(e, "lb_rstd_bwd launch");
}

int lb_rstd_bwd(const void *x, const float *r, const float *gr, void *gx, int64_t n_tok, int d, int dtype, void *stream) {
    return rstd_bwd_common(x, r, gr, gx, n_tok, d, dtype, 0, stream);
}

int lb_rstd_bwd_acc(const void *x, const float *r, const float *gr, void *dv, int64_t n_tok, int d, int dtype,
                    void *stream) {
    return rstd_bwd_common(x, r, gr, dv, n_tok, d, dtype, 1, stream);
}

int lb_scores(const void *V, const float *q, float *dots, int64_t n_tok, int d, int N, int n, int dtype, void *stream) {
    int rc = check_common(n_tok, d, dtype);
    if (rc) return rc;
    if (!V || !q || !dots) return fail(LB_ERR_ARG, "lb_scores: NULL pointer");
    if (n < 1 || n > N) return fail(LB_ERR_ARG, "lb_scores: n=%d outside [1, N=%d]", n, N);
    if (!aligned16(V) || !aligned16(q)) return fail(LB_ERR_ALIGN, "lb_scores: V and q must be 16-byte aligned");
    DeviceInfo di;
    if ((rc = device_info(&di))) return rc;
    cudaError_t e = lb::launch_scores(dtype, V, q, dots, n_tok, d, n, di.sms, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? LB_OK : cuda_fail(e, "lb_scores launch");
}

static int read_fwd_impl(const void *V, const float *R, const float *DOTS, int qi, const void *base, const void *h0,
                         float beta, const float *cbar, const float *tc_prev, float lam, const float *c0, void *out,
                         float *TC, float *LG, float *LSE, float *LSE0, int64_t n_tok, int d, int N, int n, int dtype,
                         void *stream);

int lb_read_fwd(const void *V, const float *R, const float *DOTS, int qi, const void *base, const float *cbar,
                const float *c0, void *out, float *TC, float *LG, float *LSE, float *LSE0, int64_t n_tok, int d, int N,
                int n, int dtype, void *stream) {
    if (!cbar) return fail(LB_ERR_ARG, "lb_read_fwd: NULL pointer");
    return read_fwd_impl(V, R, DOTS, qi, base, nullptr, 0.f, cbar, nullptr, 1.f, c0, out, TC, LG, LSE, LSE0, n_tok, d, N, n,
                         dtype, stream);
}

int lb_combine_fwd(const void *V, const float *R, const float *DOTS, int qi, const void *proposal, const void *h0,
                   float beta, const float *tc_prev, float lam, const float *c0, void *out, float *TC, float *LG,
                   float *LSE, float *LSE0, int64_t n_tok, int d, int N, int n, int dtype, void *stream) {
    if (n < 2 || !tc_prev) return fail(LB_ERR_ARG, "lb_combine_fwd: needs n >= 2 and the previous read's coefficients");
    if (h0 && !aligned16(h0)) return fail(LB_ERR_ALIGN, "lb_combine_fwd: h0 must be 16-byte aligned");
    return read_fwd_impl(V, R, DOTS, qi, proposal, h0, beta, nullptr, tc_prev, lam, c0, out, TC, LG, LSE, LSE0, n_tok, d,
                         N, n, dtype, stream);
}

static int read_fwd_impl(const void *V, const float *R, const float *DOTS, int qi, const void *base, const void *h0,
                         float beta, const float *cbar, const float *tc_prev, float lam, const float *c0, void *out,
                         float *TC, float *LG, float *LSE, float *LSE0, int64_t n_tok, int d, int N, int n, int dtype,
                         void *stream) {
    int rc = check_common(n_tok, d, dtype);
    if (rc) return rc;
    if (!V || !R || !DOTS || !base || (!cbar && !tc_prev) || !c0 || !out || !TC) return fail(LB_ERR_ARG, "lb_read_fwd: NULL pointer");
    if ((LG != nullptr) != (LSE != nullptr) || (LG != nullptr) != (LSE0 != nullptr))
        return fail(LB_ERR_ARG, "lb_read_fwd: LG, LSE and LSE0 must be given together");
    if (n < 1 || n > N) return fail(LB_ERR_ARG, "lb_read_fwd: n=%d outside [1, N=%d]", n, N);
    if (n > LB_MAX_SOURCES) return fail(LB_ERR_UNSUPPORTED, "lb_read_fwd: n=%d exceeds LB_MAX_SOURCES=%d", n, LB_MAX_SOURCES);
    if (qi < 0) return fail(LB_ERR_ARG, "lb_read_fwd: query row %d is negative", qi);
    if (!aligned16(V) || !aligned16(base) || !aligned16(out))
        return fail(LB_ERR_ALIGN, "lb_read_fwd: V, base and out must be 16-byte aligned");
    if (n_tok == 0) return LB_OK;
    DeviceInfo di;
    if ((rc = device_info(&di))) return rc;

    const int nch = chunks_of(d, dtype);
    const int elem = dtype == LB_DTYPE_BF16 ? 2 : 4;
    const bool rank4 = !g_opt.tma_per_chunk && (d * elem) % lb::kChunkBytes == 0;
    // Tile shape: consumer warps (16, 12 or 8), warps per token and fragments per warp. A tile normally spans the
    // whole row (one column group); the choice avoids idle fragments first, then prefers stages near 16 KiB.
    // With too few tokens to give every SM a tile, the row is cut into column groups instead (8-token tiles).
    int ncw = 0, wpt = 0, fr = 0, best_cost = 1 << 30;
    static const int kNcw[3] = {8, 12, 16};
    for (int a = 0; a < 3; ++a) {
        if (g_opt.fwd_warps && g_opt.fwd_warps != kNcw[a]) continue;
        for (int w = 1; w <= kNcw[a]; ++w) {
            if (kNcw[a] % w) continue;
            const int f = (nch + w - 1) / w;
            if (f > 4 || (g_opt.fwd_fr && g_opt.fwd_fr != f)) continue;
            const int stage_kb = nch * (kNcw[a] / w) / 2;
            const int off = stage_kb > 16 ? stage_kb - 16 : 16 - stage_kb;
            const int cost = (f * w - nch) * 64 + off * 2 + a;
            if (cost < best_cost) { best_cost = cost; ncw = kNcw[a]; wpt = w; fr = f; }
        }
    }
    if (ncw == 0) return fail(LB_ERR_UNSUPPORTED, "lb_read_fwd: no tile shape covers d=%d (row of %d chunks)", d, nch);
    int bt = ncw / wpt;
    long long tok_tiles = (n_tok + bt - 1) / bt;
    int cg = 1;
    if (tok_tiles < di.sms) {            // few tokens: 8 tokens x (fr chunks) tiles, as many column groups as it takes
        ncw = 8; wpt = 1; bt = 8;
        tok_tiles = (n_tok + 7) / 8;
        fr = nch < 4 ? nch : 4;
        while (fr > 1 && tok_tiles * ((nch + fr - 1) / fr) < di.sms) --fr;
        cg = (nch + fr - 1) / fr;
    }
    // ring depth: 6 stages of a full-size (12-16 KiB) tile measured best (8 and more cost 2-4 %: more requests in
    // flight than the memory system orders well); small tiles (decode-sized batches) get a deeper ring so that a CTA
    // still keeps ~128 KiB in flight
    // Small tiles also take several sources per stage (one TMA box over the source axis): the hand-shake of a stage
    // costs about as much for 4 KiB as for 16 KiB, and a decode-sized read is made of nothing else.
    const int tile_bytes = fr * ncw * lb::kChunkBytes;
    int sps = 1;
    if (rank4 && n >= 4) sps = tile_bytes <= 4 * 1024 ? 4 : (tile_bytes <= 8 * 1024 ? 2 : 1);
    if (rank4 && g_opt.fwd_sps >= 1 && g_opt.fwd_sps <= 4) sps = g_opt.fwd_sps;
    const int stage_bytes = sps * tile_bytes;
    int stages = g_opt.fwd_stages > 0 ? g_opt.fwd_stages : 6;
    if (g_opt.fwd_stages <= 0 && stage_bytes < 12 * 1024) stages = 128 * 1024 / stage_bytes;
    if (stages > 32) stages = 32;
    while (stages > 2 && lb::read_fwd_smem_bytes(fr, ncw, stages, sps) > kMaxSmem) --stages;

    CUtensorMap tmV, tmB, tmH;
    if ((rc = make_map(&tmV, V, dtype, n_tok, d, N, bt, rank4 ? fr * wpt : 0, sps))) return rc;
    if ((rc = make_map(&tmB, base, dtype, n_tok, d, 0, bt, rank4 ? fr * wpt : 0))) return rc;
    if ((rc = make_map(&tmH, h0 ? h0 : base, dtype, n_tok, d, 0, bt, rank4 ? fr * wpt : 0))) return rc;

    lb::ReadFwdParams p;
    p.R = R;
    p.dots = DOTS + (long long)qi * N * n_tok;
    p.cbar = cbar; p.tc_prev = tc_prev; p.lam = lam; p.blend = h0 ? 1 : 0; p.beta = beta;
    p.c0 = c0; p.out = out; p.TC = TC; p.LG = LG; p.LSE = LSE; p.LSE0 = LSE0;
    p.n_tok = n_tok; p.d = d; p.n = n; p.chunks = nch; p.wpt = wpt; p.col_groups = cg; p.tok_tiles = tok_tiles;
    p.stages = stages; p.sps = sps;
    p.rank4 = rank4 ? 1 : 0;
    p.inv_sqrt_d = 1.0f / sqrtf((float)d);
    p.err_word = di.err_word;
    p.wait_cycles = wait_limit(); p.test_skip_item = g_opt.test_skip_item;
    const long long tiles = tok_tiles * cg;
    int cap = g_opt.grid_cap > 0 ? g_opt.grid_cap : di.sms;
    if (cap > kMaxGrid) cap = kMaxGrid;
    const int grid = (int)(tiles < cap ? tiles : cap);
    cudaError_t e = lb::launch_read_fwd(dtype, fr, ncw, tmV, tmB, tmH, p, grid, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? LB_OK : cuda_fail(e, "lb_read_fwd launch");
}

int lb_step_fwd(const void *h, const void *x, const void *h0, float beta, void *V, float *R, const float *Q,
                const float *tc_prev, float lam, const float *c0, void *out, float *TC, float *LG, float *LSE, float *LSE0,
                int64_t n_tok, int d, int N, int s, float eps, int dtype, void *stream) {
    int rc = check_common(n_tok, d, dtype);
    if (rc) return rc;
    if (!h || !x || !V || !R || !Q || !tc_prev || !c0 || !out || !TC) return fail(LB_ERR_ARG, "lb_step_fwd: NULL pointer");
    if ((LG != nullptr) != (LSE != nullptr) || (LG != nullptr) != (LSE0 != nullptr))
        return fail(LB_ERR_ARG, "lb_step_fwd: LG, LSE and LSE0 must be given together");
    if (s < 1 || s >= N) return fail(LB_ERR_ARG, "lb_step_fwd: step %d outside [1, N=%d)", s, N);
    if (s + 1 > LB_MAX_SOURCES) return fail(LB_ERR_UNSUPPORTED, "lb_step_fwd: %d sources exceed LB_MAX_SOURCES=%d", s + 1, LB_MAX_SOURCES);
    if (!aligned16(h) || !aligned16(x) || !aligned16(V) || !aligned16(out) || !aligned16(Q) || (h0 && !aligned16(h0)))
        return fail(LB_ERR_ALIGN, "lb_step_fwd: h, x, h0, V, out and Q must be 16-byte aligned");
    if (((long long)d * 4) % 16) return fail(LB_ERR_ALIGN, "lb_step_fwd: the query rows must be multiples of 16 bytes");
    if (n_tok > 65535LL * 16) return fail(LB_ERR_UNSUPPORTED, "lb_step_fwd: meant for decode-sized batches; %lld tokens is not one", (long long)n_tok);
    if (n_tok == 0) return LB_OK;
    DeviceInfo di;
    if ((rc = device_info(&di))) return rc;
    const int elem = dtype == LB_DTYPE_BF16 ? 2 : 4;
    lb::StepSmallParams p;
    p.h = h; p.x = x; p.h0 = h0; p.V = V; p.R = R; p.q = Q + (long long)(s - 1) * d; p.tc_prev = tc_prev; p.c0 = c0;
    p.out = out; p.TC = TC; p.LG = LG; p.LSE = LSE; p.LSE0 = LSE0;
    p.n_tok = n_tok; p.d = d; p.n = s + 1; p.lam = lam; p.beta = beta; p.eps = eps; p.inv_sqrt_d = 1.0f / sqrtf((float)d);
    p.blend = h0 ? 1 : 0;
    const int frags = (d * elem + 15) / 16;
    p.ct = (frags + 31) / 32 * 32;
    p.sg = p.ct >= 1024 ? 1 : (1024 / p.ct > 4 ? 4 : 1024 / p.ct);
    if (lb::step_small_smem_bytes(p.ct, p.sg, 16 / elem) > kMaxSmem) return fail(LB_ERR_UNSUPPORTED, "lb_step_fwd: row too wide");
    cudaError_t e = lb::launch_step_small(dtype, p, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? LB_OK : cuda_fail(e, "lb_step_fwd launch");
}

size_t lb_read_bwd_scratch_bytes(int d) { return d > 0 ? (size_t)kMaxGrid * (size_t)d * sizeof(float) : 0; }

// what a finalising backward hands out beyond dV / dR when the write and the read of update n-1 are one autograd node
struct StepGrads {
    void *dh = nullptr;        // gradient of the block output
    void *dh0 = nullptr;       // gradient of the loop input (an iteration's last read only)
    int dh0_accum = 0;
    int blend = 0;
    float beta = 0.f;
    int skip_final_store = 0;
    // the deferred form (G != null): no gradient stack; `dV` of read_bwd_impl is then the g stack
    float *Wt = nullptr, *KQt = nullptr;
    const float *Qall = nullptr;
    int deferred = 0;
    void *dv0 = nullptr, *dx0 = nullptr;
};

static int read_bwd_impl(const void *V, const float *R, void *dV, float *dR, const float *q, const void *g,
                         const float *gt, const float *cbar, const float *tc_prev, float lam, const float *c0,
                         const float *LG, const float *LSE, const float *LSE0, float *dcbar, float *dq, void *scratch,
                         int64_t n_tok, int d, int N, int n, int accum, int finalize, void *neg_out, int dtype,
                         void *stream, const StepGrads &sg = StepGrads());

int lb_read_bwd(const void *V, const float *R, void *dV, float *dR, const float *q, const void *g, const float *gt,
                const float *cbar, const float *c0, const float *LG, const float *LSE, const float *LSE0, float *dcbar,
                float *dq, void *scratch, int64_t n_tok, int d, int N, int n, int accum, int dtype, void *stream) {
    if (!cbar) return fail(LB_ERR_ARG, "lb_read_bwd: NULL pointer");
    return read_bwd_impl(V, R, dV, dR, q, g, gt, cbar, nullptr, 1.f, c0, LG, LSE, LSE0, dcbar, dq, scratch, n_tok, d, N, n,
                         accum, 0, nullptr, dtype, stream);
}

int lb_combine_bwd(const void *V, const float *R, void *dV, float *dR, const float *q, const void *g, const float *gt,
                   const float *tc_prev, float lam, const float *c0, const float *LG, const float *LSE,
                   const float *LSE0, float *dtc_prev, float *dq, void *scratch, void *neg_out, int finalize,
                   int64_t n_tok, int d, int N, int n, int accum, int dtype, void *stream) {
    if (n < 2 || !tc_prev) return fail(LB_ERR_ARG, "lb_combine_bwd: needs n >= 2 and the previous read's coefficients");
    if (neg_out && !aligned16(neg_out)) return fail(LB_ERR_ALIGN, "lb_combine_bwd: neg_out must be 16-byte aligned");
    return read_bwd_impl(V, R, dV, dR, q, g, gt, nullptr, tc_prev, lam, c0, LG, LSE, LSE0, dtc_prev, dq, scratch, n_tok, d,
                         N, n, accum, finalize, neg_out, dtype, stream);
}

int lb_read_bwd_final(const void *V, const float *R, void *dV, float *dR, const float *q, const void *g,
                      const float *gt, const float *cbar, const float *c0, const float *LG, const float *LSE,
                      const float *LSE0, float *dcbar, float *dq, void *scratch, void *neg_out, int64_t n_tok, int d,
                      int N, int n, int accum, int dtype, void *stream) {
    if (neg_out && !aligned16(neg_out)) return fail(LB_ERR_ALIGN, "lb_read_bwd_final: neg_out must be 16-byte aligned");
    if (!cbar) return fail(LB_ERR_ARG, "lb_read_bwd_final: NULL pointer");
    return read_bwd_impl(V, R, dV, dR, q, g, gt, cbar, nullptr, 1.f, c0, LG, LSE, LSE0, dcbar, dq, scratch, n_tok, d, N, n,
                         accum, 1, neg_out, dtype, stream);
}

int lb_step_bwd(const void *V, const float *R, void *dV, float *dR, const float *q, const void *g, const float *gt,
                const float *tc_prev, float lam, const float *c0, const float *LG, const float *LSE, const float *LSE0,
                float *dtc_prev, float *dq, void *scratch, void *dh, void *dx, void *dh0, int dh0_accum, int blend,
                float beta, int64_t n_tok, int d, int N, int n, int accum, int dtype, void *stream) {
    if (n < 2 || !tc_prev) return fail(LB_ERR_ARG, "lb_step_bwd: needs n >= 2 and the previous read's coefficients");
    if (!dh || !dx) return fail(LB_ERR_ARG, "lb_step_bwd: dh and dx must be non-NULL");
    if (!aligned16(dh) || !aligned16(dx) || (dh0 && !aligned16(dh0)))
        return fail(LB_ERR_ALIGN, "lb_step_bwd: dh, dx and dh0 must be 16-byte aligned");
    if (dh0 && !blend) return fail(LB_ERR_ARG, "lb_step_bwd: dh0 is only produced by a read that closes an iteration");
    StepGrads sg;
    sg.dh = dh; sg.dh0 = dh0; sg.dh0_accum = dh0 ? dh0_accum : 0; sg.blend = blend ? 1 : 0; sg.beta = beta;
    sg.skip_final_store = 1;
    return read_bwd_impl(V, R, dV, dR, q, g, gt, nullptr, tc_prev, lam, c0, LG, LSE, LSE0, dtc_prev, dq, scratch, n_tok, d,
                         N, n, accum, 1, dx, dtype, stream, sg);
}

size_t lb_permuted_query_row_floats(int d, int dtype) {
    if (d <= 0 || (dtype != LB_DTYPE_BF16 && dtype != LB_DTYPE_F32)) return 0;
    return (size_t)chunks_of(d, dtype) * (lb::kChunkBytes / (dtype == LB_DTYPE_BF16 ? 2 : 4));
}

int lb_permute_queries(const float *Q, float *Qp, int NQ, int d, int dtype, void *stream) {
    int rc = check_common(0, d, dtype);
    if (rc) return rc;
    if (!Q || !Qp || NQ < 0) return fail(LB_ERR_ARG, "lb_permute_queries: NULL pointer or negative size");
    cudaError_t e = lb::launch_permute_queries(Q, Qp, NQ, d, dtype == LB_DTYPE_BF16 ? 8 : 4,
                                               (int)lb_permuted_query_row_floats(d, dtype), static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? LB_OK : cuda_fail(e, "lb_permute_queries launch");
}

int lb_peer_flag_words(void) { return lb::kPeerFlagWords; }

int lb_peer_allreduce(const float *const *bufs, unsigned int *const *flags, int rank, int world, float *out, int64_t n,
                      void *stream) {
    if (!bufs || !flags || !out) return fail(LB_ERR_ARG, "lb_peer_allreduce: NULL pointer");
    if (world < 1 || world > lb::kMaxPeers || rank < 0 || rank >= world)
        return fail(LB_ERR_ARG, "lb_peer_allreduce: needs 1 <= world <= LB_MAX_PEERS and 0 <= rank < world");
    if (n < 0 || n % 4) return fail(LB_ERR_ARG, "lb_peer_allreduce: n must be a non-negative multiple of 4 floats");
    if (n == 0) return LB_OK;
    lb::PeerReduceParams p{};
    for (int r = 0; r < world; ++r) {
        if (!bufs[r] || !flags[r]) return fail(LB_ERR_ARG, "lb_peer_allreduce: NULL peer pointer");
        if (!aligned16(bufs[r]) || ((uintptr_t)flags[r] & 3u)) return fail(LB_ERR_ALIGN, "lb_peer_allreduce: buffers must be 16-byte aligned");
        p.bufs[r] = bufs[r]; p.flags[r] = flags[r];
    }
    if (!aligned16(out)) return fail(LB_ERR_ALIGN, "lb_peer_allreduce: out must be 16-byte aligned");
    DeviceInfo di;
    int rc;
    if ((rc = device_info(&di))) return rc;
    p.out = out; p.n4 = n / 4; p.rank = rank; p.world = world;
    p.wait_cycles = wait_limit(); p.err_word = di.err_word;
    cudaError_t e = lb::launch_peer_allreduce(p, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? LB_OK : cuda_fail(e, "lb_peer_allreduce launch");
}

int lb_step_bwd_deferred(const void *V, const float *R, void *G, float *dR, float *Wt, float *KQt, const float *Q,
                         const float *Qp, const void *g, const float *gt, const float *tc_prev, float lam, const float *c0, const float *LG,
                         const float *LSE, const float *LSE0, float *dtc_prev, float *dq, void *scratch, void *dh, void *dx,
                         void *dh0, int dh0_accum, int blend, float beta, void *dv0, void *dx0, int64_t n_tok, int d, int N,
                         int n, int first, int dtype, void *stream) {
    if (n < 2 || !tc_prev) return fail(LB_ERR_ARG, "lb_step_bwd_deferred: needs n >= 2 and the previous read's coefficients");
    if (!G || !Wt || !KQt || !Q || !Qp || !dh || !dx) return fail(LB_ERR_ARG, "lb_step_bwd_deferred: NULL pointer");
    if (!aligned16(G) || !aligned16(Q) || !aligned16(Qp) || !aligned16(dh) || !aligned16(dx) || (dh0 && !aligned16(dh0)) ||
        (dv0 && !aligned16(dv0)) || (dx0 && !aligned16(dx0)))
        return fail(LB_ERR_ALIGN, "lb_step_bwd_deferred: G, Q, dh, dx, dh0, dv0 and dx0 must be 16-byte aligned");
    if (((long long)d * 4) % 16) return fail(LB_ERR_ALIGN, "lb_step_bwd_deferred: the query rows must be multiples of 16 bytes");
    if (dh0 && !blend) return fail(LB_ERR_ARG, "lb_step_bwd_deferred: dh0 is only produced by a read that closes an iteration");
    if ((dv0 != nullptr) != (dx0 != nullptr) || (dv0 && n != 2))
        return fail(LB_ERR_ARG, "lb_step_bwd_deferred: dv0 and dx0 come together, from the step-1 backward (n == 2) only");
    StepGrads sg;
    sg.dh = dh; sg.dh0 = dh0; sg.dh0_accum = dh0 ? dh0_accum : 0; sg.blend = blend ? 1 : 0; sg.beta = beta;
    sg.skip_final_store = 1;
    sg.deferred = 1; sg.Wt = Wt; sg.KQt = KQt; sg.Qall = Qp; sg.dv0 = dv0; sg.dx0 = dx0;
    return read_bwd_impl(V, R, G, dR, Q + (long long)(n - 2) * d, g, gt, nullptr, tc_prev, lam, c0, LG, LSE, LSE0, dtc_prev, dq,
                         scratch, n_tok, d, N, n, first ? 0 : 1, 1, dx, dtype, stream, sg);
}

static int read_bwd_impl(const void *V, const float *R, void *dV, float *dR, const float *q, const void *g,
                         const float *gt, const float *cbar, const float *tc_prev, float lam, const float *c0,
                         const float *LG, const float *LSE, const float *LSE0, float *dcbar, float *dq, void *scratch,
                         int64_t n_tok, int d, int N, int n, int accum, int finalize, void *neg_out, int dtype,
                         void *stream, const StepGrads &sg) {
    int rc = check_common(n_tok, d, dtype);
    if (rc) return rc;
    if (!V || !R || !dV || !dR || !q || !g || (!cbar && !tc_prev) || !c0 || !LG || !LSE || !LSE0 || !dcbar || !dq || !scratch)
        return fail(LB_ERR_ARG, "lb_read_bwd: NULL pointer");
    if (n < 1 || n > N) return fail(LB_ERR_ARG, "lb_read_bwd: n=%d outside [1, N=%d]", n, N);
    if (n > LB_MAX_SOURCES) return fail(LB_ERR_UNSUPPORTED, "lb_read_bwd: n=%d exceeds LB_MAX_SOURCES=%d", n, LB_MAX_SOURCES);
    if (!aligned16(V) || !aligned16(dV) || !aligned16(g) || !aligned16(q) || !aligned16(scratch))
        return fail(LB_ERR_ALIGN, "lb_read_bwd: V, dV, g, q and scratch must be 16-byte aligned");
    DeviceInfo di;
    if ((rc = device_info(&di))) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (n_tok == 0) {
        cudaError_t e0 = cudaMemsetAsync(dq, 0, sizeof(float) * d, st);
        return e0 == cudaSuccess ? LB_OK : cuda_fail(e0, "cudaMemsetAsync(dq)");
    }

    const int nch = chunks_of(d, dtype);
    const int elem = dtype == LB_DTYPE_BF16 ? 2 : 4;
    const bool rank4 = !g_opt.tma_per_chunk && (d * elem) % lb::kChunkBytes == 0;
    // Tile shape. A row of at most 4 chunks goes to ONE warp per token (8 consumer warps, 8 tokens per tile): no
    // exchange between warps and the most work per barrier wait. Wider rows are split over several warps per token:
    // consumer warps (12, 16 or 8), warps per token and fragments per warp are chosen for no idle fragments first,
    // then tiles of at least 12 KiB, then 2 fragments per warp.
    int ncw = 0, wpt = 0, fr = 0, best_cost = 1 << 30;
    static const int kNcw[3] = {12, 16, 8}, kFrMax[3] = {2, 2, 4};
    if (nch <= 4 && g_opt.bwd_wpt <= 1 && (g_opt.bwd_warps == 0 || g_opt.bwd_warps == 8 || g_opt.bwd_warps == 4)) {
        // 8 consumer warps and one CTA per SM, or ("bwd_warps" = 4) half-size CTAs of 4 consumer warps, two per SM:
        // two independent pipelines whose phases drift apart (no faster since phase 1 became straight-line code: an option only)
        const bool half = g_opt.bwd_warps == 4;
        ncw = half ? 4 : 8; wpt = 1; fr = nch;
    } else if (sg.deferred && !g_opt.bwd_warps && !g_opt.bwd_wpt && (nch == 8 || nch == 16 || nch == 32)) {
        // the deferred form keeps g packed and has registers for 3 or 4 fragments per warp: 8 consumer warps, fewer warps
        // per token to exchange partial dot products between (measured: -15 % at 8 chunks, -6 % at 12)
        ncw = 8; fr = 4; wpt = nch / 4;
    } else if (sg.deferred && !g_opt.bwd_warps && !g_opt.bwd_wpt && (nch == 6 || nch == 12 || nch == 24)) {
        ncw = 8; fr = 3; wpt = nch / 3;
    } else {
        for (int a = 0; a < 3; ++a) {
            if (g_opt.bwd_warps && g_opt.bwd_warps != kNcw[a]) continue;
            for (int w = 2; w <= kNcw[a]; ++w) {
                if (kNcw[a] % w || kNcw[a] / w > 8) continue;     // named barriers 1..8: one per token of the tile
                if (g_opt.bwd_wpt && g_opt.bwd_wpt != w) continue;
                const int f = (nch + w - 1) / w;
                if (f > kFrMax[a]) continue;
                const int stage = nch * (kNcw[a] / w) * lb::kChunkBytes;
                const int cost = (f * w - nch) * 64 + (stage < 12 * 1024 ? 16 : 0) + (f == 2 ? 0 : (f == 3 ? 2 : (f == 1 ? 3 : 4))) * 2 + a;
                if (cost < best_cost) { best_cost = cost; ncw = kNcw[a]; wpt = w; fr = f; }
            }
        }
    }
    if (ncw == 0) return fail(LB_ERR_UNSUPPORTED, "lb_read_bwd: no tile shape covers d=%d (row of %d chunks)", d, nch);
    const int bt = ncw / wpt;
    const int vec = dtype == LB_DTYPE_BF16 ? 8 : 4;
    int stages = g_opt.bwd_stages > 0 ? g_opt.bwd_stages : 8;
    if (stages > 12) stages = 12;
    const int earlier = sg.deferred ? N - n : 0, qrow = sg.deferred ? (int)lb_permuted_query_row_floats(d, dtype) * 4 : 0;
    const size_t smem_cap = ncw == 4 ? (kMaxSmem - 2048) / 2 : kMaxSmem;      // two half-size CTAs share an SM
    while (stages > 2 && lb::read_bwd_smem_bytes(fr, ncw, wpt, stages, n, vec, earlier, qrow) > smem_cap) --stages;
    if (lb::read_bwd_smem_bytes(fr, ncw, wpt, stages, n, vec, earlier, qrow) > smem_cap)
        return fail(LB_ERR_UNSUPPORTED, "lb_read_bwd: shared memory does not fit for d=%d, n=%d", d, n);

    CUtensorMap tmV, tmG, tmDV, tmH0;
    if ((rc = make_map(&tmV, V, dtype, n_tok, d, N, bt, rank4 ? nch : 0))) return rc;
    if ((rc = make_map(&tmG, g, dtype, n_tok, d, 0, bt, rank4 ? nch : 0))) return rc;
    if ((rc = make_map(&tmDV, dV, dtype, n_tok, d, N, bt, rank4 ? nch : 0))) return rc;
    if ((rc = make_map(&tmH0, sg.dh0 ? sg.dh0 : g, dtype, n_tok, d, 0, bt, rank4 ? nch : 0))) return rc;

    lb::ReadBwdParams p;
    p.R = R; p.dR = dR; p.dV = dV; p.q = q; p.gt = gt; p.cbar = cbar; p.tc_prev = tc_prev; p.lam = lam; p.c0 = c0; p.LSE = LSE; p.LSE0 = LSE0; p.LG = LG;
    p.dcbar = dcbar; p.dq_part = static_cast<float *>(scratch);
    p.n_tok = n_tok; p.tok_tiles = (n_tok + bt - 1) / bt; p.d = d; p.n = n; p.chunks = nch; p.wpt = wpt;
    p.stages = stages; p.rank4 = rank4 ? 1 : 0; p.accum = accum ? 1 : 0; p.finalize = finalize ? 1 : 0;
    p.neg_out = finalize ? neg_out : nullptr; p.inv_sqrt_d = 1.0f / sqrtf((float)d);
    p.dh_out = finalize ? sg.dh : nullptr; p.dh0 = finalize ? sg.dh0 : nullptr; p.dh0_accum = sg.dh0_accum;
    p.blend = sg.blend; p.beta = sg.beta; p.skip_final_store = finalize ? sg.skip_final_store : 0;
    p.err_word = di.err_word; p.wait_cycles = wait_limit();
    if (sg.deferred) {
        p.Gst = dV; p.Wt = sg.Wt; p.KQt = sg.KQt; p.Qall = sg.Qall; p.qrow_bytes = qrow; p.n_total = N;
        p.fin2 = sg.dv0 ? 1 : 0; p.dv0_out = sg.dv0; p.neg0_out = sg.dx0;
    }
    int cap = g_opt.grid_cap > 0 ? g_opt.grid_cap : di.sms * (ncw == 4 ? 2 : 1);
    if (cap > kMaxGrid) cap = kMaxGrid;
    const int grid = (int)(p.tok_tiles < cap ? p.tok_tiles : cap);
    cudaError_t e = lb::launch_read_bwd(dtype, fr, ncw, tmV, tmG, tmDV, tmH0, p, grid, st);
    if (e != cudaSuccess) return cuda_fail(e, "lb_read_bwd launch");
    if (p.dh0 != nullptr && wpt > 1) {
        // shapes with several warps per token leave the loop input's gradient to a small kernel of its own (in their
        // main kernel the extra code cost every launch 2-3 %, boundary read or not)
        e = lb::launch_scale_acc(dtype, g, p.dh0, p.beta, p.dh0_accum, (long long)n_tok * d, di.sms, st);
        if (e != cudaSuccess) return cuda_fail(e, "lb_step_bwd h0-gradient launch");
    }
    e = lb::launch_dq_reduce(p.dq_part, grid, dq, d, p.inv_sqrt_d, st);
    return e == cudaSuccess ? LB_OK : cuda_fail(e, "lb_read_bwd dq reduction launch");
}

// ---------------------------------------------------------------------------------------------------------
// what surrounds a block
// ---------------------------------------------------------------------------------------------------------
static int check_block(const char *who, int64_t n_tok, int d, int dtype, int wdtype) {
    const int rc = check_common(n_tok, d, dtype);
    if (rc) return rc;
    if (wdtype != dtype && wdtype != LB_DTYPE_F32)
        return fail(LB_ERR_ARG, "%s: parameters have the rows' storage type or fp32 (dtype %d, wdtype %d)", who, dtype, wdtype);
    return LB_OK;
}

static int check_drop(const char *who, int threshold, const int64_t *rng, const int64_t *rng_used) {
    if (threshold < 0 || threshold > 65535) return fail(LB_ERR_ARG, "%s: threshold %d outside [0, 65535]", who, threshold);
    if ((reinterpret_cast<uintptr_t>(rng) & 7u) || (reinterpret_cast<uintptr_t>(rng_used) & 7u))
        return fail(LB_ERR_ALIGN, "%s: rng and rng_used must be 8-byte aligned", who);
    return LB_OK;
}

// the "block_frags" knob: 1..4, else chosen by size
static int block_frags() { return g_opt.block_frags >= 1 && g_opt.block_frags <= 4 ? g_opt.block_frags : 0; }

static lb::DropParams drop_params(int threshold, const int64_t *rng, int64_t seed, int64_t offset, int64_t *rng_used) {
    lb::DropParams dp;
    dp.threshold = (unsigned)threshold;
    dp.keep_scale = (float)(65536.0 / (65536.0 - threshold));
    dp.rng = reinterpret_cast<const long long *>(rng);
    dp.seed = seed; dp.offset = offset;
    dp.rng_used = reinterpret_cast<long long *>(rng_used);
    return dp;
}

static size_t block_part_floats(int d) { return 2 * (size_t)kMaxGrid * (size_t)d; }

size_t lb_block_scratch_bytes(int d) {
    if (d <= 0) return 0;
    return sizeof(float) * block_part_floats(d) + sizeof(double) * (((size_t)d + 31) / 32) + 16;
}

// the parts of `scratch`, and zeros for the parameters' gradients of an empty batch
static int finish_block_bwd(const char *who, lb::BlockParams &p, void *scratch, int dtype, int wdtype, bool residual,
                            cudaStream_t st) {
    DeviceInfo di;
    const int rc = device_info(&di);
    if (rc) return rc;
    cudaError_t e = cudaSuccess;
    if (p.n_tok == 0) {
        const size_t wb = (size_t)p.d * (wdtype == LB_DTYPE_BF16 ? 2 : 4);
        if (p.dw) e = cudaMemsetAsync(p.dw, 0, wb, st);
        if (e == cudaSuccess && p.dw_next) e = cudaMemsetAsync(p.dw_next, 0, wb, st);
        if (e == cudaSuccess && p.dgate && p.gate_kind == lb::kGateChannel) e = cudaMemsetAsync(p.dgate, 0, wb, st);
        if (e == cudaSuccess && p.dscale) e = cudaMemsetAsync(p.dscale, 0, sizeof(float), st);
        return e == cudaSuccess ? LB_OK : cuda_fail(e, who);
    }
    p.need_a = p.dw || p.dscale || (p.dgate && p.gate_kind == lb::kGateChannel);
    if (p.need_a || p.dw_next) {
        if (!scratch) return fail(LB_ERR_ARG, "%s: parameter gradients need scratch", who);
        if (!aligned16(scratch)) return fail(LB_ERR_ALIGN, "%s: scratch must be 16-byte aligned", who);
        p.part = static_cast<float *>(scratch);
        p.ds_part = reinterpret_cast<double *>(p.part + block_part_floats(p.d));
        if (p.dscale) p.counter = reinterpret_cast<unsigned *>(p.ds_part + (p.d + 31) / 32);
    }
    e = lb::launch_block(dtype, wdtype, residual, true, p, di.sms, st);
    return e == cudaSuccess ? LB_OK : cuda_fail(e, who);
}

int lb_norm_fwd(const void *x, const void *w, void *u, float *r, int64_t n_tok, int d, float eps, int dtype, int wdtype,
                void *stream) {
    int rc = check_block("lb_norm_fwd", n_tok, d, dtype, wdtype);
    if (rc) return rc;
    if (n_tok == 0) return LB_OK;
    if (!x || !w || !u) return fail(LB_ERR_ARG, "lb_norm_fwd: x, w and u must be non-NULL");
    if (!aligned16(x) || !aligned16(w) || !aligned16(u)) return fail(LB_ERR_ALIGN, "lb_norm_fwd: x, w and u must be 16-byte aligned");
    DeviceInfo di;
    if ((rc = device_info(&di))) return rc;
    lb::BlockParams p;
    p.x = x; p.w_next = w; p.u = u; p.r_o = r; p.n_tok = n_tok; p.d = d; p.eps = eps;
    p.frags = d / (dtype == LB_DTYPE_BF16 ? 8 : 4); p.most_frags = block_frags();
    const cudaError_t e = lb::launch_block(dtype, wdtype, false, false, p, di.sms, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? LB_OK : cuda_fail(e, "lb_norm_fwd launch");
}

int lb_norm_bwd(const void *x, const void *w, const float *r, const void *du, void *dx, void *dw, void *scratch,
                int64_t n_tok, int d, int dtype, int wdtype, void *stream) {
    const int rc = check_block("lb_norm_bwd", n_tok, d, dtype, wdtype);
    if (rc) return rc;
    if (n_tok > 0 && (!x || !w || !r || !du)) return fail(LB_ERR_ARG, "lb_norm_bwd: x, w, r and du must be non-NULL");
    if (!aligned16(x) || !aligned16(w) || !aligned16(du) || !aligned16(dx))
        return fail(LB_ERR_ALIGN, "lb_norm_bwd: x, w, du and dx must be 16-byte aligned");
    lb::BlockParams p;
    p.x = x; p.w_next = w; p.r_o = const_cast<float *>(r); p.d_u = du; p.dx = dx; p.dw_next = dw; p.n_tok = n_tok; p.d = d;
    p.frags = d / (dtype == LB_DTYPE_BF16 ? 8 : 4); p.most_frags = block_frags();
    return finish_block_bwd("lb_norm_bwd", p, scratch, dtype, wdtype, false, static_cast<cudaStream_t>(stream));
}

static int check_gate(const char *who, const void *gate, int kind) {
    if (kind < LB_GATE_NONE || kind > LB_GATE_FULL) return fail(LB_ERR_ARG, "%s: unknown gate kind %d", who, kind);
    if ((kind != LB_GATE_NONE) != (gate != nullptr)) return fail(LB_ERR_ARG, "%s: gate and gate_kind do not agree", who);
    if (kind >= LB_GATE_CHANNEL && !aligned16(gate)) return fail(LB_ERR_ALIGN, "%s: gate must be 16-byte aligned", who);
    return LB_OK;
}

int lb_residual_fwd(const void *x, const void *y, const void *w, const void *gate, int gate_kind, const float *scale_dev,
                    float scale, const void *next_w, void *out, void *u, float *r_y, float *r_o, int threshold,
                    const int64_t *rng, int64_t seed, int64_t offset, int64_t *rng_used, int64_t n_tok, int d, float eps,
                    int dtype, int wdtype, void *stream) {
    int rc = check_block("lb_residual_fwd", n_tok, d, dtype, wdtype);
    if (rc || (rc = check_drop("lb_residual_fwd", threshold, rng, rng_used))) return rc;
    if (n_tok == 0) return LB_OK;
    if ((rc = check_gate("lb_residual_fwd", gate, gate_kind))) return rc;
    if (!x || !y || !out || (next_w && !u)) return fail(LB_ERR_ARG, "lb_residual_fwd: x, y, out (and u with next_w) must be non-NULL");
    if (!aligned16(x) || !aligned16(y) || !aligned16(w) || !aligned16(next_w) || !aligned16(out) || !aligned16(u))
        return fail(LB_ERR_ALIGN, "lb_residual_fwd: rows and weights must be 16-byte aligned");
    DeviceInfo di;
    if ((rc = device_info(&di))) return rc;
    lb::BlockParams p;
    p.x = x; p.y = y; p.w = w; p.gate = gate; p.gate_kind = gate_kind; p.scale_dev = scale_dev; p.scale = scale; p.w_next = next_w;
    p.out = out; p.u = u; p.r_y = r_y; p.r_o = r_o; p.n_tok = n_tok; p.d = d; p.eps = eps;
    p.drop = drop_params(threshold, rng, seed, offset, rng_used);
    p.frags = d / (dtype == LB_DTYPE_BF16 ? 8 : 4); p.most_frags = block_frags();
    const cudaError_t e = lb::launch_block(dtype, wdtype, true, false, p, di.sms, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? LB_OK : cuda_fail(e, "lb_residual_fwd launch");
}

int lb_residual_bwd(const void *x, const void *y, const void *w, const void *gate, int gate_kind, const float *scale_dev,
                    float scale, const void *next_w, const float *r_y, const float *r_o, int threshold, const int64_t *rng,
                    int64_t seed, int64_t offset, const void *d_out, const void *d_u, void *dx, void *dy, void *dw,
                    void *dgate, float *dscale, void *dnext_w, void *scratch, int64_t n_tok, int d, int dtype, int wdtype,
                    void *stream) {
    int rc = check_block("lb_residual_bwd", n_tok, d, dtype, wdtype);
    if (rc || (rc = check_drop("lb_residual_bwd", threshold, rng, nullptr))) return rc;
    if (n_tok > 0) {
        if ((rc = check_gate("lb_residual_bwd", gate, gate_kind))) return rc;
        if (!x || !y || (!d_out && !d_u)) return fail(LB_ERR_ARG, "lb_residual_bwd: x, y and an upstream gradient must be non-NULL");
        if ((d_u && (!next_w || !r_o)) || (w && !r_y)) return fail(LB_ERR_ARG, "lb_residual_bwd: a norm's backward needs its weight and row scales");
    }
    if ((dw && !w) || (dnext_w && !next_w) || (dgate && gate_kind == LB_GATE_NONE) || (dscale && !scale_dev))
        return fail(LB_ERR_ARG, "lb_residual_bwd: a gradient is wanted of a parameter that is not there");
    if (!aligned16(x) || !aligned16(y) || !aligned16(w) || !aligned16(next_w) || !aligned16(d_out) || !aligned16(d_u) ||
        !aligned16(dx) || !aligned16(dy) || (gate_kind == LB_GATE_FULL && !aligned16(dgate)))
        return fail(LB_ERR_ALIGN, "lb_residual_bwd: rows and weights must be 16-byte aligned");
    lb::BlockParams p;
    p.x = x; p.y = y; p.w = w; p.gate = gate; p.gate_kind = gate_kind; p.scale_dev = scale_dev; p.scale = scale; p.w_next = next_w;
    p.r_y = const_cast<float *>(r_y); p.r_o = const_cast<float *>(r_o); p.d_out = d_out; p.d_u = d_u;
    p.dx = dx; p.dy = dy; p.dw = dw; p.dgate = dgate; p.dscale = dscale; p.dw_next = dnext_w; p.n_tok = n_tok; p.d = d;
    p.drop = drop_params(threshold, rng, seed, offset, nullptr);
    p.frags = d / (dtype == LB_DTYPE_BF16 ? 8 : 4); p.most_frags = block_frags();
    if (!d_u) p.dw_next = nullptr;
    rc = finish_block_bwd("lb_residual_bwd", p, scratch, dtype, wdtype, true, static_cast<cudaStream_t>(stream));
    if (rc || d_u || !dnext_w) return rc;
    const cudaError_t e = cudaMemsetAsync(dnext_w, 0, (size_t)d * (wdtype == LB_DTYPE_BF16 ? 2 : 4), static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? LB_OK : cuda_fail(e, "lb_residual_bwd");
}

int lb_dropout(const void *x, void *out, int threshold, const int64_t *rng, int64_t seed, int64_t offset, int64_t *rng_used,
               int64_t n_elem, int dtype, void *stream) {
    if (dtype != LB_DTYPE_BF16 && dtype != LB_DTYPE_F32) return fail(LB_ERR_ARG, "bad dtype %d", dtype);
    if (n_elem < 0) return fail(LB_ERR_ARG, "lb_dropout: negative size");
    int rc = check_drop("lb_dropout", threshold, rng, rng_used);
    if (rc) return rc;
    if (n_elem > 0 && (!x || !out || x == out)) return fail(LB_ERR_ARG, "lb_dropout: x and out must be non-NULL and two buffers");
    if (!aligned16(x) || !aligned16(out)) return fail(LB_ERR_ALIGN, "lb_dropout: x and out must be 16-byte aligned");
    DeviceInfo di;
    if ((rc = device_info(&di))) return rc;
    const cudaError_t e = lb::launch_dropout(dtype, x, out, n_elem, drop_params(threshold, rng, seed, offset, rng_used), di.sms,
                                             static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? LB_OK : cuda_fail(e, "lb_dropout launch");
}

// ---------------------------------------------------------------------------------------------------------
// the gated feed-forward block
// ---------------------------------------------------------------------------------------------------------
// 2-D bf16 matrix [rows][cols], `ld` columns from row to row; boxes of 64 columns x box_rows rows, 128-byte swizzle (or 32
// columns, 64-byte swizzle)
static int make_map_tile(CUtensorMap *m, const void *base, long long rows, long long cols, long long ld, int box_rows,
                         int box_cols = 64) {
    auto fn = encode_fn();
    if (!fn) return fail(LB_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
    cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1, 1};
    CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void *>(base), dims, strides, box, estr,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, box_cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(LB_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
    return LB_OK;
}

// the fp32 slices [splits][rows][cols] of a product split along k; boxes of 32 columns x 32 rows
static int make_map_part(CUtensorMap *m, void *base, long long rows, long long cols, int splits) {
    auto fn = encode_fn();
    if (!fn) return fail(LB_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
    cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)splits};
    cuuint64_t strides[2] = {(cuuint64_t)cols * 4, (cuuint64_t)cols * 4 * (cuuint64_t)rows};
    cuuint32_t box[3] = {32, 32, 1};
    cuuint32_t estr[3] = {1, 1, 1};
    CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(LB_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
    return LB_OK;
}

struct GemmPlan {
    int tile = 0, splits = 1;
    bool cluster = false;              // k split over the CTAs of a cluster, no slices
    int m_tiles = 0, n_tiles = 0, m_tiles2 = 0, n_tiles2 = 0;
    double us = 1e30;                  // estimated
};

// Tile shape and split along k of an m x n product over `blocks` blocks of 64 (and an m2 x n2 one beside it): the least
// estimated time.
static GemmPlan plan_gemm(long long m, long long n, long long blocks, int epi, bool may_split, int sms, long long m2 = 0,
                          long long n2 = 0) {
    GemmPlan best;
    const bool gate = epi == lb::kEpiGate, plain = epi == lb::kEpiStore;
    const int shapes = lb::kGemmTileCount - !plain;                    // the last one is for plain products
    for (int i = 0; i < shapes; ++i) {
        if (g_opt.ffn_tile > 0 && g_opt.ffn_tile <= shapes && g_opt.ffn_tile - 1 != i) continue;
        const int cg = lb::kGemmTiles[i].cg, bn = lb::kGemmTiles[i].bn;
        const long long tm = 128LL * cg, tn = gate ? bn / 2 : bn, groups = sms / cg;
        const long long mt = (m + tm - 1) / tm, nt = (n + tn - 1) / tn, mt2 = (m2 + tm - 1) / tm, nt2 = (n2 + tn - 1) / tn;
        const int most = !may_split || blocks < 8 || bn > 256 ? 1 : blocks / 4 < 16 ? (int)(blocks / 4) : 16;
        const int forced = g_opt.ffn_splits <= 0 || most == 1 ? 0 : g_opt.ffn_splits < most ? g_opt.ffn_splits : most;
        for (int s = forced ? forced : 1; s <= (forced ? forced : most); ++s) {
            const double waves = (double)((mt * nt * s + mt2 * nt2 + groups - 1) / groups);
            // us per block of 64 of a tile, as measured with the SMs busy (a 128 x 128 tile is bound by what L2 delivers, the
            // 256-row ones by the tensor cores), a launch's fixed part, and the slices' way out and in
            const double rate = bn == 512 ? 0.58 : cg == 2 ? 0.345 : bn == 256 ? 0.39 : 0.30;
            double us = waves * (double)((blocks + s - 1) / s) * rate + 4.5 + bn / 128. + (cg == 2 ? 1.0 : 0.0);
            if (s > 1) us += 2.0 + (double)s * m * n * 8. / 9.0e6;
            if (us < best.us) {
                best.us = us; best.tile = i; best.splits = s; best.cluster = false;
                best.m_tiles = (int)mt; best.n_tiles = (int)nt; best.m_tiles2 = (int)mt2; best.n_tiles2 = (int)nt2;
            }
        }
    }
    return best;
}

// ... and the same with k split over a cluster, where the whole product is resident at once (two CTAs to an SM, less what the
// clusters' shapes leave unused). The constants are fitted to 100 .. 2048 rows of 768 .. 2048 columns over 32 .. 88 blocks.
static void plan_cluster(GemmPlan *best, long long m, long long n, long long blocks, int sms) {
    if (g_opt.ffn_tile > 0 && g_opt.ffn_tile != lb::kGemmTileCount + 1) return;
    const long long mt = (m + 127) / 128, nt = (n + 127) / 128;
    const int most = blocks / 2 < lb::kClusterSplits ? (int)(blocks / 2) : lb::kClusterSplits;
    for (int s = 2; s <= most && mt * nt * s * 4 <= 7LL * sms; ++s) {
        if (g_opt.ffn_splits > 0 && s != (g_opt.ffn_splits < most ? g_opt.ffn_splits : most)) continue;
        const double full = (double)(mt * nt * s) / sms;
        const double us = 5.5 + (full > 1.0 ? 0.50 : 0.25 + 0.10 * full) * (double)((blocks + s - 1) / s) + 0.45 * s;
        if (us < best->us || g_opt.ffn_tile == lb::kGemmTileCount + 1) {
            best->us = us; best->tile = 0; best->splits = s; best->cluster = true;
            best->m_tiles = (int)mt; best->n_tiles = (int)nt; best->m_tiles2 = best->n_tiles2 = 0;
        }
    }
}

struct Operand {
    const void *base;
    long long rows, cols, ld;         // as it lies in memory
};

// One product m x n over `segs` segments of k columns each, c[0] (through `part` where k is split); or, where the plan says so,
// two products over the same k: a[0] b[0] -> c[0] and a[1] b[1] -> c[1].
static int run_gemm(const char *who, int epi, int form, const GemmPlan &pl, const Operand *a, const Operand *b, const Operand *c,
                    void *kept, void *part, long long m, long long n, long long k, int segs, int act,
                    const DeviceInfo &di, cudaStream_t st) {
    lb::GemmMaps maps;
    memset(&maps, 0, sizeof maps);
    lb::GemmParams p;
    const int cg = lb::kGemmTiles[pl.tile].cg, bn = lb::kGemmTiles[pl.tile].bn;
    int rc;
    const bool split = pl.splits > 1 && !pl.cluster, two = pl.m_tiles2 > 0;
    const int pairs = two ? 2 : segs;
    for (int s = 0; s < pairs; ++s)
        if ((rc = make_map_tile(&maps.a[s], a[s].base, a[s].rows, a[s].cols, a[s].ld, form == lb::kFormMN ? 64 : 128))) return rc;
    for (int s = 0; s < (epi == lb::kEpiGate ? 2 : pairs); ++s)
        if ((rc = make_map_tile(&maps.b[s], b[s].base, b[s].rows, b[s].cols, b[s].ld,
                                form != lb::kFormKK ? 64 : epi == lb::kEpiGate ? bn / 2 : (bn < 256 ? bn : 256) / cg))) return rc;
    if (split) {
        if ((rc = make_map_part(&maps.c[0], part, m, n, pl.splits))) return rc;
    } else {
        for (int i = 0; i < (epi == lb::kEpiStore && !two ? 1 : 2); ++i)
            if (c[i].base && (rc = make_map_tile(&maps.c[i], c[i].base, c[i].rows, c[i].cols, c[i].ld, 32,
                                                    epi == lb::kEpiGate || epi == lb::kEpiGateBwd ? 32 : 64))) return rc;
    }
    p.m = (int)m; p.n = (int)n; p.kblocks = (int)((k + 63) / 64); p.segs = segs;
    p.m_tiles = pl.m_tiles; p.n_tiles = pl.n_tiles; p.splits = pl.splits; p.m_tiles2 = pl.m_tiles2; p.n_tiles2 = pl.n_tiles2;
    p.m2 = two ? (int)c[1].rows : 0; p.n2 = two ? (int)c[1].cols : 0; p.act = act; p.test_skip_item = g_opt.test_skip_item; p.kept = static_cast<uint8_t *>(kept);
    p.err_word = di.err_word; p.wait_cycles = wait_limit();
    if (pl.cluster) {
        const cudaError_t e = lb::launch_gemm_cluster(form, maps, p, const_cast<void *>(c[0].base), st);
        return e == cudaSuccess ? LB_OK : cuda_fail(e, who);
    }
    cudaError_t err = lb::launch_gemm(pl.tile, split ? (int)lb::kEpiPartial : epi, form, maps, p, di.sms, st);
    if (err == cudaSuccess && split)
        err = lb::launch_gemm_sum(static_cast<const float *>(part), const_cast<void *>(c[0].base), pl.splits, m * n, di.sms, st);
    return err == cudaSuccess ? LB_OK : cuda_fail(err, who);
}

struct FfnPlan {
    GemmPlan up, down, dh, dx, dw_gu, dw_down, dw_both;
    bool together = false;                              // both weight gradients in one launch
    size_t part = 0, bytes = 0;                         // offset of the slices in the workspace (dg | du, or h, lie before them), its size
};

// few rows and nothing kept: the kernels of lb_ffn_small.cu. The "ffn_small" knob: rows up to which they are taken (-1: never).
static bool ffn_small(long long t, int kind) {
    const int most = g_opt.ffn_small < 0 ? 0 : g_opt.ffn_small > 0 && g_opt.ffn_small < lb::kFfnSmallTokens ? g_opt.ffn_small : lb::kFfnSmallTokens;
    return kind == LB_FFN_INFERENCE && t <= most;
}

static FfnPlan plan_ffn(long long t, long long d, long long f, int kind, int sms) {
    FfnPlan q;
    const bool bwd = kind == LB_FFN_BACKWARD;
    if (ffn_small(t, kind)) {
        q.bytes = (size_t)t * (size_t)f * 2;
        return q;
    }
    const auto blocks = [](long long k) { return (k + 63) / 64; };
    size_t part = 0;
    const auto need = [&](const GemmPlan &g, long long m, long long n) {
        const size_t b = g.splits > 1 && !g.cluster ? (size_t)g.splits * (size_t)m * (size_t)n * 4 : 0;
        if (b > part) part = b;
    };
    if (!bwd) {
        q.up = plan_gemm(t, f, blocks(d), lb::kEpiGate, false, sms);
        q.down = plan_gemm(t, d, blocks(f), lb::kEpiStore, true, sms);
        plan_cluster(&q.down, t, d, blocks(f), sms);
        need(q.down, t, d);
    } else {
        q.dh = plan_gemm(t, f, blocks(d), lb::kEpiGateBwd, false, sms);
        q.dx = plan_gemm(t, d, 2 * blocks(f), lb::kEpiStore, true, sms);
        q.dw_gu = plan_gemm(2 * f, d, blocks(t), lb::kEpiStore, true, sms);
        q.dw_down = plan_gemm(d, f, blocks(t), lb::kEpiStore, true, sms);
        plan_cluster(&q.dx, t, d, 2 * blocks(f), sms);
        plan_cluster(&q.dw_gu, 2 * f, d, blocks(t), sms);
        plan_cluster(&q.dw_down, d, f, blocks(t), sms);
        // the two weight gradients are sums over the same rows: in one launch their tiles fill the last round together
        // (8192 x 1024 x 2816: 134 us apart)
        q.dw_both = plan_gemm(2 * f, d, blocks(t), lb::kEpiStore, false, sms, d, f);
        q.together = q.dw_both.us < q.dw_gu.us + q.dw_down.us;
        need(q.dx, t, d);
        need(q.dw_gu, 2 * f, d);
        need(q.dw_down, d, f);
    }
    const auto align = [](size_t b) { return (b + 255) / 256 * 256; };
    q.part = bwd ? align((size_t)t * (size_t)f * 4) : kind == LB_FFN_INFERENCE ? align((size_t)t * (size_t)f * 2) : 0;
    q.bytes = q.part + part;
    return q;
}

static int check_ffn(const char *who, int64_t n_tok, int d, int f, int act, int dtype) {
    if (dtype != LB_DTYPE_BF16) return fail(LB_ERR_UNSUPPORTED, "%s: the products run in bf16 (dtype %d)", who, dtype);
    if (act != LB_ACT_SILU && act != LB_ACT_GELU) return fail(LB_ERR_ARG, "%s: unknown activation %d", who, act);
    if (n_tok < 0 || d <= 0 || f <= 0) return fail(LB_ERR_ARG, "%s: n_tok=%lld, d=%d, f=%d: sizes must be positive", who, (long long)n_tok, d, f);
    if (d % 8 || f % 8) return fail(LB_ERR_ALIGN, "%s: d=%d and f=%d must be multiples of 8 (rows of 16-byte units)", who, d, f);
    if (d > (1 << 20) || f > (1 << 20) || n_tok >= (1LL << 31) - 512)
        return fail(LB_ERR_UNSUPPORTED, "%s: n_tok=%lld, d=%d, f=%d exceed the kernels' 32-bit coordinates", who, (long long)n_tok, d, f);
    return LB_OK;
}

size_t lb_ffn_workspace_bytes(int64_t n_tok, int d, int f, int kind) {
    if (check_ffn("lb_ffn_workspace_bytes", n_tok, d, f, LB_ACT_SILU, LB_DTYPE_BF16)) return 0;
    if (kind != LB_FFN_FORWARD && kind != LB_FFN_BACKWARD && kind != LB_FFN_INFERENCE) {
        fail(LB_ERR_ARG, "lb_ffn_workspace_bytes: unknown kind %d", kind);
        return 0;
    }
    DeviceInfo di;
    if (device_info(&di)) return 0;
    return plan_ffn(n_tok, d, f, kind, di.sms).bytes + 16;
}

size_t lb_ffn_kept_bytes(int64_t n_tok, int f) {
    if (check_ffn("lb_ffn_kept_bytes", n_tok, 8, f, LB_ACT_SILU, LB_DTYPE_BF16)) return 0;
    return (size_t)((n_tok + 31) / 32) * (size_t)((f + 31) / 32) * 12 * 512 + 16;
}

int lb_ffn_fwd(const void *x, const void *w_gate, const void *w_up, const void *w_down, void *y, void *h, void *kept,
               void *workspace, size_t workspace_bytes, int64_t n_tok, int d, int f, int act, int dtype, void *stream) {
    const char *who = "lb_ffn_fwd";
    int rc = check_ffn(who, n_tok, d, f, act, dtype);
    if (rc) return rc;
    if (n_tok == 0) return LB_OK;
    if (!x || !w_gate || !w_up || !w_down || !y || !workspace || (kept && !h)) return fail(LB_ERR_ARG, "%s: NULL pointer", who);
    if (!aligned16(x) || !aligned16(w_gate) || !aligned16(w_up) || !aligned16(w_down) || !aligned16(y) || !aligned16(h) ||
        !aligned16(kept) || !aligned16(workspace))
        return fail(LB_ERR_ALIGN, "%s: every pointer must be 16-byte aligned", who);
    DeviceInfo di;
    if ((rc = device_info(&di))) return rc;
    const int kind = h ? LB_FFN_FORWARD : LB_FFN_INFERENCE;
    const FfnPlan q = plan_ffn(n_tok, d, f, kind, di.sms);
    if (workspace_bytes < q.bytes) return fail(LB_ERR_ARG, "%s: workspace of %zu bytes, %zu are needed", who, workspace_bytes, q.bytes);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (!h) h = workspace;
    if (ffn_small(n_tok, kind)) {
        const int rows = lb::ffn_small_rows(n_tok);
        CUtensorMap m0, m1, mx;
        lb::FfnSmallParams p;
        p.n_tok = (int)n_tok; p.act = act; p.err_word = di.err_word; p.wait_cycles = wait_limit();
        p.test_skip_item = g_opt.test_skip_item;
        if ((rc = make_map_tile(&m0, w_gate, f, d, d, 64)) || (rc = make_map_tile(&m1, w_up, f, d, d, 64)) ||
            (rc = make_map_tile(&mx, x, n_tok, d, d, rows))) return rc;
        p.out = h; p.n = f; p.kblocks = (d + 63) / 64;
        cudaError_t e = lb::launch_ffn_small(true, rows, m0, m1, mx, p, di.sms, st);
        if (e != cudaSuccess) return cuda_fail(e, who);
        if ((rc = make_map_tile(&m0, w_down, d, f, f, 128)) || (rc = make_map_tile(&mx, h, n_tok, f, f, rows))) return rc;
        p.out = y; p.n = d; p.kblocks = (f + 63) / 64;
        e = lb::launch_ffn_small(false, rows, m0, m0, mx, p, di.sms, st);
        return e == cudaSuccess ? LB_OK : cuda_fail(e, who);
    }
    void *part = static_cast<char *>(workspace) + q.part;
    const Operand xs[1] = {{x, n_tok, d, d}}, w2[2] = {{w_gate, f, d, d}, {w_up, f, d, d}}, hs[2] = {{h, n_tok, f, f}, {}};
    if ((rc = run_gemm(who, lb::kEpiGate, lb::kFormKK, q.up, xs, w2, hs, kept, nullptr, n_tok, f, d, 1, act, di, st))) return rc;
    const Operand wd[1] = {{w_down, d, f, f}}, ys[2] = {{y, n_tok, d, d}, {}};
    return run_gemm(who, lb::kEpiStore, lb::kFormKK, q.down, hs, wd, ys, nullptr, part, n_tok, d, f, 1, act, di, st);
}

int lb_ffn_bwd(const void *x, const void *w_gate, const void *w_up, const void *w_down, const void *h, const void *kept,
               const void *dy, void *dx, void *dw_gate_up, void *dw_down, void *workspace, size_t workspace_bytes,
               int64_t n_tok, int d, int f, int dtype, void *stream) {
    const char *who = "lb_ffn_bwd";
    int rc = check_ffn(who, n_tok, d, f, LB_ACT_SILU, dtype);
    if (rc) return rc;
    if (!aligned16(x) || !aligned16(w_gate) || !aligned16(w_up) || !aligned16(w_down) || !aligned16(h) || !aligned16(kept) ||
        !aligned16(dy) || !aligned16(dx) || !aligned16(dw_gate_up) || !aligned16(dw_down) || !aligned16(workspace))
        return fail(LB_ERR_ALIGN, "%s: every pointer must be 16-byte aligned", who);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (n_tok == 0) {
        cudaError_t e = cudaSuccess;
        if (dw_gate_up) e = cudaMemsetAsync(dw_gate_up, 0, (size_t)4 * d * f, st);
        if (e == cudaSuccess && dw_down) e = cudaMemsetAsync(dw_down, 0, (size_t)2 * d * f, st);
        return e == cudaSuccess ? LB_OK : cuda_fail(e, who);
    }
    if (!x || !w_gate || !w_up || !w_down || !h || !kept || !dy || !workspace) return fail(LB_ERR_ARG, "%s: NULL pointer", who);
    DeviceInfo di;
    if ((rc = device_info(&di))) return rc;
    const FfnPlan q = plan_ffn(n_tok, d, f, LB_FFN_BACKWARD, di.sms);
    if (workspace_bytes < q.bytes) return fail(LB_ERR_ARG, "%s: workspace of %zu bytes, %zu are needed", who, workspace_bytes, q.bytes);
    void *part = static_cast<char *>(workspace) + q.part;
    char *dg = static_cast<char *>(workspace), *du = dg + (size_t)f * 2;          // [n_tok][2 f]: dg | du
    const long long t = n_tok, f2 = 2LL * f;
    const Operand dys[1] = {{dy, t, d, d}}, hs[1] = {{h, t, f, f}};
    if (dx || dw_gate_up) {
        // dh = dy Wd, turned into dg and du as it leaves the accumulators
        const Operand wds[1] = {{w_down, d, f, f}}, outs[2] = {{dg, t, f, f2}, {du, t, f, f2}};
        if ((rc = run_gemm(who, lb::kEpiGateBwd, lb::kFormKN, q.dh, dys, wds, outs, const_cast<void *>(kept), nullptr, t, f, d, 1, 0,
                           di, st))) return rc;
    }
    if (dx) {
        const Operand as[2] = {{dg, t, f, f2}, {du, t, f, f2}}, bs[2] = {{w_gate, f, d, d}, {w_up, f, d, d}};
        const Operand cs[2] = {{dx, t, d, d}, {}};
        if ((rc = run_gemm(who, lb::kEpiStore, lb::kFormKN, q.dx, as, bs, cs, nullptr, part, t, d, f, 2, 0, di, st))) return rc;
    }
    const Operand as[2] = {{dg, t, f2, f2}, dys[0]}, bs[2] = {{x, t, d, d}, hs[0]};
    const Operand cs[2] = {{dw_gate_up, f2, d, d}, {dw_down, d, f, f}}, none[2] = {cs[1], {}};
    if (dw_gate_up && dw_down && q.together)
        return run_gemm(who, lb::kEpiStore, lb::kFormMN, q.dw_both, as, bs, cs, nullptr, part, f2, d, t, 1, 0, di, st);
    if (dw_gate_up && (rc = run_gemm(who, lb::kEpiStore, lb::kFormMN, q.dw_gu, as, bs, cs, nullptr, part, f2, d, t, 1, 0, di, st)))
        return rc;
    if (dw_down && (rc = run_gemm(who, lb::kEpiStore, lb::kFormMN, q.dw_down, as + 1, bs + 1, none, nullptr, part, d, f, t, 1, 0, di, st)))
        return rc;
    return LB_OK;
}

}  // extern "C"
#pragma GCC visibility pop
