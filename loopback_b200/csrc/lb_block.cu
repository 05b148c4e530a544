// What surrounds a shared block between two reads: the norm before it, the norm after it with its gate, dropout, residual
// scale and the next block's norm, and their backward; and dropout on its own. All of it streams rows once:
//
//   n(v) = v rsqrt(mean(v^2) + eps)
//   norm       u = w n(x)
//   residual   o = x + s g m b,  b = w n(y) or y;   u = w' n(o)
//   backward   oh = o r_o, yh = y r_y (or y):  D = dout + r_o (w' du - oh mean(w' du oh)) = dx
//              E = s g m D,  dy = r_y (w E - yh mean(w E yh)) (or E)
//              per column A = sum_t g_t m D yh (g_t: a gate per token or per element; a channel's gate is applied at the end),
//              B = sum_t du oh:  dw = s g A, dgate = s w A, ds = sum_j g_j w_j A_j, dw' = B
//
// The backward recomputes o from x and y (both have to be read for dx and dy anyway), so neither o nor the mask is saved:
// only the two fp32 scales of each row. It reads and writes each row once.
//
// A row is handled by `wpt` warps (1, 2, 4 or 8 of the CTA's 8); a lane keeps FR fragments of 16 bytes of every row in
// registers, so the row is read once although its statistics are needed before its result. All arithmetic is fp32 with one
// rounding at each store.
#include "lb_common.cuh"
#include "lb_kernels.h"

namespace lb {

constexpr int kBlkThreads = 256;
constexpr int kBlkWarps = kBlkThreads / 32;

// ---------------------------------------------------------------------------------------------------------
// dropout's numbers: Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", 2011) with
// counter (group, offset) and key seed. A group is 8 consecutive elements; element j of it takes half j (low half first) of
// the four words, 16 bits: one call serves a 16-byte fragment of bf16, at half the integer work of a word per element.
// ---------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint4 philox4x32_10(unsigned long long group, unsigned long long offset, unsigned long long seed) {
    uint32_t c0 = (uint32_t)group, c1 = (uint32_t)(group >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const unsigned long long a = (unsigned long long)c0 * 0xD2511F53u, b = (unsigned long long)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}

// keeps or clears the VEC elements that start at linear index `e` (a multiple of VEC); a dropped element becomes 0 whatever
// it held
template <int VEC>
__device__ __forceinline__ void drop_fragment(float (&v)[VEC], unsigned long long e, const DropParams &dp,
                                              unsigned long long seed, unsigned long long offset) {
    const uint4 q = philox4x32_10(e >> 3, offset, seed);
    const bool high = VEC == 4 && (e & 4) != 0;
    const uint32_t w[4] = {high ? q.z : q.x, high ? q.w : q.y, q.z, q.w};
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        const uint32_t h = (j & 1) ? w[j >> 1] >> 16 : w[j >> 1] & 0xffffu;
        v[j] = h >= dp.threshold ? v[j] * dp.keep_scale : 0.f;
    }
}

__device__ __forceinline__ void drop_state(const DropParams &dp, unsigned long long &seed, unsigned long long &offset) {
    seed = dp.rng ? (unsigned long long)dp.rng[0] : (unsigned long long)dp.seed;
    offset = dp.rng ? (unsigned long long)dp.rng[1] : (unsigned long long)dp.offset;
}

// VEC weights (storage type W) from column c on
template <typename W, int VEC>
__device__ __forceinline__ void load_weights(const W *p, long long c, float (&f)[VEC]) {
    if constexpr (Store<W>::kVec == VEC) {
        Store<W>::unpack(*reinterpret_cast<const uint4 *>(p + c), f);
    } else {                                            // bf16 rows, fp32 weights
        const float4 a = *reinterpret_cast<const float4 *>(p + c), b = *reinterpret_cast<const float4 *>(p + c + 4);
        f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
        f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    }
}

// The sum over a row's `wpt` warps; every lane gets it. Two slot sets used in turn: a warp can write a set again only after
// every warp of the row has passed the barrier that follows its reads.
__device__ __forceinline__ float row_sum(float v, int wpt, int grp, int wl, int lane, float (*slots)[kBlkWarps], int &turn) {
    v = warp_sum(v);
    if (wpt == 1) return v;
    float *s = slots[turn] + grp * wpt;
    turn ^= 1;
    if (lane == 0) s[wl] = v;
    named_bar_sync(1 + grp, wpt * 32);
    float t = 0.f;
    for (int i = 0; i < wpt; ++i) t += s[i];
    return t;
}

template <typename T, typename W, int FR, bool RES>
__global__ void __launch_bounds__(kBlkThreads) block_fwd_kernel(const BlockParams p) {
    using S = Store<T>;
    constexpr int VEC = S::kVec;
    __shared__ float slots[2][kBlkWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int wpt = p.wpt, groups = kBlkWarps / wpt, grp = warp / wpt, wl = warp % wpt;
    const T *x = static_cast<const T *>(p.x), *y = static_cast<const T *>(p.y);
    const W *w = static_cast<const W *>(p.w), *w2 = static_cast<const W *>(p.w_next);
    T *out = static_cast<T *>(p.out), *u = static_cast<T *>(p.u);
    const float s = RES ? (p.scale_dev ? *p.scale_dev : p.scale) : 0.f;
    const float inv_d = 1.f / (float)p.d;
    unsigned long long seed = 0, offset = 0;
    if (RES && p.drop.threshold) {
        drop_state(p.drop, seed, offset);
        if (p.drop.rng_used && blockIdx.x == 0 && threadIdx.x == 0) {
            p.drop.rng_used[0] = (long long)seed;
            p.drop.rng_used[1] = (long long)offset;
        }
    }
    int turn = 0;
    const long long step = (long long)gridDim.x * groups;
    for (long long tok = (long long)blockIdx.x * groups + grp; tok < p.n_tok; tok += step) {
        const long long row = tok * p.d;
        uint4 xq[FR], yq[RES ? FR : 1];
#pragma unroll
        for (int k = 0; k < FR; ++k) {
            const int f = (k * wpt + wl) * 32 + lane;
            const bool in = f < p.frags;
            xq[k] = in ? ld_global_stream_v4(x + row + f * VEC) : make_uint4(0, 0, 0, 0);
            if constexpr (RES) yq[k] = in ? ld_global_stream_v4(y + row + f * VEC) : make_uint4(0, 0, 0, 0);
        }
        float o[FR][VEC];
        if constexpr (RES) {
            float ry = 1.f;
            if (w) {
                float ss = 0.f;
#pragma unroll
                for (int k = 0; k < FR; ++k) {
                    float v[VEC];
                    S::unpack(yq[k], v);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) ss = fmaf(v[e], v[e], ss);
                }
                ry = rsqrtf(row_sum(ss, wpt, grp, wl, lane, slots, turn) * inv_d + p.eps);
                if (p.r_y && wl == 0 && lane == 0) p.r_y[tok] = ry;
            }
            const float gt = p.gate_kind == kGateToken ? S::load1(static_cast<const T *>(p.gate) + tok) : 1.f;
            const float sg = s * gt;
#pragma unroll
            for (int k = 0; k < FR; ++k) {
                const int f = (k * wpt + wl) * 32 + lane;
                const bool in = f < p.frags;
                float b[VEC], g[VEC];
                S::unpack(yq[k], b);
                S::unpack(xq[k], o[k]);
                if (in) {
                    if (w) {
                        load_weights<W, VEC>(w, f * VEC, g);
#pragma unroll
                        for (int e = 0; e < VEC; ++e) b[e] = g[e] * (b[e] * ry);
                    }
                    if (p.drop.threshold) drop_fragment<VEC>(b, (unsigned long long)(row + f * VEC), p.drop, seed, offset);
                    if (p.gate_kind == kGateChannel) load_weights<W, VEC>(static_cast<const W *>(p.gate), f * VEC, g);
                    else if (p.gate_kind == kGateFull) S::unpack(ld_global_stream_v4(static_cast<const T *>(p.gate) + row + f * VEC), g);
                    if (p.gate_kind >= kGateChannel) {
#pragma unroll
                        for (int e = 0; e < VEC; ++e) b[e] *= g[e];
                    }
#pragma unroll
                    for (int e = 0; e < VEC; ++e) o[k][e] = fmaf(sg, b[e], o[k][e]);
                    st_global_v4(out + row + f * VEC, S::pack(o[k]));
                }
            }
            if (!w2) continue;
        } else {
#pragma unroll
            for (int k = 0; k < FR; ++k) S::unpack(xq[k], o[k]);
        }
        float ss = 0.f;
#pragma unroll
        for (int k = 0; k < FR; ++k)
#pragma unroll
            for (int e = 0; e < VEC; ++e) ss = fmaf(o[k][e], o[k][e], ss);
        const float ro = rsqrtf(row_sum(ss, wpt, grp, wl, lane, slots, turn) * inv_d + p.eps);
        if (p.r_o && wl == 0 && lane == 0) p.r_o[tok] = ro;
#pragma unroll
        for (int k = 0; k < FR; ++k) {
            const int f = (k * wpt + wl) * 32 + lane;
            if (f < p.frags) {
                float g[VEC];
                load_weights<W, VEC>(w2, f * VEC, g);
#pragma unroll
                for (int e = 0; e < VEC; ++e) g[e] *= o[k][e] * ro;
                st_global_v4(u + row + f * VEC, S::pack(g));
            }
        }
    }
}

// Per-CTA column sums leave through p.part[CTA][2][d] (A, then B); block_param_kernel adds the CTAs' rows in a fixed order.
template <typename T, typename W, int FR, bool RES>
__global__ void __launch_bounds__(kBlkThreads) block_bwd_kernel(const BlockParams p) {
    using S = Store<T>;
    constexpr int VEC = S::kVec;
    __shared__ float slots[2][kBlkWarps];
    extern __shared__ float cols[];                      // [2][d], only when several rows share the CTA
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int wpt = p.wpt, groups = kBlkWarps / wpt, grp = warp / wpt, wl = warp % wpt;
    const T *x = static_cast<const T *>(p.x), *y = static_cast<const T *>(p.y);
    const T *dout = static_cast<const T *>(p.d_out), *du = static_cast<const T *>(p.d_u);
    const W *w = static_cast<const W *>(p.w), *w2 = static_cast<const W *>(p.w_next);
    T *dx = static_cast<T *>(p.dx), *dy = static_cast<T *>(p.dy);
    const float s = RES ? (p.scale_dev ? *p.scale_dev : p.scale) : 0.f;
    const float inv_d = 1.f / (float)p.d;
    unsigned long long seed = 0, offset = 0;
    if (RES && p.drop.threshold) drop_state(p.drop, seed, offset);
    if (blockIdx.x == 0 && threadIdx.x == 0 && p.counter) *p.counter = 0;    // block_param_kernel counts its CTAs here
    float colA[RES ? FR : 1][VEC], colB[FR][VEC];
#pragma unroll
    for (int k = 0; k < FR; ++k)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            colB[k][e] = 0.f;
            if constexpr (RES) colA[k][e] = 0.f;
        }
    int turn = 0;
    const long long step = (long long)gridDim.x * groups;
    for (long long tok = (long long)blockIdx.x * groups + grp; tok < p.n_tok; tok += step) {
        const long long row = tok * p.d;
        const float ry = RES && w ? p.r_y[tok] : 1.f;
        const float ro = du ? p.r_o[tok] : 0.f;
        const float gt = RES && p.gate_kind == kGateToken ? S::load1(static_cast<const T *>(p.gate) + tok) : 1.f;
        const uint4 zero = make_uint4(0, 0, 0, 0);
        uint4 xq[FR], uq[FR], yq[RES ? FR : 1], gq[RES ? FR : 1];
        float D[FR][VEC];
#pragma unroll
        for (int k = 0; k < FR; ++k) {
            const int f = (k * wpt + wl) * 32 + lane;
            const bool in = f < p.frags;
            uq[k] = in && du ? ld_global_stream_v4(du + row + f * VEC) : zero;
            xq[k] = in && du ? ld_global_stream_v4(x + row + f * VEC) : zero;
            if constexpr (RES) {
                yq[k] = in ? ld_global_stream_v4(y + row + f * VEC) : zero;
                gq[k] = in && dout ? ld_global_stream_v4(dout + row + f * VEC) : zero;
            }
        }
        // the gradient of o through its norm
        float oh[FR][VEC];
        float acc = 0.f;
#pragma unroll
        for (int k = 0; k < FR; ++k) {
            const int f = (k * wpt + wl) * 32 + lane;
#pragma unroll
            for (int e = 0; e < VEC; ++e) D[k][e] = oh[k][e] = 0.f;
            if (f < p.frags && du) {
                float g[VEC];
                S::unpack(xq[k], oh[k]);
                if constexpr (RES) {
                    float b[VEC];
                    S::unpack(yq[k], b);
                    if (w) {
                        load_weights<W, VEC>(w, f * VEC, g);
#pragma unroll
                        for (int e = 0; e < VEC; ++e) b[e] = g[e] * (b[e] * ry);
                    }
                    if (p.drop.threshold) drop_fragment<VEC>(b, (unsigned long long)(row + f * VEC), p.drop, seed, offset);
                    if (p.gate_kind == kGateChannel) load_weights<W, VEC>(static_cast<const W *>(p.gate), f * VEC, g);
                    else if (p.gate_kind == kGateFull) S::unpack(ld_global_stream_v4(static_cast<const T *>(p.gate) + row + f * VEC), g);
                    if (p.gate_kind >= kGateChannel) {
#pragma unroll
                        for (int e = 0; e < VEC; ++e) b[e] *= g[e];
                    }
#pragma unroll
                    for (int e = 0; e < VEC; ++e) oh[k][e] = fmaf(s * gt, b[e], oh[k][e]);
                }
                float uu[VEC];
                S::unpack(uq[k], uu);
                load_weights<W, VEC>(w2, f * VEC, g);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    oh[k][e] *= ro;
                    colB[k][e] = fmaf(uu[e], oh[k][e], colB[k][e]);
                    D[k][e] = g[e] * uu[e];
                    acc = fmaf(D[k][e], oh[k][e], acc);
                }
            }
        }
        if (du) {
            const float c1 = row_sum(acc, wpt, grp, wl, lane, slots, turn) * inv_d;
#pragma unroll
            for (int k = 0; k < FR; ++k)
#pragma unroll
                for (int e = 0; e < VEC; ++e) D[k][e] = ro * fmaf(-c1, oh[k][e], D[k][e]);
        }
        if constexpr (!RES) {
#pragma unroll
            for (int k = 0; k < FR; ++k) {
                const int f = (k * wpt + wl) * 32 + lane;
                if (f < p.frags && dx) st_global_v4(dx + row + f * VEC, S::pack(D[k]));
            }
        } else {
            float S1 = 0.f;                              // sum of w g (m D) yh: the token gate's gradient and the norm's mean
#pragma unroll
            for (int k = 0; k < FR; ++k) {
                const int f = (k * wpt + wl) * 32 + lane;
                if (f >= p.frags) continue;
                float v[VEC];
                S::unpack(gq[k], v);
#pragma unroll
                for (int e = 0; e < VEC; ++e) D[k][e] += v[e];
                if (dx) st_global_v4(dx + row + f * VEC, S::pack(D[k]));
                if (p.drop.threshold) drop_fragment<VEC>(D[k], (unsigned long long)(row + f * VEC), p.drop, seed, offset);
                float yh[VEC], g[VEC];
                S::unpack(yq[k], yh);
#pragma unroll
                for (int e = 0; e < VEC; ++e) yh[e] *= ry;
                if (p.gate_kind == kGateChannel) {
                    load_weights<W, VEC>(static_cast<const W *>(p.gate), f * VEC, g);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        colA[k][e] = fmaf(D[k][e], yh[e], colA[k][e]);
                        D[k][e] *= g[e];
                    }
                } else if (p.gate_kind == kGateFull) {
                    float dg[VEC];
                    if (w) load_weights<W, VEC>(w, f * VEC, dg);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) dg[e] = s * ((w ? dg[e] : 1.f) * (D[k][e] * yh[e]));
                    if (p.dgate) st_global_v4(static_cast<T *>(p.dgate) + row + f * VEC, S::pack(dg));
                    S::unpack(ld_global_stream_v4(static_cast<const T *>(p.gate) + row + f * VEC), g);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        D[k][e] *= g[e];
                        colA[k][e] = fmaf(D[k][e], yh[e], colA[k][e]);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < VEC; ++e) colA[k][e] = fmaf(gt * D[k][e], yh[e], colA[k][e]);
                }
                if (w) {
                    load_weights<W, VEC>(w, f * VEC, g);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) D[k][e] *= g[e];
                }
#pragma unroll
                for (int e = 0; e < VEC; ++e) S1 = fmaf(D[k][e], yh[e], S1);
            }
            if (w || p.gate_kind == kGateToken) S1 = row_sum(S1, wpt, grp, wl, lane, slots, turn);
            if (p.gate_kind == kGateToken && p.dgate && wl == 0 && lane == 0) S::store1(static_cast<T *>(p.dgate) + tok, s * S1);
            if (dy) {
                const float sg = s * gt, c2 = w ? S1 * inv_d : 0.f;
#pragma unroll
                for (int k = 0; k < FR; ++k) {
                    const int f = (k * wpt + wl) * 32 + lane;
                    if (f >= p.frags) continue;
                    float yh[VEC];
                    S::unpack(yq[k], yh);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) D[k][e] = sg * (ry * fmaf(-c2, yh[e] * ry, D[k][e]));
                    st_global_v4(dy + row + f * VEC, S::pack(D[k]));
                }
            }
        }
    }
    if (!p.part) return;
    float *mine = p.part + (long long)blockIdx.x * 2 * p.d;
    if (groups == 1) {
#pragma unroll
        for (int k = 0; k < FR; ++k) {
            const int f = (k * wpt + wl) * 32 + lane;
            if (f >= p.frags) continue;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                if constexpr (RES) mine[f * VEC + e] = colA[k][e];
                mine[p.d + f * VEC + e] = colB[k][e];
            }
        }
        return;
    }
    for (int g = 0; g < groups; ++g) {                   // the CTA's rows in order: the sums do not depend on timing
        if (grp == g) {
#pragma unroll
            for (int k = 0; k < FR; ++k) {
                const int f = (k * wpt + wl) * 32 + lane;
                if (f >= p.frags) continue;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    if constexpr (RES) cols[f * VEC + e] = (g ? cols[f * VEC + e] : 0.f) + colA[k][e];
                    cols[p.d + f * VEC + e] = (g ? cols[p.d + f * VEC + e] : 0.f) + colB[k][e];
                }
            }
        }
        __syncthreads();
    }
    for (int c = threadIdx.x; c < p.d; c += kBlkThreads) {
        if constexpr (RES) mine[c] = cols[c];
        mine[p.d + c] = cols[p.d + c];
    }
}

// Column sums over the CTAs' rows, in fp64, and the parameters' gradients from them. 32 columns per CTA, 8 row strides.
// The residual scale's gradient needs all columns: the CTA that comes last adds the others' parts, in order.
template <typename W>
__global__ void __launch_bounds__(kBlkThreads) block_param_kernel(const BlockParams p, int rows) {
    __shared__ double sa[8][33], sb[8][33];
    __shared__ bool last;
    const int c = threadIdx.x & 31, r0 = threadIdx.x >> 5;
    const int col = blockIdx.x * 32 + c;
    double a = 0., b = 0.;
    if (col < p.d) {
        for (int r = r0; r < rows; r += 8) {
            const float *q = p.part + (long long)r * 2 * p.d;
            if (p.need_a) a += q[col];
            if (p.dw_next) b += q[p.d + col];
        }
    }
    sa[r0][c] = a;
    sb[r0][c] = b;
    __syncthreads();
    if (r0 == 0) {
        for (int i = 1; i < 8; ++i) {
            a += sa[i][c];
            b += sb[i][c];
        }
        double ds = 0.;
        if (col < p.d) {
            const float s = p.scale_dev ? *p.scale_dev : p.scale;
            const float w = p.w ? Store<W>::load1(static_cast<const W *>(p.w) + col) : 1.f;
            const float g = p.gate_kind == kGateChannel ? Store<W>::load1(static_cast<const W *>(p.gate) + col) : 1.f;
            if (p.dw) Store<W>::store1(static_cast<W *>(p.dw) + col, (float)(a * s * g));
            if (p.dgate && p.gate_kind == kGateChannel) Store<W>::store1(static_cast<W *>(p.dgate) + col, (float)(a * s * w));
            if (p.dw_next) Store<W>::store1(static_cast<W *>(p.dw_next) + col, (float)b);
            ds = a * w * g;
        }
        if (p.dscale) {
            for (int o = 16; o > 0; o >>= 1) ds += __shfl_xor_sync(0xffffffffu, ds, o);
            if (c == 0) p.ds_part[blockIdx.x] = ds;
        }
    }
    if (!p.dscale) return;
    if (threadIdx.x == 0) {
        __threadfence();
        last = atomicAdd(p.counter, 1u) == gridDim.x - 1;
        if (last) {
            __threadfence();
            double t = 0.;
            for (unsigned i = 0; i < gridDim.x; ++i) t += *reinterpret_cast<volatile double *>(p.ds_part + i);
            *p.dscale = (float)t;
        }
    }
}

// out = m x over n elements in row-major order: forward, and backward with the gradient as x
template <typename T>
__global__ void __launch_bounds__(256) dropout_kernel(const T *__restrict__ x, T *__restrict__ out, long long n, DropParams dp) {
    using S = Store<T>;
    constexpr int VEC = S::kVec;
    unsigned long long seed, offset;
    drop_state(dp, seed, offset);
    if (dp.rng_used && blockIdx.x == 0 && threadIdx.x == 0) {
        dp.rng_used[0] = (long long)seed;
        dp.rng_used[1] = (long long)offset;
    }
    const long long frags = n / VEC, stride = (long long)gridDim.x * blockDim.x;
    long long f = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    for (; f < frags; f += stride) {
        float v[VEC];
        S::unpack(ld_global_stream_v4(x + f * VEC), v);
        drop_fragment<VEC>(v, (unsigned long long)(f * VEC), dp, seed, offset);
        st_global_v4(out + f * VEC, S::pack(v));
    }
    if (f == frags && frags * VEC < n) {                 // the elements behind the last whole fragment: one thread
        float v[VEC];
        for (int e = 0; e < VEC; ++e) v[e] = frags * VEC + e < n ? S::load1(x + frags * VEC + e) : 0.f;
        drop_fragment<VEC>(v, (unsigned long long)(frags * VEC), dp, seed, offset);
        for (int e = 0; e < VEC; ++e)
            if (frags * VEC + e < n) S::store1(out + frags * VEC + e, v[e]);
    }
}

// ---------------------------------------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------------------------------------
// Fragments per lane and warps per row. Rows enough to fill the GPU: as few warps per row as hold it at `most` fragments per
// lane (no exchange between warps up to 32 * most fragments). Few rows (a decode step): more warps per row, since then the
// time is the latency of one row.
static bool block_shape(int frags, long long n_tok, int sms, int most, int *fr, int *wpt) {
    int w = 1;
    while (w < kBlkWarps && frags > w * 32 * most) w *= 2;
    while (w < kBlkWarps && frags > w * 32 && n_tok * w * 2 <= 8LL * sms) w *= 2;
    const int need = (frags + w * 32 - 1) / (w * 32);
    *fr = need;
    *wpt = w;
    return need <= 4;
}

template <typename T, typename W, bool RES>
static cudaError_t launch_block_t(BlockParams p, bool bwd, int sms, cudaStream_t stream) {
    int fr;
    if (!block_shape(p.frags, p.n_tok, sms, 4, &fr, &p.wpt)) return cudaErrorInvalidValue;
    const int groups = kBlkWarps / p.wpt;
    const long long need = (p.n_tok + groups - 1) / groups;
    const long long cap = bwd ? block_bwd_rows(sms) : 8LL * sms;
    const int grid = (int)(need < cap ? need : cap);
    const size_t smem = bwd && groups > 1 ? sizeof(float) * 2 * p.d : 0;
#define LB_BLK(FR_)                                                                                                  \
    case FR_:                                                                                                        \
        if (bwd) {                                                                                                   \
            if (smem > 48 * 1024) {                                                                                  \
                const cudaError_t e = cudaFuncSetAttribute(block_bwd_kernel<T, W, FR_, RES>,                         \
                                                           cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);  \
                if (e != cudaSuccess) return e;                                                                      \
            }                                                                                                        \
            block_bwd_kernel<T, W, FR_, RES><<<grid, kBlkThreads, smem, stream>>>(p);                                \
        } else block_fwd_kernel<T, W, FR_, RES><<<grid, kBlkThreads, 0, stream>>>(p);                                \
        break;
    switch (fr) {
        LB_BLK(1) LB_BLK(2) LB_BLK(3) LB_BLK(4)
    }
#undef LB_BLK
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess || !bwd || !p.part) return e;
    block_param_kernel<W><<<(p.d + 31) / 32, kBlkThreads, 0, stream>>>(p, grid);
    return cudaGetLastError();
}

int block_bwd_rows(int sms) { return 2 * sms < 304 ? 2 * sms : 304; }

cudaError_t launch_block(int dtype, int wdtype, bool residual, bool bwd, const BlockParams &p, int sms, cudaStream_t stream) {
    if (dtype == LB_DTYPE_F32)
        return residual ? launch_block_t<float, float, true>(p, bwd, sms, stream)
                        : launch_block_t<float, float, false>(p, bwd, sms, stream);
    if (wdtype == LB_DTYPE_F32)
        return residual ? launch_block_t<__nv_bfloat16, float, true>(p, bwd, sms, stream)
                        : launch_block_t<__nv_bfloat16, float, false>(p, bwd, sms, stream);
    return residual ? launch_block_t<__nv_bfloat16, __nv_bfloat16, true>(p, bwd, sms, stream)
                    : launch_block_t<__nv_bfloat16, __nv_bfloat16, false>(p, bwd, sms, stream);
}

cudaError_t launch_dropout(int dtype, const void *x, void *out, long long n, const DropParams &dp, int sms, cudaStream_t stream) {
    if (n == 0) return cudaSuccess;
    const int vec = dtype == LB_DTYPE_BF16 ? 8 : 4;
    const long long need = (n / vec + 1 + 255) / 256, cap = 16LL * sms;
    const int grid = (int)(need < cap ? need : cap);
    if (dtype == LB_DTYPE_BF16)
        dropout_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(static_cast<const __nv_bfloat16 *>(x),
                                                                static_cast<__nv_bfloat16 *>(out), n, dp);
    else
        dropout_kernel<float><<<grid, 256, 0, stream>>>(static_cast<const float *>(x), static_cast<float *>(out), n, dp);
    return cudaGetLastError();
}

}  // namespace lb
