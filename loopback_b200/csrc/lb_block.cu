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
// A row is handled by `wpt` warps (1, 2, 4 or 8 of the CTA's 8); a lane owns FR fragments of 16 bytes of every row, so the row
// is read once although its statistics are needed before its result. The rows to come are on their way into shared memory
// (cp.async, two rows ahead, each lane fetching the fragments it will read itself: no barrier); per-channel parameters lie
// there as fp32. All arithmetic is fp32, in pairs (fma.rn.f32x2), with one rounding at each store.
//
// Measured for 32768 x 1024 bf16: norm 21 us forward (134 MB, 0.97 of the copy rate) and 43 backward (201 MB; each row's exchange
// is what a warp waits for), residual with both norms 43 us forward (268 MB, 0.95; 48 with dropout) and 79 backward (403 MB, 0.78;
// 95 with dropout: its instructions, Philox's multiplies, masks, unpacking). With direct loads, two exchanges per row and every
// form decided at run time the four were 26, 57, 74 (with dropout) and 197.
#include "lb_common.cuh"
#include "lb_kernels.h"
#include "lb_launch.cuh"

namespace lb {

constexpr int kBlkThreads = 256;
constexpr int kBlkWarps = kBlkThreads / 32;

// ---------------------------------------------------------------------------------------------------------
// dropout's numbers: Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", 2011) with
// counter (group, offset) and key seed. A group is 8 consecutive elements; element j of it takes half j (low half first) of
// the four words, 16 bits: one call serves a 16-byte fragment of bf16, at half the integer work of a word per element.
// ---------------------------------------------------------------------------------------------------------
// The ten rounds' keys (seed + r times the two constants) come from where the kernel has room: added up as they are needed
// (integer pipe), kept in registers, or from shared memory (k0, k1 of round 0, 1, ..: 20 words, broadcast loads).
struct KeysAdded {
    uint32_t k0, k1;
    __device__ __forceinline__ uint2 at(int r) const { return make_uint2(k0 + r * 0x9E3779B9u, k1 + r * 0xBB67AE85u); }
};
struct KeysHeld {
    uint32_t k0[10], k1[10];
    __device__ __forceinline__ uint2 at(int r) const { return make_uint2(k0[r], k1[r]); }
};
struct KeysShared {
    uint32_t base;
    __device__ __forceinline__ uint2 at(int r) const {
        uint2 k;
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(k.x), "=r"(k.y) : "r"(base + r * 8));
        return k;
    }
};
template <typename Keys>
__device__ __forceinline__ uint4 philox4x32_10(unsigned long long group, unsigned long long offset, const Keys &keys) {
    uint32_t c0 = (uint32_t)group, c1 = (uint32_t)(group >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint2 k = keys.at(r);
        const unsigned long long a = (unsigned long long)c0 * 0xD2511F53u, b = (unsigned long long)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k.x;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k.y;
        c3 = (uint32_t)a;
    }
    return make_uint4(c0, c1, c2, c3);
}

// The words that decide over the fragment at linear index `e` (a multiple of 2 P), one per pair of elements
template <int P, typename Keys>
__device__ __forceinline__ void drop_words(uint32_t (&w)[P], unsigned long long e, const Keys &keys, unsigned long long offset) {
    const uint4 q = philox4x32_10(e >> 3, offset, keys);
    if constexpr (P == 4) {
        w[0] = q.x; w[1] = q.y; w[2] = q.z; w[3] = q.w;
    } else {
        const bool high = (e & 4) != 0;
        w[0] = high ? q.z : q.x; w[1] = high ? q.w : q.y;
    }
}
// clears what is dropped, whatever it held; the factor of what stays is applied elsewhere. The upper half is at least t
// where the word is at least t << 16, the lower one where the word shifted up is.
template <int P>
__device__ __forceinline__ void drop_pairs(float2 (&v)[P], const uint32_t (&w)[P], uint32_t threshold) {
    const uint32_t t = threshold << 16;
#pragma unroll
    for (int i = 0; i < P; ++i) {
        v[i].x = (w[i] << 16) >= t ? v[i].x : 0.f;
        v[i].y = w[i] >= t ? v[i].y : 0.f;
    }
}

// the pair in use, which also goes to rng_used
__device__ __forceinline__ void drop_state(const DropParams &dp, unsigned long long &seed, unsigned long long &offset) {
    seed = dp.rng ? (unsigned long long)dp.rng[0] : (unsigned long long)dp.seed;
    offset = dp.rng ? (unsigned long long)dp.rng[1] : (unsigned long long)dp.offset;
    if (dp.rng_used && blockIdx.x == 0 && threadIdx.x == 0) {
        dp.rng_used[0] = (long long)seed;
        dp.rng_used[1] = (long long)offset;
    }
}

__device__ __forceinline__ float2 splat(float v) { return make_float2(v, v); }

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Per-channel parameters in shared memory, fp32, in planes of 4 columns per fragment (a lane reads 16 bytes of each plane:
// no bank conflicts). dst[plane][frag][4] = a[c] * b[c], 1 where a pointer is null.
template <typename W, int VEC>
__device__ __forceinline__ void stage_channels(float *dst, const W *a, const W *b, int d, int frags) {
    for (int c = threadIdx.x; c < d; c += kBlkThreads) {
        const float v = (a ? Store<W>::load1(a + c) : 1.f) * (b ? Store<W>::load1(b + c) : 1.f);
        dst[(((c % VEC) >> 2) * frags + c / VEC) * 4 + (c & 3)] = v;
    }
}
template <int P>
__device__ __forceinline__ void channel_pairs(float2 (&v)[P], uint32_t base, uint32_t plane) {
#pragma unroll
    for (int i = 0; i < P / 2; ++i) {
        const float4 q = lds_f4(base + i * plane);
        v[2 * i] = make_float2(q.x, q.y);
        v[2 * i + 1] = make_float2(q.z, q.w);
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

__device__ __forceinline__ float3 row_sums(float3 v, int wpt, int grp, int wl, int lane, float (*slots)[3][kBlkWarps], int &turn) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
        v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
        v.z += __shfl_xor_sync(0xffffffffu, v.z, o);
    }
    if (wpt == 1) return v;
    float (*s)[kBlkWarps] = slots[turn];
    turn ^= 1;
    if (lane < 3) s[lane][grp * wpt + wl] = lane == 0 ? v.x : lane == 1 ? v.y : v.z;
    named_bar_sync(1 + grp, wpt * 32);
    float3 t = make_float3(0.f, 0.f, 0.f);
    for (int i = 0; i < wpt; ++i) {
        t.x += s[0][grp * wpt + i];
        t.y += s[1][grp * wpt + i];
        t.z += s[2][grp * wpt + i];
    }
    return t;
}

// Shared memory of both kernels: the ring [array][2 rows ahead][FR][thread] of 16 bytes, then the two channel tables; the
// backward's column sums take the ring's place at the end.
constexpr int kSlot = kBlkThreads * 16;
__host__ __device__ constexpr int ring_bytes(int arrays, int fr) { return 2 * arrays * fr * kSlot; }

// FORM 1: neither dropout nor a gate per element, known when compiled; 0: whatever the parameters say.
template <typename T, typename W, int FR, bool RES, int FORM>
__global__ void __launch_bounds__(kBlkThreads) block_fwd_kernel(const BlockParams p) {
    using S = Store<T>;
    constexpr int VEC = S::kVec, P = S::kPairs;
    __shared__ float slots[2][kBlkWarps];
    extern __shared__ __align__(16) uint8_t dyn[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int wpt = p.wpt, groups = kBlkWarps / wpt, grp = warp / wpt, wl = warp % wpt;
    const T *x = static_cast<const T *>(p.x), *y = static_cast<const T *>(p.y);
    const T *gate = FORM == 0 && p.gate_kind == kGateFull ? static_cast<const T *>(p.gate) : nullptr;
    const W *w = static_cast<const W *>(p.w), *w2 = static_cast<const W *>(p.w_next);
    T *out = static_cast<T *>(p.out), *u = static_cast<T *>(p.u);
    const int arrays = RES ? (gate ? 3 : 2) : 1;
    const int f0 = wl * FR * 32 + lane;                  // this lane's fragments: f0, f0 + 32, ..
    const long long own = (long long)f0 * VEC;
    const uint32_t ring = smem_u32(dyn) + threadIdx.x * 16;
    float *tab = reinterpret_cast<float *>(dyn + ring_bytes(arrays, FR));
    const uint32_t tab_wg = smem_u32(tab) + f0 * 16, tab_w2 = tab_wg + (RES ? p.frags * VEC * 4 : 0), plane = p.frags * 16;
    const auto slot = [&](int stage, int array, int k) { return ring + stage * (FR * kSlot) + (array * 2 * FR + k) * kSlot; };
    const auto fetch = [&](int stage, long long tok) {
        if (tok < p.n_tok) {
            const long long row = tok * p.d + own;           // this lane's first element of the row
#pragma unroll
            for (int k = 0; k < FR; ++k) {
                const int f = f0 + 32 * k;
                if (f < p.frags) {
                    cp_async16(slot(stage, 0, k), x + row + k * 32 * VEC);
                    if constexpr (RES) {
                        cp_async16(slot(stage, 1, k), y + row + k * 32 * VEC);
                        if (gate) cp_async16(slot(stage, 2, k), gate + row + k * 32 * VEC);
                    }
                }
            }
        }
        cp_async_commit();
    };
    const long long step = (long long)gridDim.x * groups;
    long long tok = (long long)blockIdx.x * groups + grp;
    grid_wait();
    grid_launch_dependents();
    fetch(0, tok);
    fetch(1, tok + step);
    if constexpr (RES) {
        stage_channels<W, VEC>(tab, w, p.gate_kind == kGateChannel ? static_cast<const W *>(p.gate) : nullptr, p.d, p.frags);
        if (w2) stage_channels<W, VEC>(tab + p.frags * VEC, w2, nullptr, p.d, p.frags);
    } else {
        stage_channels<W, VEC>(tab, w2, nullptr, p.d, p.frags);
    }
    const float s = RES ? (p.scale_dev ? *p.scale_dev : p.scale) * p.drop.keep_scale : 0.f;
    const float inv_d = 1.f / (float)p.d;
    const bool drop = RES && FORM == 0 && p.drop.threshold != 0;
    unsigned long long seed = 0, offset = 0;
    if (drop) drop_state(p.drop, seed, offset);
    const KeysAdded keys{(uint32_t)seed, (uint32_t)(seed >> 32)};
    __syncthreads();
    int turn = 0, stage = 0;
    for (; tok < p.n_tok; tok += step, stage ^= 1) {
        const long long row = tok * p.d + own;           // this lane's first element of the row
        cp_async_wait<1>();
        float2 o[FR][P];
        if constexpr (RES) {
            uint4 yq[FR];
            float ry = 1.f;
#pragma unroll
            for (int k = 0; k < FR; ++k) {
                const bool in = f0 + 32 * k < p.frags;
                yq[k] = in ? lds_v4(slot(stage, 1, k)) : make_uint4(0, 0, 0, 0);
            }
            if (w) {
                float2 ss = splat(0.f);
#pragma unroll
                for (int k = 0; k < FR; ++k) {
                    float2 v[P];
                    S::unpack2(yq[k], v);
#pragma unroll
                    for (int i = 0; i < P; ++i) ss = __ffma2_rn(v[i], v[i], ss);
                }
                ry = rsqrtf(row_sum(ss.x + ss.y, wpt, grp, wl, lane, slots, turn) * inv_d + p.eps);
                if (p.r_y && wl == 0 && lane == 0) p.r_y[tok] = ry;
            }
            const float gt = p.gate_kind == kGateToken ? S::load1(static_cast<const T *>(p.gate) + tok) : 1.f;
            const float2 sg = splat(s * gt), ry2 = splat(ry);
#pragma unroll
            for (int k = 0; k < FR; ++k) {
                const int f = f0 + 32 * k;
#pragma unroll
                for (int i = 0; i < P; ++i) o[k][i] = splat(0.f);
                if (f < p.frags) {
                    float2 b[P], c[P];
                    S::unpack2(yq[k], b);
                    channel_pairs<P>(c, tab_wg + k * 512, plane);
#pragma unroll
                    for (int i = 0; i < P; ++i) b[i] = __fmul2_rn(c[i], __fmul2_rn(b[i], ry2));
                    if (gate) {
                        S::unpack2(lds_v4(slot(stage, 2, k)), c);
#pragma unroll
                        for (int i = 0; i < P; ++i) b[i] = __fmul2_rn(b[i], c[i]);
                    }
                    if (drop) {
                        uint32_t words[P];
                        drop_words<P>(words, (unsigned long long)(row + k * 32 * VEC), keys, offset);
                        drop_pairs<P>(b, words, p.drop.threshold);
                    }
                    S::unpack2(lds_v4(slot(stage, 0, k)), o[k]);
#pragma unroll
                    for (int i = 0; i < P; ++i) o[k][i] = __ffma2_rn(sg, b[i], o[k][i]);
                    st_global_v4(out + row + k * 32 * VEC, S::pack2v(o[k]));
                }
            }
        } else {
#pragma unroll
            for (int k = 0; k < FR; ++k) {
                const bool in = f0 + 32 * k < p.frags;
                S::unpack2(in ? lds_v4(slot(stage, 0, k)) : make_uint4(0, 0, 0, 0), o[k]);
            }
        }
        fetch(stage, tok + 2 * step);
        if (RES && !w2) continue;
        float2 ss = splat(0.f);
#pragma unroll
        for (int k = 0; k < FR; ++k)
#pragma unroll
            for (int i = 0; i < P; ++i) ss = __ffma2_rn(o[k][i], o[k][i], ss);
        const float ro = rsqrtf(row_sum(ss.x + ss.y, wpt, grp, wl, lane, slots, turn) * inv_d + p.eps);
        if (p.r_o && wl == 0 && lane == 0) p.r_o[tok] = ro;
#pragma unroll
        for (int k = 0; k < FR; ++k) {
            const int f = f0 + 32 * k;
            if (f < p.frags) {
                float2 c[P];
                channel_pairs<P>(c, tab_w2 + k * 512, plane);
#pragma unroll
                for (int i = 0; i < P; ++i) c[i] = __fmul2_rn(c[i], __fmul2_rn(o[k][i], splat(ro)));
                st_global_v4(u + row + k * 32 * VEC, S::pack2v(c));
            }
        }
    }
}

// Per-CTA column sums leave through p.part[CTA][2][d] (A, then B); block_param_kernel adds the CTAs' rows in a fixed order.
// FORM 1 / 2: both upstream gradients, no gate per element, without / with dropout, known when compiled; 0: whatever the
// parameters say.
template <typename T, typename W, int FR, bool RES, int FORM>
__global__ void __launch_bounds__(kBlkThreads, FR <= 2 || !RES || (FR == 3 && sizeof(T) == 4) ? 2 : 1) block_bwd_kernel(const BlockParams p) {
    using S = Store<T>;
    constexpr int VEC = S::kVec, P = S::kPairs;
    __shared__ float slots[2][kBlkWarps], slots3[2][3][kBlkWarps];
    __shared__ __align__(16) uint32_t keys_[20];
    extern __shared__ __align__(16) uint8_t dyn[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int wpt = p.wpt, groups = kBlkWarps / wpt, grp = warp / wpt, wl = warp % wpt;
    const T *x = static_cast<const T *>(p.x), *y = static_cast<const T *>(p.y);
    const T *dout = static_cast<const T *>(p.d_out), *du = static_cast<const T *>(p.d_u);
    const T *gate = FORM == 0 && p.gate_kind == kGateFull ? static_cast<const T *>(p.gate) : nullptr;
    const W *w = static_cast<const W *>(p.w), *w2 = static_cast<const W *>(p.w_next);
    T *dx = static_cast<T *>(p.dx), *dy = static_cast<T *>(p.dy);
    const bool has_u = FORM != 0 || du != nullptr, has_out = FORM != 0 || dout != nullptr;
    // arrays of the ring: du, x, then y, dout, gate
    const int arrays = RES ? (gate ? 5 : 4) : 2;
    const int f0 = wl * FR * 32 + lane;                  // this lane's fragments: f0, f0 + 32, ..
    const long long own = (long long)f0 * VEC;
    const uint32_t ring = smem_u32(dyn) + threadIdx.x * 16;
    float *tab = reinterpret_cast<float *>(dyn + ring_bytes(arrays, FR));
    const uint32_t tab_wg = smem_u32(tab) + f0 * 16, tab_w2 = tab_wg + (RES ? p.frags * VEC * 4 : 0), plane = p.frags * 16;
    const auto slot = [&](int stage, int array, int k) { return ring + stage * (FR * kSlot) + (array * 2 * FR + k) * kSlot; };
    const auto fetch = [&](int stage, long long tok) {
        if (tok < p.n_tok) {
            const long long row = tok * p.d + own;           // this lane's first element of the row
#pragma unroll
            for (int k = 0; k < FR; ++k) {
                const int f = f0 + 32 * k;
                if (f < p.frags) {
                    if (has_u) {
                        cp_async16(slot(stage, 0, k), du + row + k * 32 * VEC);
                        cp_async16(slot(stage, 1, k), x + row + k * 32 * VEC);
                    }
                    if constexpr (RES) {
                        cp_async16(slot(stage, 2, k), y + row + k * 32 * VEC);
                        if (has_out) cp_async16(slot(stage, 3, k), dout + row + k * 32 * VEC);
                        if (gate) cp_async16(slot(stage, 4, k), gate + row + k * 32 * VEC);
                    }
                }
            }
        }
        cp_async_commit();
    };
    const long long step = (long long)gridDim.x * groups;
    long long tok = (long long)blockIdx.x * groups + grp;
    grid_wait();
    grid_launch_dependents();
    fetch(0, tok);
    fetch(1, tok + step);
    if constexpr (RES) {
        stage_channels<W, VEC>(tab, w, p.gate_kind == kGateChannel ? static_cast<const W *>(p.gate) : nullptr, p.d, p.frags);
        if (has_u) stage_channels<W, VEC>(tab + p.frags * VEC, w2, nullptr, p.d, p.frags);
    } else {
        stage_channels<W, VEC>(tab, w2, nullptr, p.d, p.frags);
    }
    const float s = RES ? (p.scale_dev ? *p.scale_dev : p.scale) * p.drop.keep_scale : 0.f;
    const float inv_d = 1.f / (float)p.d;
    const bool drop = RES && (FORM == 0 ? p.drop.threshold != 0 : FORM == 2);
    unsigned long long seed = 0, offset = 0;
    if (drop) drop_state(p.drop, seed, offset);
    const KeysAdded added{(uint32_t)seed, (uint32_t)(seed >> 32)};
    if (threadIdx.x < 10) {                              // registers are what this kernel is short of
        keys_[2 * threadIdx.x] = added.at(threadIdx.x).x;
        keys_[2 * threadIdx.x + 1] = added.at(threadIdx.x).y;
    }
    const KeysShared keys{smem_u32(keys_)};
    if (blockIdx.x == 0 && threadIdx.x == 0 && p.counter) *p.counter = 0;    // block_param_kernel counts its CTAs here
    float2 colA[RES ? FR : 1][P], colB[FR][P];
#pragma unroll
    for (int k = 0; k < FR; ++k)
#pragma unroll
        for (int i = 0; i < P; ++i) {
            colB[k][i] = splat(0.f);
            if constexpr (RES) colA[k][i] = splat(0.f);
        }
    __syncthreads();
    int turn = 0, stage = 0;
    for (; tok < p.n_tok; tok += step, stage ^= 1) {
        const long long row = tok * p.d + own;           // this lane's first element of the row
        const float ry = RES && w ? p.r_y[tok] : 1.f;
        const float ro = has_u ? p.r_o[tok] : 0.f;
        const float gt = RES && p.gate_kind == kGateToken ? S::load1(static_cast<const T *>(p.gate) + tok) : 1.f;
        const float2 ry2 = splat(ry), ro2 = splat(ro);
        cp_async_wait<1>();
        float2 D[FR][P], oh[FR][P];
        uint32_t words[RES ? FR : 1][P];
        // One exchange per row: with t = w' du and b = w g m yh, the sums of t oh, b (dout + r_o t) and b oh give both means,
        // mean(t oh) and the sum of b D that the norm after the block and the token gate's gradient want
        float2 s1 = splat(0.f), s2 = splat(0.f), s3 = splat(0.f);
#pragma unroll
        for (int k = 0; k < FR; ++k) {
            const bool in = f0 + 32 * k < p.frags;
#pragma unroll
            for (int i = 0; i < P; ++i) D[k][i] = oh[k][i] = splat(0.f);
            float2 b[P], c[P];
            if constexpr (RES) {
                if (in) {
                    S::unpack2(lds_v4(slot(stage, 2, k)), b);
                    channel_pairs<P>(c, tab_wg + k * 512, plane);
#pragma unroll
                    for (int i = 0; i < P; ++i) b[i] = __fmul2_rn(c[i], __fmul2_rn(b[i], ry2));
                    if (gate) {
                        S::unpack2(lds_v4(slot(stage, 4, k)), c);
#pragma unroll
                        for (int i = 0; i < P; ++i) b[i] = __fmul2_rn(b[i], c[i]);
                    }
                    if (drop) {
                        drop_words<P>(words[k], (unsigned long long)(row + k * 32 * VEC), keys, offset);
                        drop_pairs<P>(b, words[k], p.drop.threshold);
                    }
                    if (has_out) {
                        S::unpack2(lds_v4(slot(stage, 3, k)), c);
#pragma unroll
                        for (int i = 0; i < P; ++i) s2 = __ffma2_rn(b[i], c[i], s2);
                    }
                }
            }
            if (in && has_u) {
                float2 uu[P];
                S::unpack2(lds_v4(slot(stage, 1, k)), oh[k]);
                S::unpack2(lds_v4(slot(stage, 0, k)), uu);
                channel_pairs<P>(c, tab_w2 + k * 512, plane);
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    if constexpr (RES) oh[k][i] = __ffma2_rn(splat(s * gt), b[i], oh[k][i]);
                    oh[k][i] = __fmul2_rn(oh[k][i], ro2);
                    colB[k][i] = __ffma2_rn(uu[i], oh[k][i], colB[k][i]);
                    D[k][i] = __fmul2_rn(c[i], uu[i]);
                    s1 = __ffma2_rn(D[k][i], oh[k][i], s1);
                    if constexpr (RES) {
                        s2 = __ffma2_rn(b[i], __fmul2_rn(ro2, D[k][i]), s2);
                        s3 = __ffma2_rn(b[i], oh[k][i], s3);
                    }
                }
            }
        }
        if constexpr (!RES) {
            fetch(stage, tok + 2 * step);
            const float2 c1 = splat(-row_sum(s1.x + s1.y, wpt, grp, wl, lane, slots, turn) * inv_d);
#pragma unroll
            for (int k = 0; k < FR; ++k) {
                if (f0 + 32 * k >= p.frags || !dx) continue;
#pragma unroll
                for (int i = 0; i < P; ++i) D[k][i] = __fmul2_rn(ro2, __ffma2_rn(c1, oh[k][i], D[k][i]));
                st_global_v4(dx + row + k * 32 * VEC, S::pack2v(D[k]));
            }
        } else {
            float3 sums = row_sums(make_float3(s1.x + s1.y, s2.x + s2.y, s3.x + s3.y), wpt, grp, wl, lane, slots3, turn);
            const float mean = sums.x * inv_d, S1 = fmaf(-ro * mean, sums.z, sums.y);
            if (p.gate_kind == kGateToken && p.dgate && wl == 0 && lane == 0) S::store1(static_cast<T *>(p.dgate) + tok, s * S1);
            const float2 c1 = splat(-mean), k1 = splat(s * gt * ry), c2 = splat(-S1 * inv_d);
#pragma unroll
            for (int k = 0; k < FR; ++k) {
                if (f0 + 32 * k >= p.frags) continue;
                float2 v[P], yh[P];
                if (has_out) S::unpack2(lds_v4(slot(stage, 3, k)), v);
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    D[k][i] = __ffma2_rn(c1, oh[k][i], D[k][i]);
                    D[k][i] = has_out ? __ffma2_rn(ro2, D[k][i], v[i]) : __fmul2_rn(ro2, D[k][i]);
                }
                if (dx) st_global_v4(dx + row + k * 32 * VEC, S::pack2v(D[k]));
                if (drop) drop_pairs<P>(D[k], words[k], p.drop.threshold);
                S::unpack2(lds_v4(slot(stage, 2, k)), yh);
                if (drop && !w) drop_pairs<P>(yh, words[k], p.drop.threshold);      // what is dropped may be anything
#pragma unroll
                for (int i = 0; i < P; ++i) yh[i] = __fmul2_rn(yh[i], ry2);
                channel_pairs<P>(v, tab_wg + k * 512, plane);
                if (gate) {
                    float2 g[P];
                    if (p.dgate) {
#pragma unroll
                        for (int i = 0; i < P; ++i) g[i] = __fmul2_rn(splat(s), __fmul2_rn(v[i], __fmul2_rn(D[k][i], yh[i])));
                        st_global_v4(static_cast<T *>(p.dgate) + row + k * 32 * VEC, S::pack2v(g));
                    }
                    S::unpack2(lds_v4(slot(stage, 4, k)), g);
#pragma unroll
                    for (int i = 0; i < P; ++i) D[k][i] = __fmul2_rn(D[k][i], g[i]);
                    if (drop) drop_pairs<P>(D[k], words[k], p.drop.threshold);
                }
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    const float2 a = p.gate_kind == kGateToken ? __fmul2_rn(splat(gt), D[k][i]) : D[k][i];
                    colA[k][i] = __ffma2_rn(a, yh[i], colA[k][i]);
                    D[k][i] = __fmul2_rn(D[k][i], v[i]);
                }
                if (w) {                                 // without the norm dy does not depend on y, which may be infinite
#pragma unroll
                    for (int i = 0; i < P; ++i) D[k][i] = __ffma2_rn(c2, yh[i], D[k][i]);
                }
#pragma unroll
                for (int i = 0; i < P; ++i) D[k][i] = __fmul2_rn(k1, D[k][i]);
                if (dy) st_global_v4(dy + row + k * 32 * VEC, S::pack2v(D[k]));
            }
            fetch(stage, tok + 2 * step);
        }
    }
    if (!p.part) return;
    float *mine = p.part + (long long)blockIdx.x * 2 * p.d;
    float *cols = reinterpret_cast<float *>(dyn);        // [2][d]
    cp_async_wait<0>();
    __syncthreads();
    for (int g = 0; g < groups; ++g) {                   // the CTA's rows in order: the sums do not depend on timing
        if (grp == g) {
#pragma unroll
            for (int k = 0; k < FR; ++k) {
                const int f = f0 + 32 * k;
                if (f >= p.frags) continue;
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    const int c = f * VEC + 2 * i;
                    if constexpr (RES) {
                        cols[c] = (g ? cols[c] : 0.f) + colA[k][i].x;
                        cols[c + 1] = (g ? cols[c + 1] : 0.f) + colA[k][i].y;
                    }
                    cols[p.d + c] = (g ? cols[p.d + c] : 0.f) + colB[k][i].x;
                    cols[p.d + c + 1] = (g ? cols[p.d + c + 1] : 0.f) + colB[k][i].y;
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

// Column sums over the CTAs' rows, in fp64, and the parameters' gradients from them. 32 columns per CTA, 32 row strides.
// The residual scale's gradient needs all columns: the CTA that comes last adds the others' parts, in order.
template <typename W>
__global__ void __launch_bounds__(1024) block_param_kernel(const BlockParams p, int rows) {
    __shared__ double sa[32][33], sb[32][33];
    grid_wait();
    grid_launch_dependents();
    const int c = threadIdx.x & 31, r0 = threadIdx.x >> 5;
    const int col = blockIdx.x * 32 + c;
    double a = 0., b = 0.;
    if (col < p.d) {
        const float *q = p.part + (long long)r0 * 2 * p.d + col;
        for (int r = r0; r < rows; r += 128, q += 256LL * p.d) {             // four rows in flight
            float va[4], vb[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool in = r + 32 * i < rows;
                va[i] = in && p.need_a ? q[64LL * i * p.d] : 0.f;
                vb[i] = in && p.dw_next ? q[64LL * i * p.d + p.d] : 0.f;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                a += va[i];
                b += vb[i];
            }
        }
    }
    sa[r0][c] = a;
    sb[r0][c] = b;
    __syncthreads();
    if (r0 == 0) {
        for (int i = 1; i < 32; ++i) {
            a += sa[i][c];
            b += sb[i][c];
        }
        double ds = 0.;
        if (col < p.d) {
            const float s = (p.scale_dev ? *p.scale_dev : p.scale) * p.drop.keep_scale;
            const float w = p.w ? Store<W>::load1(static_cast<const W *>(p.w) + col) : 1.f;
            const float g = p.gate_kind == kGateChannel ? Store<W>::load1(static_cast<const W *>(p.gate) + col) : 1.f;
            if (p.dw) Store<W>::store1(static_cast<W *>(p.dw) + col, (float)(a * s * g));
            if (p.dgate && p.gate_kind == kGateChannel) Store<W>::store1(static_cast<W *>(p.dgate) + col, (float)(a * s * w));
            if (p.dw_next) Store<W>::store1(static_cast<W *>(p.dw_next) + col, (float)b);
            ds = a * w * g * p.drop.keep_scale;
        }
        if (p.dscale) {
            for (int o = 16; o > 0; o >>= 1) ds += __shfl_xor_sync(0xffffffffu, ds, o);
            if (c == 0) p.ds_part[blockIdx.x] = ds;
        }
    }
    if (!p.dscale) return;
    if (threadIdx.x == 0) {
        __threadfence();
        if (atomicAdd(p.counter, 1u) == gridDim.x - 1) {
            __threadfence();
            double t = 0.;
            for (unsigned i = 0; i < gridDim.x; ++i) t += *reinterpret_cast<volatile double *>(p.ds_part + i);
            *p.dscale = (float)t;
        }
    }
}

// out = m x over n elements in row-major order: forward, and backward with the gradient as x
template <typename T>
// (four CTAs per SM with two fragments in flight per thread: 25 us for 32768 x 1024 bf16; three with four 29)
__global__ void __launch_bounds__(256, 4) dropout_kernel(const T *__restrict__ x, T *__restrict__ out, long long n, DropParams dp) {
    using S = Store<T>;
    constexpr int VEC = S::kVec;
    grid_wait();
    grid_launch_dependents();
    unsigned long long seed, offset;
    drop_state(dp, seed, offset);
    const KeysAdded added{(uint32_t)seed, (uint32_t)(seed >> 32)};
    KeysHeld keys;
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        keys.k0[r] = added.at(r).x;
        keys.k1[r] = added.at(r).y;
        asm volatile("" : "+r"(keys.k0[r]), "+r"(keys.k1[r]));   // held, not added up again at every use
    }
    constexpr int P = S::kPairs;
    const long long frags = n / VEC, stride = (long long)gridDim.x * blockDim.x;
    const float2 scale = splat(dp.keep_scale);
    const auto masked = [&](const uint4 &q, long long f) {
        float2 v[P];
        uint32_t words[P];
        S::unpack2(q, v);
        drop_words<P>(words, (unsigned long long)(f * VEC), keys, offset);
#pragma unroll
        for (int i = 0; i < P; ++i) v[i] = __fmul2_rn(v[i], scale);
        drop_pairs<P>(v, words, dp.threshold);
        return S::pack2v(v);
    };
    long long f = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    for (; f + stride < frags; f += 2 * stride) {
        const uint4 q0 = ld_global_stream_v4(x + f * VEC), q1 = ld_global_stream_v4(x + (f + stride) * VEC);
        st_global_v4(out + f * VEC, masked(q0, f));
        st_global_v4(out + (f + stride) * VEC, masked(q1, f + stride));
    }
    for (; f < frags; f += stride) st_global_v4(out + f * VEC, masked(ld_global_stream_v4(x + f * VEC), f));
    if (f == frags && frags * VEC < n) {                 // the elements behind the last whole fragment: one thread
        uint32_t words[P];
        drop_words<P>(words, (unsigned long long)(frags * VEC), keys, offset);
        for (int e = 0; frags * VEC + e < n; ++e) {
            const uint32_t h = e & 1 ? words[e >> 1] >> 16 : words[e >> 1] & 0xffffu;
            S::store1(out + frags * VEC + e, h >= dp.threshold ? S::load1(x + frags * VEC + e) * dp.keep_scale : 0.f);
        }
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

// CTAs of 256 threads an SM holds, by registers (of 65,536, in units of 256 per warp) and shared memory
static int registers_of(void (*kernel)(const BlockParams)) {
    cudaFuncAttributes at;
    if (cudaFuncGetAttributes(&at, reinterpret_cast<const void *>(kernel)) == cudaSuccess) return at.numRegs;
    cudaGetLastError();
    return 255;
}
static int resident(int regs, size_t smem) {
    const int by_regs = 65536 / (kBlkWarps * ((regs * 32 + 255) / 256 * 256));
    const int by_smem = (int)((size_t)(228 * 1024) / (smem + 384 + 1024));
    const int n = by_regs < by_smem ? by_regs : by_smem;
    return n < 1 ? 1 : n > 8 ? 8 : n;
}

template <typename T, typename W, bool RES>
static cudaError_t launch_block_t(BlockParams p, bool bwd, int sms, cudaStream_t stream) {
    int fr;
    if (!block_shape(p.frags, p.n_tok, sms, p.most_frags ? p.most_frags : 4, &fr, &p.wpt)) return cudaErrorInvalidValue;
    if (bwd && RES && !p.most_frags && fr > 2) {
        // the residual's backward holds the most per fragment: two per lane let a second CTA onto the SM (32768 x 1024 bf16:
        // 95 us instead of 100; 16384 x 2048: 99 instead of 104), unless that leaves many lanes idle (1536 columns in threes)
        int fr2, wpt2;
        if (block_shape(p.frags, p.n_tok, sms, 2, &fr2, &wpt2) && fr2 * wpt2 * 10 <= fr * p.wpt * 12) {
            fr = fr2;
            p.wpt = wpt2;
        }
    }
    const int groups = kBlkWarps / p.wpt;
    const bool full = p.gate_kind == kGateFull;
    const int arrays = bwd ? (RES ? 4 + full : 2) : (RES ? 2 + full : 1);
    size_t smem = ring_bytes(arrays, fr) + sizeof(float) * (RES ? 2 : 1) * p.frags * Store<T>::kVec;
    if (bwd && smem < sizeof(float) * 2 * p.d) smem = sizeof(float) * 2 * p.d;
    const long long need = (p.n_tok + groups - 1) / groups;
    using Kernel = void (*)(const BlockParams);
    // the form (see the kernels) and its registers per thread, looked up once
    const int form = !RES ? 0 : bwd ? (full || !p.d_u || !p.d_out ? 0 : p.drop.threshold ? 2 : 1) : !full && !p.drop.threshold;
#define LB_BLK(FR_)                                                                                                  \
    case FR_: {                                                                                                      \
        static const Kernel kernels[5] = {block_fwd_kernel<T, W, FR_, RES, 0>, block_fwd_kernel<T, W, FR_, RES, RES ? 1 : 0>, \
                                          block_bwd_kernel<T, W, FR_, RES, 0>, block_bwd_kernel<T, W, FR_, RES, RES ? 1 : 0>, \
                                          block_bwd_kernel<T, W, FR_, RES, RES ? 2 : 0>};                            \
        static const int regs[5] = {registers_of(kernels[0]), registers_of(kernels[1]), registers_of(kernels[2]),    \
                                    registers_of(kernels[3]), registers_of(kernels[4])};                             \
        const int which = (bwd ? 2 : 0) + form;                                                                      \
        const Kernel kernel = kernels[which];                                                                        \
        if (smem > 40 * 1024) {                                                                                      \
            const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem); \
            if (e != cudaSuccess) return e;                                                                          \
        }                                                                                                            \
        long long cap = (long long)sms * resident(regs[which], smem);                                                \
        if (bwd && cap > block_bwd_rows(sms)) cap = block_bwd_rows(sms);                                             \
        grid = (int)(need < cap ? need : cap);                                                                       \
        err = launch_overlapped(kernel, dim3(grid), dim3(kBlkThreads), smem, stream, 1, p);                         \
        break;                                                                                                       \
    }
    int grid = 0;
    cudaError_t err = cudaSuccess;
    switch (fr) {
        LB_BLK(1) LB_BLK(2) LB_BLK(3) LB_BLK(4)
    }
#undef LB_BLK
    if (err != cudaSuccess || !bwd || !p.part) return err;
    return launch_overlapped(block_param_kernel<W>, dim3((p.d + 31) / 32), dim3(1024), 0, stream, 1, p, grid);
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
        return launch_overlapped(dropout_kernel<__nv_bfloat16>, dim3(grid), dim3(256), 0, stream, 1, static_cast<const __nv_bfloat16 *>(x),
                            static_cast<__nv_bfloat16 *>(out), n, dp);
    return launch_overlapped(dropout_kernel<float>, dim3(grid), dim3(256), 0, stream, 1, static_cast<const float *>(x),
                        static_cast<float *>(out), n, dp);
}

}  // namespace lb
