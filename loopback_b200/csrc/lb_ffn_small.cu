// The gated feed-forward block for few rows (a decode step, up to 64), bound by reading the weights once. At 128 rows the products
// of lb_gemm.cuh are as fast (2048 x 5632: 27.5 us both), at 64 slower (26.9 against 22.2; 1 row 30.7 against 18.1).
//
// Operands change places: a tile of 128 WEIGHT rows is the tensor core's A (M = 128), the tokens are its B (N = 16, 32 or 64), so
// every weight byte passes through shared memory once and the padding is on the small side. A cluster of CTAs shares a tile
// and splits k; their partial sums meet through distributed shared memory, in rank order, so the result does not depend on
// timing and no fp32 slice travels through memory. As many CTAs as fit two to an SM, each with its whole ring of TMA loads in
// flight: that is what keeps HBM busy (a decode step has no second tile to hide a first one's latency under).
//
//   projections  tile = 64 rows of Wg over 64 rows of Wu, k over d;  epilogue h = act(g) u
//   down         tile = 128 rows of Wd, k over f. Launched with programmatic stream serialisation: its CTAs take the SMs as
//                the projections' leave them and have their first weights in flight before h is there. (Measured and left out
//                for 1 x 2048 x 5632: asking for Wd into L2 from the projections' CTAs, which made those as much longer, 19.7 us
//                against 18.1; tiles of 64 rows of Wd, 19.3; shorter rings, so that both launches' CTAs are resident, 18.7 and
//                31 instead of 23 at 64 rows.)
#include "lb_gemm.cuh"

// 1 x 2048 x 5632: 69 MB in 18.1 us where the copy rate would take 10.6; the rest is the two launches' edges and the wait for h
// between them (4096 x 11008: 47.6 of 41.3).

namespace lb {

constexpr int kSmallThreads = 192;

template <int N, bool GATED>
__global__ void __launch_bounds__(kSmallThreads) ffn_small_kernel(const __grid_constant__ CUtensorMap map_w0, const __grid_constant__ CUtensorMap map_w1,
                                                                  const __grid_constant__ CUtensorMap map_x, const FfnSmallParams p) {
    constexpr int kA = 128 * 128, kStage = kA + N * 128;
    constexpr uint32_t kCols = N < 32 ? 32 : N;
    extern __shared__ uint8_t raw[];
    const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
    const int ST = p.stages;
    const uint32_t bars = base + ST * kStage;
    const uint32_t full = bars, empty = full + 8 * ST, done = empty + 8 * ST, mdone = done + 8, slot = mdone + 8, abort_flag = slot + 4;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = p.split > 1 ? cluster_rank() : 0;
    const int tile = blockIdx.x / p.split;
    WaitCtx wc{abort_flag, p.err_word, p.wait_cycles};
    const int kb0 = (int)((long long)p.kblocks * rank / p.split), kb1 = (int)((long long)p.kblocks * (rank + 1) / p.split);
    const int row0 = tile * (GATED ? 64 : 128);
    const int ahead = kb1 - kb0 < ST ? kb1 - kb0 : ST;
    const auto weights = [&](int s, int kb) {
        const uint32_t sa = base + s * kStage, bar = full + 8 * s;
        mbar_arrive_expect_tx(bar, kStage);
        if (p.test_skip_item != 0 && blockIdx.x == 0 && kb + 1 == p.test_skip_item) return;      // test hook: never comes
        tma_load_2d(sa, &map_w0, bar, kb * kGemmK, row0);
        if constexpr (GATED) tma_load_2d(sa + kA / 2, &map_w1, bar, kb * kGemmK, row0);
    };
    const auto tokens = [&](int s, int kb) { tma_load_2d(base + s * kStage + kA, &map_x, full + 8 * s, kb * kGemmK, 0); };
    if (threadIdx.x == 0) {
        for (int i = 0; i < ST; ++i) {
            mbar_init(full + 8 * i, 1);
            mbar_init(empty + 8 * i, 1);
        }
        mbar_init(done, 1);
        mbar_init(mdone, 1);
        sts_s32(abort_flag, 0);
        fence_mbar_init();
        if (GATED) grid_wait();
        for (int i = 0; i < ahead; ++i) weights(i, kb0 + i);     // before anything else of the CTA is ready
    }
    __syncwarp();
    if (warp == 1) tmem_alloc<1>(slot, kCols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = (uint32_t)lds_volatile_s32(slot);
    if (warp == 0) {
        if (lane == 0) {
            if constexpr (GATED) grid_launch_dependents();
            else grid_wait();                            // h is complete
            for (int i = 0; i < ahead; ++i) tokens(i, kb0 + i);
            int s = 0;
            uint32_t ph = 1;
            bool ok = true;
            int issued = ahead;
            for (int kb = kb0 + ahead; kb < kb1; ++kb) {
                if (!(ok = mbar_wait(empty + 8 * s, ph ^ 1, wc, kDevWaitEmpty))) break;
                weights(s, kb);
                tokens(s, kb);
                ++issued;
                if (++s == ST) { s = 0; ph ^= 1; }
            }
            // every copy has landed before this CTA's shared memory is used again or goes away
            for (int i = issued > ST ? issued - ST : 0; i < issued; ++i) {
                const long long t0 = clock64();
                while (!mbar_try_wait(full + 8 * (i % ST), (uint32_t)(i / ST) & 1) && clock64() - t0 < p.wait_cycles) {}
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t idesc = mma_idesc(128, N, false, false);
            int s = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!(ok = mbar_wait(full + 8 * s, ph, wc, kDevWaitFull))) break;
                tc_fence_after();
                const uint32_t sa = base + s * kStage;
                const uint64_t da = tile_desc(sa, false, 0), db = tile_desc(sa + kA, false, 0);
#pragma unroll
                for (int k = 0; k < kGemmK / 16; ++k) tc_mma<1>(tmem, da + 2 * k, db + 2 * k, idesc, kb > kb0 || k > 0);
                tc_commit<1>(empty + 8 * s);
                if (++s == ST) { s = 0; ph ^= 1; }
            }
            if (ok) tc_commit<1>(done);
            tc_drain<1>(mdone, p.wait_cycles);
        }
    } else if (warp_wait(done, 0, wc, kDevWaitTmem)) {
        // this CTA's sums, [token][128 weight rows] fp32, over the ring (all its tiles have been read)
        tc_fence_after();
        const int quad = warp & 3;
        constexpr int W = N < 32 ? N : 32;
#pragma unroll 1
        for (int c = 0; c < N; c += 32) {
            float v[32];
            tmem_ld32(tmem + ((uint32_t)(quad * 32) << 16) + c, v);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < W; ++i) sts_f32(base + (uint32_t)(((c + i) * 128 + quad * 32 + lane) * 4), v[i]);
        }
        tc_fence_before();
    }
    __syncwarp();
    if (p.split > 1) cluster_sync();
    else __syncthreads();
    // the ranks share the tile's tokens: a warp sums one token's row over the CTAs, in rank order
    for (int t = (int)rank + p.split * warp; t < p.n_tok; t += p.split * (kSmallThreads / 32)) {
        const uint32_t from = base + t * 512 + (GATED ? lane * 8 : lane * 16);
        float v[8][4];
#pragma unroll
        for (int r = 0; r < 8; ++r) {                    // every CTA's at once: one round trip instead of one per CTA
            if (r >= p.split) break;
            const uint32_t src = p.split > 1 ? map_rank(from, r) : from;
            if constexpr (GATED) {
                asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v[r][0]), "=f"(v[r][1]) : "r"(src));
                asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v[r][2]), "=f"(v[r][3]) : "r"(src + 256));
            } else {
                asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                             : "=f"(v[r][0]), "=f"(v[r][1]), "=f"(v[r][2]), "=f"(v[r][3]) : "r"(src));
            }
        }
        float a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int r = 0; r < 8; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) a[i] += r < p.split ? v[r][i] : 0.f;
        __nv_bfloat16 *out = static_cast<__nv_bfloat16 *>(p.out) + (long long)t * p.n;
        using B = Store<__nv_bfloat16>;
        if constexpr (GATED) {
            const int col = row0 + 2 * lane;
            float g0, g1, slope;
            if (p.act == LB_ACT_SILU) {
                act_both<LB_ACT_SILU>(a[0], g0, slope);
                act_both<LB_ACT_SILU>(a[1], g1, slope);
            } else {
                act_both<LB_ACT_GELU>(a[0], g0, slope);
                act_both<LB_ACT_GELU>(a[1], g1, slope);
            }
            if (col < p.n) *reinterpret_cast<uint32_t *>(out + col) = B::pack2(g0 * a[2], g1 * a[3]);
        } else {
            const int col = row0 + 4 * lane;
            if (col < p.n) *reinterpret_cast<uint2 *>(out + col) = make_uint2(B::pack2(a[0], a[1]), B::pack2(a[2], a[3]));
        }
    }
    __syncwarp();
    tc_fence_before();
    if (p.split > 1) cluster_sync();                     // nobody leaves while its sums are read
    else __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_free<1>(tmem, kCols);
}

int ffn_small_rows(long long n_tok) { return n_tok <= 16 ? 16 : n_tok <= 32 ? 32 : 64; }

template <int N, bool GATED>
static cudaError_t launch_small_t(const CUtensorMap &w0, const CUtensorMap &w1, const CUtensorMap &x, FfnSmallParams p, int sms,
                                  cudaStream_t stream) {
    constexpr int kStage = 128 * 128 + N * 128;
    const int tiles = (p.n + (GATED ? 63 : 127)) / (GATED ? 64 : 128);
    // k split over as many CTAs of a cluster as leave two CTAs per SM (8 at most, two blocks of k each at least)
    int split = 2 * sms / tiles;
    if (split > 8) split = 8;
    if (split > p.kblocks / 2) split = p.kblocks / 2;
    if (split < 1) split = 1;
    p.split = split;
    const int per = (p.kblocks + split - 1) / split;
    // Half an SM's shared memory, also where there are fewer CTAs than SMs: clusters of CTAs that each want a whole SM do not
    // all find room in the GPCs at once (2048 x 5632: 16 clusters of 8 took two rounds, 15 us instead of 7).
    constexpr int kExtra = 1024 + 256, kRing = (113 * 1024 - kExtra) / kStage * kStage;
    static_assert(kRing >= N * 512 && kRing >= 2 * kStage, "the partial sums lie over the ring");
    p.stages = kRing / kStage < per ? kRing / kStage : per;
    while (p.stages * kStage < N * 512) ++p.stages;
    const size_t smem = kExtra + (size_t)p.stages * kStage;
    auto kernel = ffn_small_kernel<N, GATED>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kGemmMaxSmem);
    if (e != cudaSuccess) return e;
    return launch_overlapped(kernel, dim3((unsigned)(tiles * split)), dim3(kSmallThreads), smem, stream, split, w0, w1, x, p);
}

cudaError_t launch_ffn_small(bool gated, int rows, const CUtensorMap &w0, const CUtensorMap &w1, const CUtensorMap &x,
                             const FfnSmallParams &p, int sms, cudaStream_t stream) {
#define LB_SMALL(N_) \
    case N_: return gated ? launch_small_t<N_, true>(w0, w1, x, p, sms, stream) : launch_small_t<N_, false>(w0, w1, x, p, sms, stream);
    switch (rows) {
        LB_SMALL(16) LB_SMALL(32) LB_SMALL(64)
    }
#undef LB_SMALL
    return cudaErrorInvalidValue;
}

}  // namespace lb
