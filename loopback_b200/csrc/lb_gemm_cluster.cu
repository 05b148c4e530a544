// A product split along k over the CTAs of a cluster, for results of few tiles: one tile of 128 x 128 per cluster, each CTA sums
// its range of k in TMEM, and the partial tiles meet through distributed shared memory, in rank order. Against slices through
// memory (kEpiPartial and gemm_sum_kernel) that saves a launch and the slices' way out and in. Two CTAs to an SM, with three
// stages each, hide one another's latencies. The gated block on 1021 x 768 x 2048 takes 20.9 us so and 22.0 with slices, on
// 512 x 2048 x 5632 45.7 and 48.1, a training step on 512 x 768 x 2048 88 and 104; from a round of tiles on the slices win
// (2048 x 1024 x 2816: 39.6 against 44.7). What bounds it is L2 on the way in: a 128 x 128 tile reads twice what a 256-row one does.
#include "lb_gemm.cuh"

namespace lb {

constexpr int kClusterThreads = 320;
constexpr int kClusterStage = 2 * 128 * 128;

template <bool A_MN, bool B_MN>
__global__ void __launch_bounds__(kClusterThreads) gemm_cluster_kernel(const __grid_constant__ GemmMaps maps, const GemmParams p, const int stages,
                                                                       __nv_bfloat16 *__restrict__ out) {
    extern __shared__ uint8_t raw[];
    const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
    const uint32_t bars = base + stages * kClusterStage;
    const uint32_t full = bars, empty = full + 8 * stages, done = empty + 8 * stages, mdone = done + 8, slot = mdone + 8, abort_flag = slot + 4;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const TileAt at = tile_at(blockIdx.x / p.splits, p);
    const int m0 = at.m * kGemmM, n0 = at.n * 128;
    const int blocks = p.kblocks * p.segs;
    const int kb0 = (int)((long long)blocks * rank / p.splits), kb1 = (int)((long long)blocks * (rank + 1) / p.splits);
    WaitCtx wc{abort_flag, p.err_word, p.wait_cycles};
    if (threadIdx.x == 0) {
        for (int i = 0; i < stages; ++i) {
            mbar_init(full + 8 * i, 1);
            mbar_init(empty + 8 * i, 1);
        }
        mbar_init(done, 1);
        mbar_init(mdone, 1);
        sts_s32(abort_flag, 0);
        fence_mbar_init();
    }
    __syncwarp();
    if (warp == 1) tmem_alloc<1>(slot, 128);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = (uint32_t)lds_volatile_s32(slot);
    grid_wait();
    grid_launch_dependents();

    if (warp == 0) {
        if (lane == 0) {
            int s = 0, issued = 0;
            uint32_t ph = 0;
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!mbar_wait(empty + 8 * s, ph ^ 1, wc, kDevWaitEmpty)) break;
                const int half = kb >= p.kblocks, k0 = (kb - half * p.kblocks) * kGemmK;
                const uint32_t sa = base + s * kClusterStage, sb = sa + kClusterStage / 2, bar = full + 8 * s;
                mbar_arrive_expect_tx(bar, kClusterStage);
                ++issued;
                if (p.test_skip_item != 0 && blockIdx.x == 0 && issued == p.test_skip_item) {
                    // test hook: this copy never comes
                } else if constexpr (!A_MN) {
                    tma_load_2d(sa, &maps.a[half], bar, k0, m0);
                } else {
                    tma_load_2d(sa, &maps.a[half], bar, m0, k0);
                    tma_load_2d(sa + 8192, &maps.a[half], bar, m0 + 64, k0);
                }
                if constexpr (!B_MN) {
                    tma_load_2d(sb, &maps.b[half], bar, k0, n0);
                } else {
                    tma_load_2d(sb, &maps.b[half], bar, n0, k0);
                    tma_load_2d(sb + 8192, &maps.b[half], bar, n0 + 64, k0);
                }
                if (++s == stages) { s = 0; ph ^= 1; }
            }
            // every copy has landed before this CTA's shared memory is used again or goes away
            for (int i = issued > stages ? issued - stages : 0; i < issued; ++i) {
                const long long t0 = clock64();
                while (!mbar_try_wait(full + 8 * (i % stages), (uint32_t)(i / stages) & 1) && clock64() - t0 < p.wait_cycles) {}
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t idesc = mma_idesc(128, 128, A_MN, B_MN);
            constexpr uint32_t ka = A_MN ? 2048 >> 4 : 32 >> 4, kb_ = B_MN ? 2048 >> 4 : 32 >> 4;
            int s = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!(ok = mbar_wait(full + 8 * s, ph, wc, kDevWaitFull))) break;
                tc_fence_after();
                const uint32_t sa = base + s * kClusterStage;
                const uint64_t da = tile_desc(sa, A_MN, 8192), db = tile_desc(sa + kClusterStage / 2, B_MN, 8192);
#pragma unroll
                for (int k = 0; k < kGemmK / 16; ++k) tc_mma<1>(tmem, da + k * ka, db + k * kb_, idesc, kb > kb0 || k > 0);
                tc_commit<1>(empty + 8 * s);
                if (++s == stages) { s = 0; ph ^= 1; }
            }
            if (ok) tc_commit<1>(done);
            tc_drain<1>(mdone, p.wait_cycles);
        }
    } else if (warp < 6 && warp_wait(done, 0, wc, kDevWaitTmem)) {
        // this CTA's sums over the ring, [column][128 rows] fp32: lanes are rows, no bank conflicts
        tc_fence_after();
        const int quad = warp & 3;
#pragma unroll 1
        for (int c = 0; c < 128; c += 32) {
            float v[32];
            tmem_ld32(tmem + ((uint32_t)(quad * 32) << 16) + c, v);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) sts_f32(base + (uint32_t)(((c + i) * 128 + quad * 32 + lane) * 4), v[i]);
        }
        tc_fence_before();
    }
    __syncwarp();
    cluster_sync();
    // 16 groups of 8 columns go round the ranks, 4 blocks of 32 rows of each round the warps; a lane has a row of a group and asks
    // every CTA for its part at once (one round trip per group, not one per CTA)
    for (int i = warp >> 2; warp < 8 && (int)rank + i * p.splits < 16; i += 2) {
        const int group = (int)rank + i * p.splits, row = (warp & 3) * 32 + lane;
        float v[kClusterSplits][8];
#pragma unroll
        for (int r = 0; r < kClusterSplits; ++r) {
            if (r >= p.splits) break;
            const uint32_t src = map_rank(base + (uint32_t)((group * 8 * 128 + row) * 4), r);
#pragma unroll
            for (int c = 0; c < 8; ++c) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v[r][c]) : "r"(src + c * 512));
        }
        float sum[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            sum[c] = v[0][c];
#pragma unroll
            for (int r = 1; r < kClusterSplits; ++r) sum[c] += r < p.splits ? v[r][c] : 0.f;
        }
        const int col = n0 + group * 8;
        if (m0 + row < p.m && col < p.n) st_global_v4(out + (long long)(m0 + row) * p.n + col, Store<__nv_bfloat16>::pack(sum));
    }
    __syncwarp();
    tc_fence_before();
    cluster_sync();                                      // nobody leaves while its sums are read
    tc_fence_after();
    if (warp == 1) tmem_free<1>(tmem, 128);
}

cudaError_t launch_gemm_cluster(int form, const GemmMaps &maps, const GemmParams &p, void *out, cudaStream_t stream) {
    const int per = (p.kblocks * p.segs + p.splits - 1) / p.splits;
    const int stages = per < 3 ? (per < 2 ? 2 : per) : 3;          // the partial tile (64 KB) lies over two of them
    const size_t smem = 1024 + (size_t)stages * kClusterStage + 256;
    const dim3 grid((unsigned)(p.m_tiles * p.n_tiles * p.splits));
    const auto go = [&](auto kernel) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
        return launch_overlapped(kernel, grid, dim3(kClusterThreads), smem, stream, p.splits, maps, p, stages, static_cast<__nv_bfloat16 *>(out));
    };
    switch (form) {
        case kFormKK: return go(gemm_cluster_kernel<false, false>);
        case kFormKN: return go(gemm_cluster_kernel<false, true>);
        case kFormMN: return go(gemm_cluster_kernel<true, true>);
    }
    return cudaErrorInvalidValue;
}

}  // namespace lb
