// The matrix products of the gated feed-forward block on sm_100a's tensor cores: tcgen05.mma with TMEM accumulators, operands
// staged by TMA, one persistent warp-specialised kernel with several epilogues.
//
//   C[m][n] = sum_k A(m, k) B(n, k)      bf16 operands, fp32 accumulation over all of k, one rounding in the epilogue
//
// Either operand may lie in memory with k contiguous (K-major: x, weights in a projection, ...) or with m / n contiguous
// (MN-major: weights in a gradient of the input, activations in a gradient of the weights): the tensor core reads both from
// 128-byte-swizzled tiles, so nothing is ever transposed in memory.
//
// A tile is 128 rows per CTA (CG = 2: 256 rows over a pair of CTAs, each of which holds half of B's tile and so stages half
// as much per multiply) by BN columns. Warp 0 issues the TMA loads into a ring of stages, warp 1 the multiplies, the others
// empty the accumulators; two accumulators in TMEM let the epilogue of one tile run under the multiplies of the next. The pair's
// tile of 512 columns (two multiplies side by side) has one accumulator, all of TMEM, and reads a quarter less per multiply:
// alone it is as fast (2816 x 1024 weight gradients 83 us against 86), but a training pass in a row, at the power cap, gains
// 3-4 % (8192 x 1024 x 2816: 397 -> 383 us, 16411 x 1536 x 4096: 1561 -> 1503). Where the tiles no longer fill the GPU it
// loses (2048 x 1024 x 2816: 162 against 128).
//
// What bounds it, for 8192 rows of 1024 with 2816 hidden columns: the pair's tile needs 64 bytes per clock and SM from L2, which
// serves the launch at 10-14 TB/s, and the power cap; 1.58 PFLOP/s for the input's gradient, 1.70 for both weight gradients,
// 1.34 down (one round of 64 tiles on 74 pairs), 1.28 for the gated projections without and 1.14 with the kept factors (whose 138 MB of writes share L2 with the
// operands; without any epilogue, in a copy made for the measurement, 1.46-1.69). The single CTA's 128 x 256 tile reached 1.23
// for the input's gradient, 128 x 128 0.81.
#pragma once

#include "lb_common.cuh"
#include "lb_kernels.h"
#include "lb_launch.cuh"

namespace lb {

constexpr int kGemmK = 64;                         // k per stage: one 128-byte swizzle row of bf16
constexpr int kGemmM = 128;                        // rows per CTA
constexpr int kGemmMaxSmem = 227 * 1024;

template <int CG, int BN, int EPI>
struct GemmShape {
    static constexpr bool kGated = EPI == kEpiGate || EPI == kEpiGateBwd;
    // the gated epilogues do more per element than one tile's multiplies leave time for with 4 or 8 warps
    static constexpr int kEpiWarps = kGated ? BN / 16 : 4;
    static constexpr int kThreads = 64 + 32 * kEpiWarps;
    static constexpr int kABytes = kGemmM * 128;
    // a tile of 512 columns is two multiplies side by side; its accumulator takes all of TMEM
    static constexpr int kParts = BN > 256 ? BN / 256 : 1, kAccs = BN > 256 ? 1 : 2;
    static constexpr int kPartRows = BN / kParts / CG;               // of B's tile in this CTA, per part
    static constexpr int kBRows = kParts * kPartRows;
    static constexpr int kStageBytes = kABytes + kBRows * 128;
    static constexpr int kBuf = kGated ? 2048 : 4096;                // result box of a warp, two of them
    static constexpr int kStaging = kEpiWarps * 2 * kBuf;
    static constexpr int kTail = 1024 + 512;                         // alignment, barriers
    static constexpr int kFit = (kGemmMaxSmem - kTail - kStaging) / kStageBytes;
    static constexpr int kStages = kFit < 8 ? kFit : 8;
    static constexpr int kSmem = kTail + kStaging + kStages * kStageBytes;
    static constexpr int kCols = kAccs * BN;                         // TMEM columns (a power of two)
    static_assert(kStages >= 2 && kCols >= 32 && kCols <= 512 && (BN & (BN - 1)) == 0 && (kParts == 1 || EPI == kEpiStore), "tile does not fit");
};

// ---------------------------------------------------------------------------------------------------------
// PTX wrappers
// ---------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// tile load; with CG = 2 the completion is counted on a barrier of the pair's first CTA
template <int CG>
__device__ __forceinline__ void tma_tile(uint32_t dst, const CUtensorMap *map, uint32_t bar, int c0, int c1) {
    if constexpr (CG == 1) {
        tma_load_2d(dst, map, bar, c0, c1);
    } else {
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
            ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
            : "memory");
    }
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap *map, uint32_t src, int c0, int c1) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];"
                 ::"l"(reinterpret_cast<uint64_t>(map)), "r"(src), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ void tma_store_3d(const CUtensorMap *map, uint32_t src, int c0, int c1, int c2) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];"
                 ::"l"(reinterpret_cast<uint64_t>(map)), "r"(src), "r"(c0), "r"(c1), "r"(c2) : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

template <int CG> __device__ __forceinline__ void tmem_alloc(uint32_t slot, uint32_t cols) {
    if constexpr (CG == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
}
template <int CG> __device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t cols) {
    if constexpr (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

template <int CG>
__device__ __forceinline__ void tc_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    if constexpr (CG == 1)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add) : "memory");
}
// arrives on `bar` (CG = 2: on both CTAs' barrier at that offset) when the multiplies issued so far are done
template <int CG> __device__ __forceinline__ void tc_commit(uint32_t bar) {
    if constexpr (CG == 1)
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                     ::"r"(bar), "h"((uint16_t)3) : "memory");
}
// Waits, with a limit, until every multiply issued has been done: shared memory and TMEM may not go away under one, whoever
// gave up a wait before.
template <int CG> __device__ __forceinline__ void tc_drain(uint32_t bar, long long limit) {
    tc_commit<CG>(bar);
    const long long t0 = clock64();
    while (!mbar_try_wait(bar, 0) && clock64() - t0 < limit) {}
}
// 32 accumulator columns of this thread's row
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float (&v)[32]) {
    uint32_t *r = reinterpret_cast<uint32_t *>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
          "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
          "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, float (&v)[16]) {
    uint32_t *r = reinterpret_cast<uint32_t *>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void sts_v4(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

// Shared-memory operand descriptor of a 128-byte-swizzled tile at `addr` (PTX ISA, tcgen05 matrix descriptors): address and
// strides in units of 16 bytes, version 1, layout 2. Groups of 8 swizzle rows lie 1024 bytes apart. K-major: rows are m / n,
// the second stride is not used; MN-major: rows are k, `block` bytes lead to the next 64 columns of m / n.
__device__ __forceinline__ uint64_t tile_desc(uint32_t addr, bool mn_major, uint32_t block) {
    const uint64_t lead = mn_major ? block >> 4 : 1;
    return (uint64_t)((addr & 0x3ffff) >> 4) | lead << 16 | (uint64_t)(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
}

// Instruction descriptor of kind::f16: fp32 accumulator, bf16 operands, their majorness, n / 8, m / 16
constexpr uint32_t mma_idesc(int m, int n, bool a_mn, bool b_mn) {
    return 1u << 4 | 1u << 7 | 1u << 10 | (a_mn ? 1u << 15 : 0) | (b_mn ? 1u << 16 : 0) | (uint32_t)(n >> 3) << 17 | (uint32_t)(m >> 4) << 24;
}

// a wait of a whole warp: all lanes go on or none
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, const WaitCtx &wc, int what) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, wc, what));
}

// act(g) and act'(g). The activation is a template parameter: as a run-time choice it put a branch behind every element of the
// epilogue (106 us instead of 83 for 8192 x 1024 -> 2 x 2816 with the factors kept).
template <int ACT>
__device__ __forceinline__ void act_both(float g, float &a, float &slope) {
    if constexpr (ACT == LB_ACT_SILU) {
        const float s = __fdividef(1.f, 1.f + __expf(-g));
        a = g * s;
        slope = s * fmaf(g, 1.f - s, 1.f);
    } else {
        const float cdf = 0.5f * (1.f + erff(g * 0.70710678118654752f));
        a = g * cdf;
        slope = fmaf(g * 0.39894228040143268f, __expf(-0.5f * g * g), cdf);
    }
}

// What the backward keeps of a row's 32 columns: act'(g) u and act(g), each cut to the upper 24 bits of its fp32 (16 bits of
// mantissa and fp32's range; in bf16 these two would be the largest error of every gradient). The buffer is laid out as the
// threads hold the values, in blocks of 32 rows x 32 columns: 12 pieces of 512 bytes, 16 per lane (= row), so both directions
// are whole-line accesses without a detour through shared memory. Pieces 0-3 / 4-7: the upper halves of the two values,
// 8-9 / 10-11: the third bytes. A step of 16 columns is two pieces of upper halves and one of third bytes for each value.
constexpr int kKeptBlock = 12 * 512;
__device__ __forceinline__ void pack_kept(const float (&v)[16], uint4 &h0, uint4 &h1, uint4 &low) {
    uint32_t l[4], h[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t a = __byte_perm(__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]), 0x0051);
        const uint32_t b = __byte_perm(__float_as_uint(v[4 * i + 2]), __float_as_uint(v[4 * i + 3]), 0x0051);
        l[i] = __byte_perm(a, b, 0x5410);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = __byte_perm(__float_as_uint(v[2 * i]), __float_as_uint(v[2 * i + 1]), 0x7632);
    h0 = make_uint4(h[0], h[1], h[2], h[3]);
    h1 = make_uint4(h[4], h[5], h[6], h[7]);
    low = make_uint4(l[0], l[1], l[2], l[3]);
}
// 8 values from their upper halves and third bytes; the lowest byte repeats the third (it was cut off)
__device__ __forceinline__ void kept_values(const uint4 &h, uint32_t l0, uint32_t l1, float (&v)[8]) {
    v[0] = __uint_as_float(__byte_perm(h.x, l0, 0x1044)); v[1] = __uint_as_float(__byte_perm(h.x, l0, 0x3255));
    v[2] = __uint_as_float(__byte_perm(h.y, l0, 0x1066)); v[3] = __uint_as_float(__byte_perm(h.y, l0, 0x3277));
    v[4] = __uint_as_float(__byte_perm(h.z, l1, 0x1044)); v[5] = __uint_as_float(__byte_perm(h.z, l1, 0x3255));
    v[6] = __uint_as_float(__byte_perm(h.w, l1, 0x1066)); v[7] = __uint_as_float(__byte_perm(h.w, l1, 0x3277));
}

// Tiles in groups of 8 row tiles, rows fastest: the tiles in flight share both operands through L2. Splits are outermost, so
// that they also share their range of k.
struct TileAt {
    int split, m, n, product;
};
__device__ __forceinline__ TileAt tile_at(int t, const GemmParams &p) {
    const int per = p.m_tiles * p.n_tiles;
    TileAt a;
    a.product = t >= per * p.splits;
    a.split = a.product ? 0 : t / per;
    const int mt = a.product ? p.m_tiles2 : p.m_tiles, nt = a.product ? p.n_tiles2 : p.n_tiles;
    const int r = a.product ? t - per * p.splits : t - a.split * per, group = 8 * nt;
    const int g = r / group, left = mt - 8 * g, rows = left < 8 ? left : 8, i = r - g * group;
    a.n = i / rows;
    a.m = 8 * g + i - a.n * rows;
    return a;
}

// the parts of a tile that hold columns of the result
template <typename Sh, bool A_MN, int BN>
__device__ __forceinline__ int parts_of(const TileAt &at, const GemmParams &p) {
    if constexpr (Sh::kParts == 1) return 1;
    const int left = (A_MN && at.product ? p.n2 : p.n) - at.n * BN;
    return left <= BN / 2 ? 1 : 2;
}

template <int CG, int BN, int EPI, bool A_MN, bool B_MN, int ACT>
__global__ void __launch_bounds__(GemmShape<CG, BN, EPI>::kThreads, 1)
gemm_kernel(const __grid_constant__ GemmMaps maps, const GemmParams p) {
    using Sh = GemmShape<CG, BN, EPI>;
    constexpr int ST = Sh::kStages, EW = Sh::kEpiWarps;
    extern __shared__ uint8_t raw[];
    const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
    const uint32_t staging = base + ST * Sh::kStageBytes;
    const uint32_t bars = staging + Sh::kStaging;
    const uint32_t full = bars, empty = full + 8 * ST, tfull = empty + 8 * ST, tempty = tfull + 16, mdone = tempty + 16,
                   slot = mdone + 8, abort_flag = slot + 4;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = CG == 2 ? cluster_rank() : 0;
    WaitCtx wc{abort_flag, p.err_word, p.wait_cycles};

    if (threadIdx.x == 0) {
        for (int i = 0; i < ST; ++i) {
            mbar_init(full + 8 * i, 1);
            mbar_init(empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(tfull + 8 * i, 1);
            mbar_init(tempty + 8 * i, CG * EW);
        }
        mbar_init(mdone, 1);
        sts_s32(abort_flag, 0);
        fence_mbar_init();
    }
    __syncwarp();
    if (warp == 1) tmem_alloc<CG>(slot, Sh::kCols);
    tc_fence_before();
    if constexpr (CG == 2) cluster_sync();
    else __syncthreads();
    tc_fence_after();
    const uint32_t tmem = (uint32_t)lds_volatile_s32(slot);
    grid_wait();
    grid_launch_dependents();

    const int tiles = p.m_tiles * p.n_tiles * p.splits + p.m_tiles2 * p.n_tiles2;
    const int first = blockIdx.x / CG, step = gridDim.x / CG;
    const int blocks = p.kblocks * p.segs;

    if (warp == 0) {
        if (lane == 0) {
            const uint32_t lead_full = CG == 2 ? map_rank(full, 0) : full;
            int s = 0;
            uint32_t ph = 0;
            long long issued = 0;
            bool ok = true;
            for (int t = first; ok && t < tiles; t += step) {
                const TileAt at = tile_at(t, p);
                const int kb0 = (int)((long long)blocks * at.split / p.splits), kb1 = (int)((long long)blocks * (at.split + 1) / p.splits);
                const int m0 = (at.m * CG + (int)rank) * kGemmM;
                const int n0 = EPI == kEpiGate ? at.n * (BN / 2) : at.n * BN + (int)rank * Sh::kPartRows;
                const int parts = parts_of<Sh, A_MN, BN>(at, p);
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (!(ok = mbar_wait(empty + 8 * s, ph ^ 1, wc, kDevWaitEmpty))) break;
                    const int half = kb >= p.kblocks, k0 = (kb - half * p.kblocks) * kGemmK;
                    const int seg = A_MN ? at.product : half;
                    const uint32_t sa = base + s * Sh::kStageBytes, sb = sa + Sh::kABytes, bar = lead_full + 8 * s;
                    if (rank == 0) mbar_arrive_expect_tx(full + 8 * s, CG * (Sh::kStageBytes - (Sh::kParts - parts) * Sh::kPartRows * 128));
                    if (p.test_skip_item != 0 && blockIdx.x == 0 && issued + 1 == p.test_skip_item) {
                        // test hook: this copy never comes
                    } else if constexpr (!A_MN) {
                        tma_tile<CG>(sa, &maps.a[seg], bar, k0, m0);
                    } else {
#pragma unroll
                        for (int j = 0; j < 2; ++j) tma_tile<CG>(sa + j * 8192, &maps.a[seg], bar, m0 + 64 * j, k0);
                    }
                    if constexpr (EPI == kEpiGate) {
                        if constexpr (CG == 2) {
                            tma_tile<CG>(sb, &maps.b[rank], bar, k0, n0);
                        } else {
                            tma_tile<CG>(sb, &maps.b[0], bar, k0, n0);
                            tma_tile<CG>(sb + (BN / 2) * 128, &maps.b[1], bar, k0, n0);
                        }
                    } else if constexpr (!B_MN) {
                        for (int q = 0; q < parts; ++q) tma_tile<CG>(sb + q * Sh::kPartRows * 128, &maps.b[seg], bar, k0, n0 + q * 256);
                    } else {
                        for (int q = 0; q < parts; ++q)
#pragma unroll
                            for (int j = 0; j < Sh::kPartRows / 64; ++j)
                                tma_tile<CG>(sb + q * Sh::kPartRows * 128 + j * 8192, &maps.b[seg], bar, n0 + q * 256 + 64 * j, k0);
                    }
                    ++issued;
                    if (++s == ST) { s = 0; ph ^= 1; }
                }
            }
            for (int i = 0; ok && i < ST; ++i) {         // the last stages' releases arrive before this CTA may leave
                ok = mbar_wait(empty + 8 * s, ph ^ 1, wc, kDevWaitDrain);
                if (++s == ST) { s = 0; ph ^= 1; }
            }
            if (!ok) {
                // unwinding: the copies in flight land before this CTA's shared memory goes away
                const long long t0 = clock64();
                if (rank == 0) {
                    for (long long i = issued > ST ? issued - ST : 0; i < issued; ++i)
                        while (!mbar_try_wait(full + 8 * (int)(i % ST), (uint32_t)(i / ST) & 1) && clock64() - t0 < p.wait_cycles) {}
                } else {
                    while (clock64() - t0 < 2000000) __nanosleep(1000);
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            constexpr uint32_t idesc = mma_idesc(kGemmM * CG, BN / Sh::kParts, A_MN, B_MN);
            constexpr uint32_t ka = A_MN ? 2048 >> 4 : 32 >> 4, kb_ = B_MN ? 2048 >> 4 : 32 >> 4;   // 16 k further
            int s = 0, acc = 0;
            uint32_t ph = 0, aph = 0;
            bool ok = true;
            for (int t = first; ok && t < tiles; t += step) {
                const TileAt at = tile_at(t, p);
                const int kb0 = (int)((long long)blocks * at.split / p.splits), kb1 = (int)((long long)blocks * (at.split + 1) / p.splits);
                const int parts = parts_of<Sh, A_MN, BN>(at, p);
                if (!(ok = mbar_wait(tempty + 8 * acc, aph ^ 1, wc, kDevWaitTmem))) break;
                tc_fence_after();
                const uint32_t d = tmem + acc * BN;
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (!(ok = mbar_wait(full + 8 * s, ph, wc, kDevWaitFull))) break;
                    tc_fence_after();
                    const uint32_t sa = base + s * Sh::kStageBytes;
                    const uint64_t da = tile_desc(sa, A_MN, 8192), db = tile_desc(sa + Sh::kABytes, B_MN, 8192);
                    for (int q = 0; q < parts; ++q)
#pragma unroll
                        for (int k = 0; k < kGemmK / 16; ++k)
                            tc_mma<CG>(d + q * 256, da + k * ka, db + q * (Sh::kPartRows * 128 >> 4) + k * kb_, idesc, kb > kb0 || k > 0);
                    tc_commit<CG>(empty + 8 * s);
                    if (++s == ST) { s = 0; ph ^= 1; }
                }
                if (!ok) break;
                tc_commit<CG>(tfull + 8 * acc);
                if (++acc == Sh::kAccs) { acc = 0; aph ^= 1; }
            }
            tc_drain<CG>(mdone, p.wait_cycles);
        }
    } else {
        const int ew = warp - 2, quad = warp & 3, half = ew >> 2;
        constexpr int HALVES = EW / 4;
        const uint32_t buf = staging + ew * 2 * Sh::kBuf;
        // a result box in shared memory: rows of 128 bytes (64 where gated), 16-byte units permuted as the copy expects them
        const uint32_t mine = lane * (Sh::kGated ? 64 : 128), sw = Sh::kGated ? lane >> 1 & 3 : lane & 7;
        const uint32_t lead_tempty = CG == 2 ? map_rank(tempty, 0) : tempty;
        int acc = 0;
        uint32_t aph = 0;
        int turn = 0;
        constexpr int CW = EPI == kEpiStore ? 64 : 32;                             // columns of a result box
        constexpr int CHUNKS = (EPI == kEpiGate ? BN / 2 : BN) / CW;
        const int kept_cols = (p.n + 31) / 32;
        const auto release = [&] {                                                 // the accumulator has been read
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (CG == 2) mbar_arrive_cluster(lead_tempty + 8 * acc);
                else mbar_arrive(tempty + 8 * acc);
            }
        };
        for (int t = first; t < tiles; t += step) {
            const TileAt at = tile_at(t, p);
            const int row0 = (at.m * CG + (int)rank) * kGemmM + quad * 32;
            const int n0 = at.n * (EPI == kEpiGate ? BN / 2 : BN);
            const int limit_n = A_MN && at.product ? p.n2 : p.n;
            const bool rows = row0 < (A_MN && at.product ? p.m2 : p.m);
            const uint32_t ta = tmem + ((uint32_t)(quad * 32) << 16) + acc * BN;
            uint8_t *kept = Sh::kGated && p.kept ? p.kept + (long long)(row0 >> 5) * kept_cols * kKeptBlock + lane * 16 : nullptr;
            // kEpiGateBwd: the first 16 columns' kept values while the multiplies run
            uint4 kq[EPI == kEpiGateBwd ? 2 : 1][6];
            const auto fetch = [&](uint4 (&q)[6], int i) {                         // step i of this warp: 16 columns
                const int col = n0 + (half + (i >> 1) * HALVES) * 32;
                if (rows && col < p.n) {
                    const uint8_t *src = kept + (long long)(col >> 5) * kKeptBlock + (i & 1) * 1024;
                    q[0] = ld_global_stream_v4(src); q[1] = ld_global_stream_v4(src + 512);
                    q[2] = ld_global_stream_v4(src + 2048); q[3] = ld_global_stream_v4(src + 2560);
                    q[4] = ld_global_stream_v4(src - (i & 1) * 512 + 4096); q[5] = ld_global_stream_v4(src - (i & 1) * 512 + 5120);
                }
            };
            if constexpr (EPI == kEpiGateBwd) fetch(kq[0], 0);
            if (!warp_wait(tfull + 8 * acc, aph, wc, kDevWaitTmem)) break;
            tc_fence_after();
            if constexpr (EPI == kEpiStore || EPI == kEpiPartial) {
#pragma unroll 1
                for (int c = half; c < CHUNKS; c += HALVES) {
                    const int col = n0 + c * CW;
                    const bool live = rows && col < limit_n;
                    const uint32_t dst = buf + turn * 4096 + mine;
                    turn ^= 1;
                    float v[CW];
                    tmem_ld32(ta + c * CW, *reinterpret_cast<float (*)[32]>(&v[0]));
                    if constexpr (CW == 64) tmem_ld32(ta + c * CW + 32, *reinterpret_cast<float (*)[32]>(&v[CW == 64 ? 32 : 0]));
                    if (lane == 0) bulk_wait_read<1>();                            // the store before last has read its buffer
                    tmem_wait_ld();
                    __syncwarp();
                    if (live) {
#pragma unroll
                        for (int q = 0; q < 8; ++q) {
                            if constexpr (EPI == kEpiStore) {
                                using B = Store<__nv_bfloat16>;
                                sts_v4(dst + ((q ^ sw) << 4), B::pack2(v[8 * q], v[8 * q + 1]), B::pack2(v[8 * q + 2], v[8 * q + 3]),
                                       B::pack2(v[8 * q + 4], v[8 * q + 5]), B::pack2(v[8 * q + 6], v[8 * q + 7]));
                            } else {
                                sts_v4(dst + ((q ^ sw) << 4), __float_as_uint(v[4 * q]), __float_as_uint(v[4 * q + 1]),
                                       __float_as_uint(v[4 * q + 2]), __float_as_uint(v[4 * q + 3]));
                            }
                        }
                        fence_async_smem();
                    }
                    __syncwarp();
                    if (lane == 0) {
                        if (live) {
                            if constexpr (EPI == kEpiStore) tma_store_2d(&maps.c[A_MN ? at.product : 0], dst - mine, col, row0);
                            else tma_store_3d(&maps.c[0], dst - mine, col, row0, at.split);
                        }
                        bulk_commit();
                    }
                }
                release();
            } else if constexpr (EPI == kEpiGate) {
                static_assert(CHUNKS == HALVES, "one box of 32 columns per warp");
                const int col = n0 + half * 32;
                const bool live = rows && col < p.n;
                const uint32_t dst = buf + turn * Sh::kBuf + mine;
                turn ^= 1;
                if (lane == 0) bulk_wait_read<1>();
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float g[16], u[16];
                    tmem_ld16(ta + half * 32 + j * 16, g);
                    tmem_ld16(ta + BN / 2 + half * 32 + j * 16, u);
                    tmem_wait_ld();
                    if (j == 1) release();
                    if (!live) continue;
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        float h[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            float a, slope;
                            act_both<ACT>(g[8 * q + e], a, slope);
                            h[e] = a * u[8 * q + e];
                            g[8 * q + e] = a;
                            u[8 * q + e] *= slope;
                        }
                        const uint4 hq = Store<__nv_bfloat16>::pack(h);
                        sts_v4(dst + (((j * 2 + q) ^ sw) << 4), hq.x, hq.y, hq.z, hq.w);
                    }
                    if (p.kept) {
                        uint8_t *to = kept + (long long)(col >> 5) * kKeptBlock;
                        uint4 h0, h1, low;
                        pack_kept(u, h0, h1, low);
                        st_global_v4(to + j * 1024, h0);
                        st_global_v4(to + j * 1024 + 512, h1);
                        st_global_v4(to + 4096 + j * 512, low);
                        pack_kept(g, h0, h1, low);
                        st_global_v4(to + 2048 + j * 1024, h0);
                        st_global_v4(to + 2048 + j * 1024 + 512, h1);
                        st_global_v4(to + 5120 + j * 512, low);
                    }
                }
                fence_async_smem();
                __syncwarp();
                if (lane == 0) {
                    if (live) tma_store_2d(&maps.c[0], dst - mine, col, row0);
                    bulk_commit();
                }
            } else {
                constexpr int STEPS = 2 * CHUNKS / HALVES;
#pragma unroll
                for (int i = 0; i < STEPS; ++i) {
                    const int c = half + (i >> 1) * HALVES, j = i & 1, col = n0 + c * 32;
                    const bool live = rows && col < p.n;
                    float v[16];
                    tmem_ld16(ta + c * 32 + j * 16, v);
                    if (i + 1 < STEPS) fetch(kq[(i + 1) & 1], i + 1);
                    if (j == 0 && lane == 0) bulk_wait_read<0>();
                    tmem_wait_ld();
                    __syncwarp();
                    if (i + 1 == STEPS) release();
                    if (live) {
                        const uint4 (&k)[6] = kq[i & 1];
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            float a[8], b[8];
                            kept_values(k[q], q ? k[4].z : k[4].x, q ? k[4].w : k[4].y, a);
                            kept_values(k[2 + q], q ? k[5].z : k[5].x, q ? k[5].w : k[5].y, b);
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                a[e] *= v[8 * q + e];
                                b[e] *= v[8 * q + e];
                            }
                            const uint32_t o = buf + mine + (((j * 2 + q) ^ sw) << 4);
                            const uint4 aq = Store<__nv_bfloat16>::pack(a), bq = Store<__nv_bfloat16>::pack(b);
                            sts_v4(o, aq.x, aq.y, aq.z, aq.w);
                            sts_v4(o + Sh::kBuf, bq.x, bq.y, bq.z, bq.w);
                        }
                    }
                    if (j == 1) {
                        fence_async_smem();
                        __syncwarp();
                        if (lane == 0 && live) {
                            tma_store_2d(&maps.c[0], buf, col, row0);
                            tma_store_2d(&maps.c[1], buf + Sh::kBuf, col, row0);
                            bulk_commit();
                        }
                    }
                }
            }
            if (++acc == Sh::kAccs) { acc = 0; aph ^= 1; }
        }
        if (lane == 0) bulk_wait_all();
    }
    __syncwarp();
    tc_fence_before();
    if constexpr (CG == 2) cluster_sync();
    else __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_free<CG>(tmem, Sh::kCols);
}

template <int CG, int BN, int EPI, bool A_MN, bool B_MN, int ACT = 0>
cudaError_t launch_gemm_t(const GemmMaps &maps, const GemmParams &p, int sms, cudaStream_t stream) {
    using Sh = GemmShape<CG, BN, EPI>;
    auto kernel = gemm_kernel<CG, BN, EPI, A_MN, B_MN, ACT>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::kSmem);
    if (e != cudaSuccess) return e;
    const long long tiles = (long long)p.m_tiles * p.n_tiles * p.splits + (long long)p.m_tiles2 * p.n_tiles2;
    const long long groups = sms / CG;
    if (tiles < 1 || tiles + groups > 0x7fffffffLL) return cudaErrorInvalidValue;
    return launch_overlapped(kernel, dim3((unsigned)(CG * (tiles < groups ? tiles : groups))), dim3(Sh::kThreads), Sh::kSmem, stream, CG,
                             maps, p);
}

}  // namespace lb
