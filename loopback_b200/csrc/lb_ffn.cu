// The gated feed-forward block's launches: which instantiation of the matrix product, and the sum of its slices along k.
#include "lb_common.cuh"
#include "lb_kernels.h"
#include "lb_launch.cuh"

namespace lb {

cudaError_t launch_gemm_kk(int tile, int epilogue, const GemmMaps &maps, const GemmParams &p, int sms, cudaStream_t stream);
cudaError_t launch_gemm_kn(int tile, int epilogue, const GemmMaps &maps, const GemmParams &p, int sms, cudaStream_t stream);
cudaError_t launch_gemm_mn(int tile, int epilogue, const GemmMaps &maps, const GemmParams &p, int sms, cudaStream_t stream);

cudaError_t launch_gemm(int tile, int epilogue, int form, const GemmMaps &maps, const GemmParams &p, int sms, cudaStream_t stream) {
    switch (form) {
        case kFormKK: return launch_gemm_kk(tile, epilogue, maps, p, sms, stream);
        case kFormKN: return launch_gemm_kn(tile, epilogue, maps, p, sms, stream);
        case kFormMN: return launch_gemm_mn(tile, epilogue, maps, p, sms, stream);
    }
    return cudaErrorInvalidValue;
}

__global__ void __launch_bounds__(256) gemm_sum_kernel(const float *__restrict__ part, __nv_bfloat16 *__restrict__ out, int splits,
                                                       long long n) {
    const long long stride = (long long)gridDim.x * blockDim.x;
    grid_wait();
    grid_launch_dependents();
    for (long long f = (long long)blockIdx.x * blockDim.x + threadIdx.x; f < n / 8; f += stride) {
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < splits; ++s) {
            const uint4 a = ld_global_stream_v4(part + s * n + f * 8), b = ld_global_stream_v4(part + s * n + f * 8 + 4);
            v[0] += __uint_as_float(a.x); v[1] += __uint_as_float(a.y); v[2] += __uint_as_float(a.z); v[3] += __uint_as_float(a.w);
            v[4] += __uint_as_float(b.x); v[5] += __uint_as_float(b.y); v[6] += __uint_as_float(b.z); v[7] += __uint_as_float(b.w);
        }
        st_global_v4(out + f * 8, Store<__nv_bfloat16>::pack(v));
    }
}

cudaError_t launch_gemm_sum(const float *part, void *out, int splits, long long n, int sms, cudaStream_t stream) {
    const long long need = (n / 8 + 255) / 256, cap = 16LL * sms;
    return launch_overlapped(gemm_sum_kernel, dim3((unsigned)(need < cap ? need : cap)), dim3(256), 0, stream, 1, part,
                        static_cast<__nv_bfloat16 *>(out), splits, n);
}

}  // namespace lb
