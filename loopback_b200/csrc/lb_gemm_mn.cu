// Instantiations of the matrix-product kernel with both with k outermost (dy^T x): gradients of the weights.
#include "lb_gemm.cuh"

namespace lb {

template <int CG, int BN>
static cudaError_t pick(int epilogue, const GemmMaps &maps, const GemmParams &p, int sms, cudaStream_t stream) {
    switch (epilogue) {
        case kEpiStore: return launch_gemm_t<CG, BN, kEpiStore, true, true>(maps, p, sms, stream);
        case kEpiPartial: return launch_gemm_t<CG, BN, kEpiPartial, true, true>(maps, p, sms, stream);
    }
    return cudaErrorInvalidValue;
}

cudaError_t launch_gemm_mn(int tile, int epilogue, const GemmMaps &maps, const GemmParams &p, int sms, cudaStream_t stream) {
    switch (tile) {
        case 0: return pick<1, 128>(epilogue, maps, p, sms, stream);
        case 1: return pick<1, 256>(epilogue, maps, p, sms, stream);
        case 2: return pick<2, 256>(epilogue, maps, p, sms, stream);
        case 3: return epilogue == kEpiStore ? launch_gemm_t<2, 512, kEpiStore, true, true>(maps, p, sms, stream) : cudaErrorInvalidValue;
    }
    return cudaErrorInvalidValue;
}

}  // namespace lb
