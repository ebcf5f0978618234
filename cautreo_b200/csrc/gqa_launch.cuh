/*
 * gqa_launch.cuh -- the decode kernels of one storage type: which head sizes
 * exist, how many CTAs of each fit an SM, and their launch.  Included once
 * by each gqa_decode_<type>.cu, so that the types compile side by side.
 */
#pragma once
#include "gqa_decode.cuh"

namespace ct_gqa {

template <int D, int DT> static int ctas() {
    using C = Cfg<D, DT>;
    int n = 0;
    int rc = ct__cuda_status(cudaFuncSetAttribute(k_gqa_decode<D, DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kRing),
                             "gqa decode");
    if (!rc)
        rc = ct__cuda_status(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, k_gqa_decode<D, DT>, kThreads, C::kRing),
                             "gqa decode");
    return rc ? 0 : n;
}

template <int D, int DT> static int run(const ct_gqa_args_t *a, uint32_t n_workers, cudaStream_t st) {
    k_gqa_decode<D, DT><<<n_workers, kThreads, Cfg<D, DT>::kRing, st>>>(*a);
    ct__count_launches(1);
    return ct__cuda_status(cudaGetLastError(), "gqa decode");
}

template <int DT> static int ctas_of(uint32_t dim) {
    switch (dim) {
        case 32: return ctas<32, DT>();
        case 64: return ctas<64, DT>();
        case 96: return ctas<96, DT>();
        case 128: return ctas<128, DT>();
        case 192: return ctas<192, DT>();
        case 256: return ctas<256, DT>();
        default: return 0;
    }
}

template <int DT> static int run_of(const ct_gqa_args_t *a, uint32_t dim, uint32_t n_workers, void *stream) {
    cudaStream_t st = (cudaStream_t)stream;
    switch (dim) {
        case 32: return run<32, DT>(a, n_workers, st);
        case 64: return run<64, DT>(a, n_workers, st);
        case 96: return run<96, DT>(a, n_workers, st);
        case 128: return run<128, DT>(a, n_workers, st);
        case 192: return run<192, DT>(a, n_workers, st);
        case 256: return run<256, DT>(a, n_workers, st);
        default: return CT_ERR_UNSUPPORTED;
    }
}

}  // namespace ct_gqa
