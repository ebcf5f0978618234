/*
 * gqa_launch.cuh -- the decode kernels of one storage type: which head sizes
 * exist, how many CTAs of each fit an SM, and their launch.  Included once
 * by each gqa_decode_<type>.cu, so that the types compile side by side.
 */
#pragma once
#include "gqa_decode.cuh"

namespace ct_gqa {

template <int D, int DT, int HT> static int ctas() {
    using C = Cfg<D, DT, HT>;
    int n[2] = {0, 0}, rc = CT_OK;
    for (int few = 0; few < 2 && !rc; few++) {
        auto kernel = few ? k_gqa_decode<D, DT, HT, true> : k_gqa_decode<D, DT, HT, false>;
        rc = ct__cuda_status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem), "gqa decode");
        if (!rc) rc = ct__cuda_status(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n[few], kernel, kThreads, C::kSmem), "gqa decode");
    }
    return rc ? 0 : n[0] < n[1] ? n[0] : n[1];
}

template <int D, int DT, int HT> static int run(const ct_gqa_args_t *a, uint32_t n_workers, cudaStream_t st) {
    const bool few = 2ull * a->n_seq * a->n_kv_heads * a->n_tiles <= n_workers;
    ct__count_launches(1);
    return ct__cuda_status(ct_gqa_launch(few ? k_gqa_decode<D, DT, HT, true> : k_gqa_decode<D, DT, HT, false>, dim3(n_workers),
                                         dim3(kThreads), Cfg<D, DT, HT>::kSmem, st, 1, *a), "gqa decode");
}

/* Groups of up to 8 query heads take one column tile, larger ones two. */
template <int DT> static int ctas_of(uint32_t dim, uint32_t group) {
    const bool one = group <= 8;
    switch (dim) {
        case 32: return one ? ctas<32, DT, 1>() : ctas<32, DT, 2>();
        case 64: return one ? ctas<64, DT, 1>() : ctas<64, DT, 2>();
        case 96: return one ? ctas<96, DT, 1>() : ctas<96, DT, 2>();
        case 128: return one ? ctas<128, DT, 1>() : ctas<128, DT, 2>();
        case 192: return one ? ctas<192, DT, 1>() : ctas<192, DT, 2>();
        case 256: return one ? ctas<256, DT, 1>() : ctas<256, DT, 2>();
        default: return 0;
    }
}

template <int DT> static int run_of(const ct_gqa_args_t *a, uint32_t dim, uint32_t n_workers, void *stream) {
    cudaStream_t st = (cudaStream_t)stream;
    const bool one = a->group <= 8;
    switch (dim) {
        case 32: return one ? run<32, DT, 1>(a, n_workers, st) : run<32, DT, 2>(a, n_workers, st);
        case 64: return one ? run<64, DT, 1>(a, n_workers, st) : run<64, DT, 2>(a, n_workers, st);
        case 96: return one ? run<96, DT, 1>(a, n_workers, st) : run<96, DT, 2>(a, n_workers, st);
        case 128: return one ? run<128, DT, 1>(a, n_workers, st) : run<128, DT, 2>(a, n_workers, st);
        case 192: return one ? run<192, DT, 1>(a, n_workers, st) : run<192, DT, 2>(a, n_workers, st);
        case 256: return one ? run<256, DT, 1>(a, n_workers, st) : run<256, DT, 2>(a, n_workers, st);
        default: return CT_ERR_UNSUPPORTED;
    }
}

}  // namespace ct_gqa
