/* gqa_decode_e4m3.cu -- gqa_decode.cuh over e4m3 pools. */
#include "../../include/hal.h"
#include "gqa_launch.cuh"

extern "C" int ct__gqa_ctas_e4m3(uint32_t dim, uint32_t group) { return ct_gqa::ctas_of<CT_KV_E4M3>(dim, group); }
extern "C" int ct__gqa_run_e4m3(const ct_gqa_args_t *a, uint32_t dim, uint32_t n_workers, void *stream) {
    return ct_gqa::run_of<CT_KV_E4M3>(a, dim, n_workers, stream);
}
