/* gqa_decode_int8.cu -- gqa_decode.cuh over int8 pools. */
#include "../../include/hal.h"
#include "gqa_launch.cuh"

extern "C" int ct__gqa_ctas_int8(uint32_t dim, uint32_t group) { return ct_gqa::ctas_of<CT_KV_INT8>(dim, group); }
extern "C" int ct__gqa_run_int8(const ct_gqa_args_t *a, uint32_t dim, uint32_t n_workers, void *stream) {
    return ct_gqa::run_of<CT_KV_INT8>(a, dim, n_workers, stream);
}
