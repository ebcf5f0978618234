/* gqa_decode_bf16.cu -- gqa_decode.cuh over bf16 pools. */
#include "../../include/hal.h"
#include "gqa_launch.cuh"

extern "C" int ct__gqa_ctas_bf16(uint32_t dim, uint32_t group) { return ct_gqa::ctas_of<CT_KV_BF16>(dim, group); }
extern "C" int ct__gqa_run_bf16(const ct_gqa_args_t *a, uint32_t dim, uint32_t n_workers, void *stream) {
    return ct_gqa::run_of<CT_KV_BF16>(a, dim, n_workers, stream);
}
