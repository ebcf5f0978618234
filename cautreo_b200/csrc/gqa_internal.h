/*
 * gqa_internal.h -- kernel arguments and launchers of the grouped-query cache
 * and its attention, shared by host/gqa.c and csrc/gqa_*.cu.
 */
#ifndef CT_GQA_INTERNAL_H
#define CT_GQA_INTERNAL_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* For dividing tokens by page_tokens (a multiple of 16 up to 512):
 * floor(2^32 / (page_tokens / 16)) + 1; 0 for pages of 16. */
static inline uint32_t ct_gqa_page_magic(uint32_t page_tokens) {
    return page_tokens == 16 ? 0u : (uint32_t)(0x100000000ull / (page_tokens / 16)) + 1u;
}

/* One decode launch.  All pointers are device pointers. */
typedef struct {
    const uint16_t *q;           /* bf16 [n_seq][n_q_heads][D], rows q_stride values apart */
    const void *pool;            /* [n_pages][2][n_kv_heads][page_tokens][D] */
    const float *scales;         /* [n_pages][2][n_kv_heads][page_tokens], 8-bit pools */
    const int32_t *block_table;  /* [n_seq][max_pages] */
    const int32_t *seq_lens;     /* [n_seq] */
    const int32_t *picked;       /* [n_seq][n_kv_heads][n_pick] logical pages, or NULL: all */
    uint16_t *out;               /* bf16 [n_seq][n_q_heads][D] */
    float *lse;                  /* [n_seq][n_q_heads] or NULL */
    float *part_o, *part_ml;     /* [2 n_workers][16][D], [2 n_workers][16][2] */
    uint32_t *counters;          /* [3 n_workers], zero between launches */
    uint64_t q_stride;
    uint32_t n_seq, n_q_heads, n_kv_heads, group, n_tiles;   /* group = query heads a kv head, tiles of 16 of them */
    uint32_t page_tokens, max_pages, n_pages, n_pick, window, blocked;
    uint32_t most_parts;         /* parts of an item, when every worker takes one part */
    float scale_log2;            /* scale x log2(e) */
    uint64_t worker_magic;       /* floor(2^64 / n_workers) + 1: division of less than 2^64 / n_workers */
    uint64_t spare_magic;        /* the same of n_workers less the batch's items, where that is positive */
    uint32_t page_magic;         /* ct_gqa_page_magic(page_tokens) */
#ifdef __CUDACC__
    __device__ __forceinline__ uint32_t page_of(uint32_t v) const;
#endif
} ct_gqa_args_t;

/* One selection launch. */
typedef struct {
    const uint16_t *q;
    const int8_t *bounds;        /* [n_pages][n_kv_heads][2][D]: upper, lower */
    const float *bound_scales;   /* [n_pages][n_kv_heads] */
    const int32_t *block_table, *seq_lens;
    int32_t *picked;             /* [n_seq][n_kv_heads][n_pick] */
    uint64_t q_stride;
    uint32_t n_seq, n_q_heads, n_kv_heads, group, dim;
    uint32_t page_tokens, max_pages, n_pages, n_pick, n_first, n_last, window, blocked;
    uint32_t n_sms;
} ct_gqa_select_args_t;

/* Whether a kernel exists for these, CTAs it runs on an SM of the current
 * device (0: none; also sets the kernel's shared-memory limit there). */
int ct__gqa_decode_ctas(uint32_t dim, uint32_t dtype, uint32_t group);
int ct__launch_gqa_decode(const ct_gqa_args_t *a, uint32_t dim, uint32_t dtype, uint32_t n_workers, void *stream);
/* The same for one storage type (gqa_decode_<type>.cu). */
int ct__gqa_ctas_bf16(uint32_t dim, uint32_t group);
int ct__gqa_ctas_int8(uint32_t dim, uint32_t group);
int ct__gqa_ctas_e4m3(uint32_t dim, uint32_t group);
int ct__gqa_run_bf16(const ct_gqa_args_t *a, uint32_t dim, uint32_t n_workers, void *stream);
int ct__gqa_run_int8(const ct_gqa_args_t *a, uint32_t dim, uint32_t n_workers, void *stream);
int ct__gqa_run_e4m3(const ct_gqa_args_t *a, uint32_t dim, uint32_t n_workers, void *stream);

/* Most pages a sequence may have for a selection; prepares the kernel on the
 * current device. */
int ct__gqa_select_prepare(void);
uint32_t ct__gqa_select_max_pages(void);
int ct__launch_gqa_select(const ct_gqa_select_args_t *a, void *stream);

int ct__launch_gqa_write(void *pool, float *scales, uint32_t dtype, uint32_t n_kv_heads, uint32_t dim, uint32_t page_tokens,
                         uint32_t n_pages, const void *k, const void *v, size_t k_stride, size_t v_stride, int src_f32,
                         const int32_t *slots, uint32_t n, void *stream);
int ct__launch_gqa_read(const void *pool, const float *scales, uint32_t dtype, uint32_t n_kv_heads, uint32_t dim,
                        uint32_t page_tokens, uint32_t n_pages, const int32_t *slots, uint32_t n, void *k, void *v,
                        size_t k_stride, size_t v_stride, int out_f32, void *stream);
int ct__launch_gqa_bounds(const void *pool, const float *scales, uint32_t dtype, uint32_t n_kv_heads, uint32_t dim,
                          uint32_t page_tokens, uint32_t n_pages, const int32_t *pages, const int32_t *counts, uint32_t n,
                          int8_t *bounds, float *bound_scales, void *stream);

#ifdef __cplusplus
}
#endif

#ifdef __CUDACC__
#include <cuda_runtime.h>
/* Page of token v (below 2^31): a product instead of a division; exact while
 * v / 16 < 2^32 / (page_tokens / 16). */
static __device__ __forceinline__ uint32_t ct_gqa_page_of(uint32_t v, uint32_t magic) {
    return magic ? __umulhi(v >> 4, magic) : v >> 4;
}
__device__ __forceinline__ uint32_t ct_gqa_args_t::page_of(uint32_t v) const { return ct_gqa_page_of(v, page_magic); }
/* These kernels are launched while the kernel before them on the stream still
 * drains (programmatic stream serialization): each first lets its own
 * successor do the same, then waits until everything before it has finished
 * and its writes are visible.  Nothing is read or written earlier, so only
 * launch latency overlaps (1 to 2 us of a small call).
 * The kernel before may write what this one reads while this one is already
 * resident, so no memory is read-only for as long as these kernels run: they
 * load with coherent loads that stay behind the wait (ordinary ones, or those
 * below), never through the non-coherent path, whose loads the wait does not
 * cover and the compiler may move. */
static __device__ __forceinline__ void ct_gqa_enter() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}
/* Loads with a cache hint, in program order with the wait above, with barriers
 * and with fences (the hinted intrinsics promise no order): values read once,
 * and what another CTA of the same launch left in L2. */
static __device__ __forceinline__ uint4 ct_gqa_load_once(const uint4 *p) {
    uint4 v;
    asm volatile("ld.global.cs.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
static __device__ __forceinline__ float4 ct_gqa_load_l2(const float4 *p) {
    float4 v;
    asm volatile("ld.global.cg.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p) : "memory");
    return v;
}
static __device__ __forceinline__ float2 ct_gqa_load_l2(const float2 *p) {
    float2 v;
    asm volatile("ld.global.cg.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "l"(p) : "memory");
    return v;
}
template <class... P, class... A>
static inline cudaError_t ct_gqa_launch(void (*k)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, uint32_t cluster,
                                        A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, k, static_cast<P>(args)...);
}
#endif

#endif /* CT_GQA_INTERNAL_H */
