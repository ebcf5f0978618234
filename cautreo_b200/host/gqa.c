/*
 * gqa.c -- grouped-query caches and their attention: argument checks, plans
 * and the calls without a handle (kv_cache.h Part 2, attention.h Part 2).
 *
 * A plan owns the scratch of its decode launches: for each worker (a CTA)
 * two partial results of 16 heads and a counter.  The split itself is found
 * on the device from the lengths inside the kernel (csrc/gqa_decode.cuh), so
 * nothing here depends on them.
 */
#include "../../include/attention.h"
#include "../../include/hal.h"
#include "../../include/kv_cache.h"
#include "../csrc/ct_internal.h"
#include "../csrc/gqa_internal.h"

#include <cuda_runtime_api.h>
#include <math.h>
#include <stdlib.h>

struct ct_gqa_plan {
    ct_gqa_shape_t shape;
    uint32_t n_seq, n_workers, n_sms;
    int device;
    float *part_o, *part_ml;     /* one allocation: partial results, their (max, sum), counters */
    uint32_t *counters;
    size_t scratch_bytes;
};

static int misaligned(const void *p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) != 0; }

/* The kernels count a row's entries in 32 bits, a block of threads at a time. */
static const uint32_t kMostSelected = 0x7FFFFFFFu;

static int bad(const char *msg) {
    ct__set_error(msg);
    return CT_ERR_ARG;
}

/* Checks a layout and fills in its defaults. */
int ct__gqa_layout(const ct_kv_gqa_layout_t *in, ct_kv_gqa_layout_t *l) {
    if (!in) return bad("gqa: no layout");
    *l = *in;
    if (l->page_tokens == 0) l->page_tokens = 64;
    if (l->n_kv_heads == 0 || l->n_kv_heads > 256u) return bad("gqa: n_kv_heads (1 .. 256)");
    if (l->page_tokens % 16 != 0 || l->page_tokens > 512) return bad("gqa: page_tokens is a multiple of 16, at most 512");
    if (l->n_pages == 0 || (uint64_t)l->n_pages * l->page_tokens > 0x7FFFFFFFu) return bad("gqa: n_pages x page_tokens");
    if ((uint64_t)l->max_pages_per_seq * l->page_tokens > 0x7FFFFFFFu) return bad("gqa: max_pages_per_seq x page_tokens");
    if (l->kv_dtype != CT_KV_BF16 && l->kv_dtype != CT_KV_INT8 && l->kv_dtype != CT_KV_E4M3) {
        ct__set_error("gqa: bf16, int8 and e4m3 pools only");
        return CT_ERR_UNSUPPORTED;
    }
    const uint32_t d = l->head_dim;
    if (d != 32 && d != 64 && d != 96 && d != 128 && d != 192 && d != 256) {
        ct__set_error("gqa: head_dim 32, 64, 96, 128, 192 or 256 only");
        return CT_ERR_UNSUPPORTED;
    }
    return CT_OK;
}

static int check_pool(const ct_kv_gqa_layout_t *l, const void *pool, const float *scales) {
    if (!pool || misaligned(pool, 16)) return bad("gqa: pool is NULL or not 16-byte aligned");
    if (l->kv_dtype != CT_KV_BF16 && (!scales || misaligned(scales, 16)))
        return bad("gqa: scales are NULL or not 16-byte aligned");
    return CT_OK;
}

/* Rows of K and V values outside the pool: dtype, alignment, stride. */
static int check_rows(const ct_kv_gqa_layout_t *l, const void *k, const void *v, uint64_t *ks, uint64_t *vs, uint32_t dtype) {
    const uint64_t width = (uint64_t)l->n_kv_heads * l->head_dim, unit = dtype == CT_KV_F32 ? 4 : 8;
    if (dtype != CT_KV_BF16 && dtype != CT_KV_F32) return bad("gqa: rows are bf16 or fp32");
    if (!k || !v || misaligned(k, 16) || misaligned(v, 16)) return bad("gqa: k or v is NULL or not 16-byte aligned");
    if (*ks == 0) *ks = width;
    if (*vs == 0) *vs = width;
    if (*ks < width || *vs < width || *ks % unit || *vs % unit) return bad("gqa: k or v stride");
    return CT_OK;
}

int ct_kv_gqa_write_slots(const ct_kv_gqa_layout_t *layout, void *pool, float *scales, const void *k, const void *v,
                          uint64_t k_stride, uint64_t v_stride, uint32_t src_dtype, const int32_t *dest_slot, uint32_t n,
                          void *stream) {
    ct_kv_gqa_layout_t l;
    int rc = ct__gqa_layout(layout, &l);
    if (rc || n == 0) return rc;
    if ((rc = check_pool(&l, pool, scales)) || (rc = check_rows(&l, k, v, &k_stride, &v_stride, src_dtype))) return rc;
    if (!dest_slot) return bad("gqa: no slots");
    if (n > 0x7FFFFFFFu) return bad("gqa: too many tokens in one call");
    return ct__launch_gqa_write(pool, scales, l.kv_dtype, l.n_kv_heads, l.head_dim, l.page_tokens, l.n_pages, k, v, k_stride,
                                v_stride, src_dtype == CT_KV_F32, dest_slot, n, stream);
}

int ct_kv_gqa_read_slots(const ct_kv_gqa_layout_t *layout, const void *pool, const float *scales, const int32_t *src_slot,
                         uint32_t n, void *k_out, void *v_out, uint64_t k_stride, uint64_t v_stride, uint32_t out_dtype,
                         void *stream) {
    ct_kv_gqa_layout_t l;
    int rc = ct__gqa_layout(layout, &l);
    if (rc || n == 0) return rc;
    if ((rc = check_pool(&l, pool, scales)) || (rc = check_rows(&l, k_out, v_out, &k_stride, &v_stride, out_dtype))) return rc;
    if (!src_slot) return bad("gqa: no slots");
    if (n > 0x7FFFFFFFu) return bad("gqa: too many tokens in one call");
    return ct__launch_gqa_read(pool, scales, l.kv_dtype, l.n_kv_heads, l.head_dim, l.page_tokens, l.n_pages, src_slot, n, k_out,
                               v_out, k_stride, v_stride, out_dtype == CT_KV_F32, stream);
}

int ct_kv_gqa_page_bounds(const ct_kv_gqa_layout_t *layout, const void *pool, const float *scales, const int32_t *pages,
                          const int32_t *counts, uint32_t n, int8_t *bounds, float *bound_scales, void *stream) {
    ct_kv_gqa_layout_t l;
    int rc = ct__gqa_layout(layout, &l);
    if (rc || n == 0) return rc;
    if ((rc = check_pool(&l, pool, scales))) return rc;
    if (!pages || !counts || !bounds || !bound_scales) return bad("gqa: NULL argument");
    if ((uint64_t)n * l.n_kv_heads > 0x7FFFFFFFu) return bad("gqa: too many pages in one call");
    return ct__launch_gqa_bounds(pool, scales, l.kv_dtype, l.n_kv_heads, l.head_dim, l.page_tokens, l.n_pages, pages, counts, n,
                                 bounds, bound_scales, stream);
}

/* ---- plans ---------------------------------------------------------------- */

int ct__gqa_decode_ctas(uint32_t dim, uint32_t dtype, uint32_t group) {
    switch (dtype) {
        case CT_KV_BF16: return ct__gqa_ctas_bf16(dim, group);
        case CT_KV_INT8: return ct__gqa_ctas_int8(dim, group);
        case CT_KV_E4M3: return ct__gqa_ctas_e4m3(dim, group);
        default: return 0;
    }
}

int ct__launch_gqa_decode(const ct_gqa_args_t *a, uint32_t dim, uint32_t dtype, uint32_t n_workers, void *stream) {
    switch (dtype) {
        case CT_KV_BF16: return ct__gqa_run_bf16(a, dim, n_workers, stream);
        case CT_KV_INT8: return ct__gqa_run_int8(a, dim, n_workers, stream);
        case CT_KV_E4M3: return ct__gqa_run_e4m3(a, dim, n_workers, stream);
        default: return CT_ERR_UNSUPPORTED;
    }
}

/* Makes `device` current; *prev is what was. */
static int enter(int device, int *prev) {
    int rc = ct__cuda_status(cudaGetDevice(prev), "gqa device");
    if (!rc && *prev != device) rc = ct__cuda_status(cudaSetDevice(device), "gqa device");
    return rc;
}

static void leave(int device, int prev) {
    if (prev != device) cudaSetDevice(prev);
}

void ct_gqa_plan_destroy(ct_gqa_plan_t *p) {
    if (!p) return;
    cudaFree(p->part_o);
    free(p);
}

ct_gqa_plan_t *ct_gqa_plan_create(const ct_gqa_shape_t *shape, uint32_t n_seq, int device) {
    ct_kv_gqa_layout_t l;
    if (!shape || ct__gqa_layout(&shape->kv, &l)) {
        if (!shape) ct__set_error("ct_gqa_plan_create: no shape");
        return NULL;
    }
    if (shape->n_q_heads == 0 || shape->n_q_heads % l.n_kv_heads || shape->head_order > CT_GQA_BLOCKED ||
        l.max_pages_per_seq == 0 || shape->n_q_heads > 65535u) {
        ct__set_error("ct_gqa_plan_create: bad shape");
        return NULL;
    }
    /* the kernel counts the sequences' steps of 16 tokens or more, the steps
     * of a sequence's items, the batch's items and a worker's part of all
     * their steps in 32 bits (5: an item's overhead, rounding; 64: fewer
     * workers than any B200 has) */
    const uint64_t most = (uint64_t)l.max_pages_per_seq * l.page_tokens / 16 + 5;
    const uint64_t items = (uint64_t)l.n_kv_heads * ((shape->n_q_heads / l.n_kv_heads + 15) / 16);     /* of a sequence */
    if (n_seq * most > 0xFFFFFFFFu || most * shape->n_q_heads > 0xFFFFFFFFu || n_seq * items > 0x7FFFFFFFu ||
        n_seq * most > (64ull << 31) / items) {
        ct__set_error("ct_gqa_plan_create: too many sequences for their longest length");
        return NULL;
    }
    ct_gqa_plan_t *p = (ct_gqa_plan_t *)calloc(1, sizeof *p);
    if (!p) { ct__set_error("ct_gqa_plan_create: out of memory"); return NULL; }
    p->shape = *shape;
    p->shape.kv = l;
    if (p->shape.scale == 0.0f) p->shape.scale = 1.0f / sqrtf((float)l.head_dim);
    p->n_seq = n_seq;
    p->device = device;
    int prev = 0;
    if (enter(device, &prev)) { free(p); return NULL; }
    int n_sms = 0, rc = ct__cuda_status(cudaDeviceGetAttribute(&n_sms, cudaDevAttrMultiProcessorCount, device), "gqa plan");
    const int ctas = rc ? 0 : ct__gqa_decode_ctas(l.head_dim, l.kv_dtype, shape->n_q_heads / l.n_kv_heads);
    if (!rc && ctas == 0) { ct__set_error("ct_gqa_plan_create: the decode kernel does not fit this device"); rc = CT_ERR_UNSUPPORTED; }
    if (!rc) rc = ct__gqa_select_prepare();
    if (!rc) {
        p->n_sms = (uint32_t)n_sms;
        p->n_workers = (uint32_t)(n_sms * ctas);
        const size_t po = (size_t)2 * p->n_workers * 16 * l.head_dim * sizeof(float);
        const size_t pm = (size_t)2 * p->n_workers * 32 * sizeof(float), pc = (size_t)3 * p->n_workers * sizeof(uint32_t);
        /* zeroed on a stream of its own: the caller's may be busy, and of any kind */
        cudaStream_t st = NULL;
        rc = ct__cuda_status(cudaMalloc((void **)&p->part_o, po + pm + pc), "gqa scratch");
        if (!rc) rc = ct__cuda_status(cudaStreamCreateWithFlags(&st, cudaStreamNonBlocking), "gqa scratch");
        if (!rc) {
            p->part_ml = p->part_o + po / sizeof(float);
            p->counters = (uint32_t *)(p->part_ml + pm / sizeof(float));
            rc = ct__cuda_status(cudaMemsetAsync(p->counters, 0, pc, st), "gqa scratch");
            if (!rc) rc = ct__cuda_status(cudaStreamSynchronize(st), "gqa scratch");
            cudaStreamDestroy(st);
        }
        p->scratch_bytes = po + pm + pc;
    }
    leave(device, prev);
    if (rc) { ct_gqa_plan_destroy(p); return NULL; }
    return p;
}

uint32_t ct_gqa_plan_workers(const ct_gqa_plan_t *p) { return p ? p->n_workers : 0; }
size_t ct_gqa_plan_scratch_bytes(const ct_gqa_plan_t *p) { return p ? p->scratch_bytes : 0; }

static int check_q(const ct_gqa_plan_t *p, const void *q, uint64_t *stride) {
    const uint64_t width = (uint64_t)p->shape.n_q_heads * p->shape.kv.head_dim;
    if (!q || misaligned(q, 16)) return bad("gqa: q is NULL or not 16-byte aligned");
    if (*stride == 0) *stride = width;
    if (*stride < width || *stride % 8) return bad("gqa: q stride");
    return CT_OK;
}

static int decode(ct_gqa_plan_t *p, const void *q, uint64_t q_stride, const void *pool, const float *scales,
                  const int32_t *block_table, const int32_t *seq_lens, const int32_t *pages, uint32_t n_select, void *out,
                  float *lse, void *stream) {
    const ct_kv_gqa_layout_t *l = &p->shape.kv;
    int rc = check_q(p, q, &q_stride);
    if (rc || (rc = check_pool(l, pool, scales))) return rc;
    if (!block_table || !seq_lens || !out || misaligned(out, 8)) return bad("gqa: table, lengths or out");
    if (p->n_seq == 0) return CT_OK;
    const uint32_t group = p->shape.n_q_heads / l->n_kv_heads;
    const uint64_t items = (uint64_t)p->n_seq * l->n_kv_heads * ((group + 15) / 16);
    const ct_gqa_args_t a = {
        .q = (const uint16_t *)q, .pool = pool, .scales = scales, .block_table = block_table, .seq_lens = seq_lens,
        .picked = pages, .out = (uint16_t *)out, .lse = lse, .part_o = p->part_o, .part_ml = p->part_ml,
        .counters = p->counters, .q_stride = q_stride, .n_seq = p->n_seq, .n_q_heads = p->shape.n_q_heads,
        .n_kv_heads = l->n_kv_heads, .group = group, .n_tiles = (group + 15) / 16, .page_tokens = l->page_tokens,
        .max_pages = l->max_pages_per_seq, .n_pages = l->n_pages, .n_pick = n_select, .window = p->shape.window_tokens,
        .blocked = p->shape.head_order == CT_GQA_BLOCKED,
        /* up to 32 parts are joined at once: somewhat fewer workers than there
         * are beat a second round of joins (one sequence of 8000 tokens,
         * 8 heads: 32 parts of 13.6 us, 37 of 14.7) */
        .most_parts = items && p->n_workers / items <= 64 ? 32u : 0xFFFFFFFFu,
        .scale_log2 = p->shape.scale * 1.4426950408889634f,
        .worker_magic = UINT64_MAX / p->n_workers + 1,
        .spare_magic = items < p->n_workers ? UINT64_MAX / (p->n_workers - items) + 1 : 0,
        .page_magic = ct_gqa_page_magic(l->page_tokens),
    };
    int prev = 0;
    if ((rc = enter(p->device, &prev))) return rc;
    rc = ct__launch_gqa_decode(&a, l->head_dim, l->kv_dtype, p->n_workers, stream);
    leave(p->device, prev);
    return rc;
}

int ct_attn_gqa_decode_paged(ct_gqa_plan_t *plan, const void *q, uint64_t q_stride, const void *pool, const float *scales,
                             const int32_t *block_table, const int32_t *seq_lens, void *out, float *lse, void *stream) {
    if (!plan) return bad("gqa: no plan");
    return decode(plan, q, q_stride, pool, scales, block_table, seq_lens, NULL, 0, out, lse, stream);
}

int ct_attn_gqa_decode_selected(ct_gqa_plan_t *plan, const void *q, uint64_t q_stride, const void *pool, const float *scales,
                                const int32_t *block_table, const int32_t *seq_lens, const int32_t *pages, uint32_t n_select,
                                void *out, float *lse, void *stream) {
    if (!plan) return bad("gqa: no plan");
    if (!pages || n_select == 0 || n_select > kMostSelected) return bad("gqa: no page list, or one too long");
    return decode(plan, q, q_stride, pool, scales, block_table, seq_lens, pages, n_select, out, lse, stream);
}

int ct_attn_gqa_select_pages(ct_gqa_plan_t *plan, const void *q, uint64_t q_stride, const int8_t *bounds,
                             const float *bound_scales, const int32_t *block_table, const int32_t *seq_lens, uint32_t n_select,
                             uint32_t n_first, uint32_t n_last, int32_t *pages_out, void *stream) {
    if (!plan) return bad("gqa: no plan");
    const ct_kv_gqa_layout_t *l = &plan->shape.kv;
    int rc = check_q(plan, q, &q_stride);
    if (rc) return rc;
    if (!bounds || misaligned(bounds, 16) || !bound_scales || !block_table || !seq_lens || !pages_out)
        return bad("gqa: bounds (16-byte aligned), table, lengths or pages");
    if (n_select > kMostSelected) return bad("gqa: n_select (at most 2^31 - 1)");
    if (n_select == 0 || (uint64_t)n_first + n_last > n_select) return bad("gqa: n_first + n_last > n_select, or nothing to select");
    if (l->max_pages_per_seq > ct__gqa_select_max_pages()) {
        ct__set_error("gqa: max_pages_per_seq is beyond the page selection");
        return CT_ERR_UNSUPPORTED;
    }
    if (plan->n_seq == 0) return CT_OK;
    const ct_gqa_select_args_t a = {
        .q = (const uint16_t *)q, .bounds = bounds, .bound_scales = bound_scales, .block_table = block_table,
        .seq_lens = seq_lens, .picked = pages_out, .q_stride = q_stride, .n_seq = plan->n_seq,
        .n_q_heads = plan->shape.n_q_heads, .n_kv_heads = l->n_kv_heads, .group = plan->shape.n_q_heads / l->n_kv_heads,
        .dim = l->head_dim, .page_tokens = l->page_tokens, .max_pages = l->max_pages_per_seq, .n_pages = l->n_pages,
        .n_pick = n_select, .n_first = n_first, .n_last = n_last, .window = plan->shape.window_tokens,
        .blocked = plan->shape.head_order == CT_GQA_BLOCKED, .n_sms = plan->n_sms,
    };
    int prev = 0;
    if ((rc = enter(plan->device, &prev))) return rc;
    rc = ct__launch_gqa_select(&a, stream);
    leave(plan->device, prev);
    return rc;
}
