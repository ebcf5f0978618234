/*
 * fake_cuda.c -- a device made of host memory, for the tests of the host
 * layer that need one to fail or to be looked into: the CUDA runtime calls and
 * kernel launchers that the paged caches and the grouped-query plans use, as
 * plain copies (bf16 pools).  fake_fail(n) makes the n-th fallible call from
 * now on fail as an allocation does, which, as in the CUDA runtime, leaves its
 * error for the next cudaGetLastError().
 */
#include <cuda_runtime_api.h>
#include <stdint.h>
#include <stdlib.h>
#include <string.h>

#include "../cautreo_b200/csrc/ct_internal.h"
#include "../cautreo_b200/csrc/gqa_internal.h"
#include "../include/hal.h"
#include "../include/kv_cache.h"

static long g_countdown = -1, g_live, g_unfinished;
static cudaError_t g_last;

void fake_fail(long n) { g_countdown = n; }
long fake_pending(void) { return g_countdown; }
long fake_live(void) { return g_live; }
/* Device work since the last wait for the device: on a GPU it may still be running. */
long fake_unfinished(void) { return g_unfinished; }

static cudaError_t step(void) {
    if (g_countdown > 0 && --g_countdown == 0) { g_countdown = -1; return g_last = cudaErrorMemoryAllocation; }
    return cudaSuccess;
}
static cudaError_t take(void **p, size_t n) {
    const cudaError_t e = step();
    if (e) return e;
    *p = aligned_alloc(256, (n + 511) / 256 * 256);
    memset(*p, 0xA5, n);
    g_live++;
    return cudaSuccess;
}
static cudaError_t give(void *p) {
    if (p) g_live--;
    free(p);
    return cudaSuccess;
}

/* ---- the runtime ---------------------------------------------------------- */

cudaError_t cudaGetLastError(void) { const cudaError_t e = g_last; g_last = cudaSuccess; return e; }
const char *cudaGetErrorString(cudaError_t e) { return e ? "made to fail" : "none"; }
cudaError_t cudaGetDeviceCount(int *n) { *n = 1; return cudaSuccess; }
cudaError_t cudaGetDevice(int *d) { *d = 0; return cudaSuccess; }
cudaError_t cudaSetDevice(int d) { return d == 0 ? cudaSuccess : (g_last = cudaErrorInvalidDevice); }
cudaError_t cudaGetDeviceProperties_v2(struct cudaDeviceProp *p, int d) { memset(p, 0, sizeof *p); return cudaSuccess; }
cudaError_t cudaDeviceGetAttribute(int *v, enum cudaDeviceAttr a, int d) { *v = 148; return cudaSuccess; }
cudaError_t cudaDeviceSynchronize(void) { g_unfinished = 0; return cudaSuccess; }
cudaError_t cudaMalloc(void **p, size_t n) { return take(p, n); }
cudaError_t cudaMallocHost(void **p, size_t n) { return take(p, n); }
cudaError_t cudaMallocAsync(void **p, size_t n, cudaStream_t s) { return take(p, n); }
cudaError_t cudaMallocFromPoolAsync(void **p, size_t n, cudaMemPool_t m, cudaStream_t s) { return take(p, n); }
cudaError_t cudaFree(void *p) { return give(p); }
cudaError_t cudaFreeHost(void *p) { return give(p); }
cudaError_t cudaFreeAsync(void *p, cudaStream_t s) { return give(p); }
cudaError_t cudaMemPoolCreate(cudaMemPool_t *m, const struct cudaMemPoolProps *p) { *m = NULL; return cudaSuccess; }
cudaError_t cudaMemPoolDestroy(cudaMemPool_t m) { return cudaSuccess; }
cudaError_t cudaMemPoolSetAttribute(cudaMemPool_t m, enum cudaMemPoolAttr a, void *v) { return cudaSuccess; }
cudaError_t cudaMemcpy(void *d, const void *s, size_t n, enum cudaMemcpyKind k) {
    const cudaError_t e = step();
    g_unfinished++;
    if (!e) memcpy(d, s, n);
    return e;
}
cudaError_t cudaMemcpyAsync(void *d, const void *s, size_t n, enum cudaMemcpyKind k, cudaStream_t st) { return cudaMemcpy(d, s, n, k); }
cudaError_t cudaMemcpy2DAsync(void *d, size_t dp, const void *s, size_t sp, size_t w, size_t h, enum cudaMemcpyKind k, cudaStream_t st) {
    const cudaError_t e = step();
    for (size_t i = 0; !e && i < h; i++) memcpy((char *)d + i * dp, (const char *)s + i * sp, w);
    return e;
}
cudaError_t cudaMemset(void *d, int v, size_t n) {
    const cudaError_t e = step();
    g_unfinished++;
    if (!e) memset(d, v, n);
    return e;
}
cudaError_t cudaMemsetAsync(void *d, int v, size_t n, cudaStream_t st) { return cudaMemset(d, v, n); }
cudaError_t cudaStreamCreateWithFlags(cudaStream_t *s, unsigned f) { *s = NULL; return step(); }
cudaError_t cudaStreamDestroy(cudaStream_t s) { return cudaSuccess; }
cudaError_t cudaStreamSynchronize(cudaStream_t s) { g_unfinished = 0; return cudaSuccess; }
cudaError_t cudaEventCreate(cudaEvent_t *e) { *e = NULL; return cudaSuccess; }
cudaError_t cudaEventCreateWithFlags(cudaEvent_t *e, unsigned f) { *e = NULL; return step(); }
cudaError_t cudaEventDestroy(cudaEvent_t e) { return cudaSuccess; }
cudaError_t cudaEventRecord(cudaEvent_t e, cudaStream_t s) { return step(); }
cudaError_t cudaEventSynchronize(cudaEvent_t e) { return cudaSuccess; }
cudaError_t cudaEventElapsedTime(float *ms, cudaEvent_t a, cudaEvent_t b) { *ms = 0; return cudaSuccess; }

/* ---- launchers: the launch itself may fail, an earlier error shows ---------- */

static int launched(void) {
    step();
    g_unfinished++;
    return ct__cuda_status(cudaGetLastError(), "launch");
}

int ct__launch_scatter_i32(int32_t *dst, const int32_t *pairs, uint32_t n, void *st) {
    const int rc = launched();
    for (uint32_t i = 0; !rc && i < n; i++) dst[pairs[2 * i]] = pairs[2 * i + 1];
    return rc;
}
int ct_kv_paged_move_pages(const void *src, const float *ss, void *dst, float *ds, const int32_t *map, uint32_t n, size_t bytes,
                           uint32_t tokens, void *st) {
    const int rc = launched();
    for (uint32_t i = 0; !rc && i < n; i++) {
        memcpy((char *)dst + i * bytes, (const char *)src + map[i] * bytes, bytes);
        if (ss) memcpy(ds + (size_t)i * tokens, ss + (size_t)map[i] * tokens, tokens * sizeof(float));
    }
    return rc;
}
int ct__launch_gqa_write(void *pool, float *scales, uint32_t dtype, uint32_t heads, uint32_t dim, uint32_t P, uint32_t n_pages,
                         const void *k, const void *v, size_t ks, size_t vs, int f32, const int32_t *slots, uint32_t n, void *st) {
    const int rc = launched();
    for (uint32_t i = 0; !rc && i < n; i++)
        for (uint32_t c = 0; slots[i] >= 0 && c < 2 * heads; c++)
            memcpy((uint16_t *)pool + (((size_t)(slots[i] / P) * 2 * heads + c) * P + slots[i] % P) * dim,
                   c < heads ? (const uint16_t *)k + i * ks + c * dim : (const uint16_t *)v + i * vs + (c - heads) * dim, dim * 2);
    return rc;
}
int ct__launch_gqa_read(const void *pool, const float *scales, uint32_t dtype, uint32_t heads, uint32_t dim, uint32_t P,
                        uint32_t n_pages, const int32_t *slots, uint32_t n, void *k, void *v, size_t ks, size_t vs, int f32,
                        void *st) {
    const int rc = launched();
    for (uint32_t i = 0; !rc && i < n; i++)
        for (uint32_t c = 0; c < 2 * heads; c++)
            memcpy(c < heads ? (uint16_t *)k + i * ks + c * dim : (uint16_t *)v + i * vs + (c - heads) * dim,
                   (const uint16_t *)pool + (((size_t)(slots[i] / P) * 2 * heads + c) * P + slots[i] % P) * dim, dim * 2);
    return rc;
}
/* Bounds: the page's tokens in every code; how many pages were listed, and whether one was listed twice. */
static uint32_t g_listed, g_twice;
uint32_t fake_listed(void) { return g_listed; }
uint32_t fake_listed_twice(void) { return g_twice; }
int ct__launch_gqa_bounds(const void *pool, const float *scales, uint32_t dtype, uint32_t heads, uint32_t dim, uint32_t P,
                          uint32_t n_pages, const int32_t *pages, const int32_t *counts, uint32_t n, int8_t *bounds, float *bs,
                          void *st) {
    const int rc = launched();
    g_listed = n;
    g_twice = 0;
    for (uint32_t i = 0; !rc && i < n; i++) {
        for (uint32_t j = 0; j < i; j++) g_twice += pages[j] == pages[i];
        memset(bounds + (size_t)pages[i] * heads * 2 * dim, counts[i] & 127, heads * 2 * dim);
        for (uint32_t h = 0; h < heads; h++) bs[(size_t)pages[i] * heads + h] = (float)counts[i];
    }
    return rc;
}
/* Whole tokens of bf16. */
int ct_kv_paged_write_slots(void *pool, float *scales, uint32_t dtype, const void *e, uint32_t src, const int32_t *slots, uint32_t n,
                            uint32_t dim, void *st) {
    const int rc = launched();
    for (uint32_t i = 0; !rc && i < n; i++)
        if (slots[i] >= 0) memcpy((uint16_t *)pool + (size_t)slots[i] * dim, (const uint16_t *)e + (size_t)i * dim, dim * 2);
    return rc;
}
int ct__launch_kv_gather(const void *pool, const float *scales, uint32_t dtype, const int32_t *row, uint32_t P, uint32_t dim,
                         uint32_t start, uint32_t n, void *out, uint32_t out_dtype, void *st) {
    const int rc = launched();
    for (uint32_t i = 0; !rc && i < n; i++)
        memcpy((uint16_t *)out + (size_t)i * dim,
               (const uint16_t *)pool + ((size_t)row[(start + i) / P] * P + (start + i) % P) * dim, dim * 2);
    return rc;
}
int ct__launch_kv_gather_batch(const void *pool, const float *scales, uint32_t dtype, const int32_t *bt, uint32_t mp, uint32_t P,
                               uint32_t dim, const void *desc, uint32_t n, uint32_t most, void *out, uint32_t od, void *st) {
    return CT_ERR_UNSUPPORTED;
}
int ct_kv_project_write_slots(const void *x, const void *w, const float *nw, float eps, uint32_t nd, uint32_t n, uint32_t n_in,
                              uint32_t dim, void *pool, float *scales, uint32_t dtype, const int32_t *slots, void *st) {
    return CT_ERR_UNSUPPORTED;
}

/* ---- plans: launches are counted, nothing is computed ----------------------- */

static uint32_t g_runs;
uint32_t fake_runs(void) { return g_runs; }
static int ran(void) { g_runs++; return launched(); }
int ct__gqa_ctas_bf16(uint32_t d, uint32_t g) { return 2; }
int ct__gqa_ctas_int8(uint32_t d, uint32_t g) { return 2; }
int ct__gqa_ctas_e4m3(uint32_t d, uint32_t g) { return 2; }
int ct__gqa_run_bf16(const ct_gqa_args_t *a, uint32_t d, uint32_t n, void *st) { return ran(); }
int ct__gqa_run_int8(const ct_gqa_args_t *a, uint32_t d, uint32_t n, void *st) { return ran(); }
int ct__gqa_run_e4m3(const ct_gqa_args_t *a, uint32_t d, uint32_t n, void *st) { return ran(); }
int ct__gqa_select_prepare(void) { return CT_OK; }
uint32_t ct__gqa_select_max_pages(void) { return 49152; }
int ct__launch_gqa_select(const ct_gqa_select_args_t *a, void *st) { return ran(); }
