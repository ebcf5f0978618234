/*
 * gqa_cache.cu -- the paged cache with K and V per head (pool
 * [page][K, V][kv head][slot][dim]): quantise-on-write, read back, and the
 * bounds of a page's keys that the page selection scores.
 *
 * A row is the D values of one token, K or V, and one head.  8-bit pools hold
 * a scale per row, with the per-token codecs' arithmetic:
 *   d = max|x| / 127 (int8) or / 448 (e4m3),  code = floor(x (1/d) + 1/2) or
 *   e4m3(x (1/d)), every operation rounded once to fp32;
 * a row that holds a NaN or an infinity has scale NaN and codes 0, so that
 * what is read back says so instead of a finite value.
 */
#include <cuda_runtime.h>
#include <float.h>
#include <math.h>

#include <type_traits>

#include "../../include/hal.h"
#include "../../include/kv_cache.h"
#include "ct_internal.h"
#include "gqa_internal.h"

namespace {

constexpr int kThreads = 256;

/* Lanes that share a row, 8 values each: the power of two >= D / 8, so that a
 * row's maximum is reduced by shuffles (a quarter of them idle at 96 and 192). */
__host__ __device__ constexpr int lanes_of(int D) { return D <= 32 ? 4 : D <= 64 ? 8 : D <= 128 ? 16 : 32; }

CT_DEV uint32_t pack2_bf16(float lo, float hi) {
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t *>(&h);
}

/* Both directions: blockIdx.y is the row's place in a token (K heads, then V
 * heads), blockIdx.x a run of tokens, so a block reads or writes a head's
 * consecutive slots as one contiguous run.  A thread moves 8 values of T
 * tokens; all its loads are in flight before the first is used, and the lanes
 * of a row find the tokens' rows once between them.  Bound by HBM in large
 * calls (16384 tokens, 8 heads of 128, bf16 -> int8 18.2 us, 5.6 TB/s of bytes
 * read and written; read back 18.7, at once, the pool still in L2, 11.5), by
 * the launch in small ones (64 tokens with their pages' bounds 5 us). */

/* Row of the pool for a token's slot, or kNoRow. */
constexpr size_t kNoRow = ~(size_t)0;
CT_DEV size_t pool_row(int32_t slot, uint32_t place, uint32_t n_kv_heads, uint32_t page_tokens, uint32_t page_magic, uint32_t n_pages) {
    const uint32_t page = ct_gqa_page_of((uint32_t)slot, page_magic);
    if (slot < 0 || page >= n_pages) return kNoRow;
    return ((size_t)page * 2 * n_kv_heads + place) * page_tokens + ((uint32_t)slot - page * page_tokens);
}
CT_DEV size_t shfl_row(size_t row, uint32_t from) {
    return ((size_t)__shfl_sync(0xFFFFFFFFu, (uint32_t)(row >> 32), from) << 32) | __shfl_sync(0xFFFFFFFFu, (uint32_t)row, from);
}

/* floor(x id + 1/2) of two values in the low bytes of lo and hi: by a
 * round-down addition into the bits of 1.5 x 2^23; two values an instruction,
 * since the 8-bit write issues as many as it can. */
CT_DEV void floor2(float x0, float x1, float id, uint32_t &lo, uint32_t &hi) {
    asm("{ .reg .b64 x, i, h, m;\n\t"
        "mov.b64 x, {%2, %3};\n\tmov.b64 i, {%4, %4};\n\tmov.b64 h, {%5, %5};\n\tmov.b64 m, {%6, %6};\n\t"
        "mul.rn.f32x2 x, x, i;\n\tadd.rn.f32x2 x, x, h;\n\tadd.rm.f32x2 x, x, m;\n\t"
        "mov.b64 {%0, %1}, x; }"
        : "=r"(lo), "=r"(hi) : "f"(x0), "f"(x1), "f"(id), "f"(0.5f), "f"(12582912.0f));
}

template <int D, int DT, bool F32, int T>
__global__ void __launch_bounds__(kThreads) k_gqa_write(void *pool, float *scales, const void *ks, const void *vs, size_t k_stride,
                                                        size_t v_stride, const int32_t *slots, uint32_t n, uint32_t n_kv_heads,
                                                        uint32_t page_tokens, uint32_t page_magic, uint32_t n_pages) {
    constexpr int L = lanes_of(D), U = D / 8, R = kThreads / L;
    const uint32_t u = threadIdx.x % L, place = blockIdx.y;
    const bool is_v = place >= n_kv_heads;
    ct_gqa_enter();
    const uint32_t t0 = blockIdx.x * (R * T) + threadIdx.x / L;
    const size_t col = (size_t)(is_v ? place - n_kv_heads : place) * D + u * 8, stride = is_v ? v_stride : k_stride;
    const void *from = is_v ? vs : ks;
    uint4 w[T][F32 ? 2 : 1];
    /* lane u finds the row of token u & (T - 1) for the lanes that share it */
    const uint32_t own = t0 + (u & (T - 1)) * R;
    const int32_t slot = own < n ? slots[own] : -1;
    #pragma unroll
    for (int i = 0; i < T; i++) {
        const uint32_t t = t0 + i * R;
        if (t >= n || u >= U) continue;
        const size_t at = (size_t)t * stride + col;
        const uint4 *p = F32 ? reinterpret_cast<const uint4 *>(static_cast<const float *>(from) + at)
                             : reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(from) + at);
        w[i][0] = ct_gqa_load_once(p);
        if (F32) w[i][F32 ? 1 : 0] = ct_gqa_load_once(p + 1);
    }
    const size_t mine = pool_row(slot, place, n_kv_heads, page_tokens, page_magic, n_pages);
    /* The four tokens' maxima are reduced together: after two exchanges a lane
     * keeps that of token u & 3, so the divisions run once, not four times. */
    uint32_t top[T];                                         /* bits of max|x|: NaN above Inf above every finite value */
    float d = 0.0f, id = 0.0f;
    if (DT != CT_KV_BF16) {
        #pragma unroll
        for (int i = 0; i < T; i++) {
            top[i] = 0;
            if (t0 + i * R >= n || u >= U) continue;
            if (F32) {
                const uint32_t ws[8] = {w[i][0].x, w[i][0].y, w[i][0].z, w[i][0].w, w[i][F32 ? 1 : 0].x, w[i][F32 ? 1 : 0].y,
                                        w[i][F32 ? 1 : 0].z, w[i][F32 ? 1 : 0].w};
                #pragma unroll
                for (int e = 0; e < 8; e++) top[i] = max(top[i], ws[e] & 0x7FFFFFFFu);
            } else {
                const uint32_t m = __vimax3_u16x2(w[i][0].x & 0x7FFF7FFFu, w[i][0].y & 0x7FFF7FFFu, w[i][0].z & 0x7FFF7FFFu);
                const uint32_t m2 = __vimax3_u16x2(m, w[i][0].w & 0x7FFF7FFFu, 0u);
                top[i] = max(m2 << 16, m2 & 0xFFFF0000u);
            }
        }
        uint32_t r = top[0];
        if (T == 4) {
            const bool b = u & 1, c = u & 2;
            const uint32_t r0 = max(b ? top[T - 3] : top[0], __shfl_xor_sync(0xFFFFFFFFu, b ? top[0] : top[T - 3], 1));
            const uint32_t r1 = max(b ? top[T - 1] : top[T - 2], __shfl_xor_sync(0xFFFFFFFFu, b ? top[T - 2] : top[T - 1], 1));
            r = max(c ? r1 : r0, __shfl_xor_sync(0xFFFFFFFFu, c ? r0 : r1, 2));
        }
        #pragma unroll
        for (int o = T; o < L; o <<= 1) r = max(r, __shfl_xor_sync(0xFFFFFFFFu, r, o));
        const bool fine = r < 0x7F800000u;
        d = fine ? __fdiv_rn(__uint_as_float(r), DT == CT_KV_INT8 ? 127.0f : 448.0f) : __uint_as_float(0x7FC00000u);
        id = fine && d > 0.0f ? fminf(__fdiv_rn(1.0f, d), FLT_MAX) : 0.0f;
    }
    #pragma unroll
    for (int i = 0; i < T; i++) {
        const uint32_t from = (threadIdx.x & (32 - L)) | (i & (L - 1));
        const float di = T == 1 ? d : __shfl_sync(0xFFFFFFFFu, d, from), idi = T == 1 ? id : __shfl_sync(0xFFFFFFFFu, id, from);
        const size_t row = T == 1 ? mine : shfl_row(mine, from);
        if (row == kNoRow || u >= U) continue;
        if (DT == CT_KV_BF16 && !F32) {
            *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(pool) + row * D + u * 8) = w[i][0];
            continue;
        }
        float x[8];
        const uint32_t ws[8] = {w[i][0].x, w[i][0].y, w[i][0].z, w[i][0].w, w[i][F32 ? 1 : 0].x, w[i][F32 ? 1 : 0].y,
                                w[i][F32 ? 1 : 0].z, w[i][F32 ? 1 : 0].w};
        #pragma unroll
        for (int e = 0; e < 8; e++)
            x[e] = F32 ? __uint_as_float(ws[e]) : __uint_as_float((e & 1) ? ws[e >> 1] & 0xFFFF0000u : ws[e >> 1] << 16);
        if (DT == CT_KV_BF16) {
            *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(pool) + row * D + u * 8) =
                make_uint4(pack2_bf16(x[0], x[1]), pack2_bf16(x[2], x[3]), pack2_bf16(x[4], x[5]), pack2_bf16(x[6], x[7]));
            continue;
        }
        uint32_t c[2] = {0u, 0u};
        if (di == di) {                                      /* a NaN or an infinity in the row: codes 0 */
            #pragma unroll
            for (int k = 0; k < 2; k++) {
                if (DT == CT_KV_INT8) {
                    /* |x id| <= 127 (1 + 2^-21), so no code passes +-127 */
                    uint32_t q[4];
                    floor2(x[4 * k], x[4 * k + 1], idi, q[0], q[1]);
                    floor2(x[4 * k + 2], x[4 * k + 3], idi, q[2], q[3]);
                    c[k] = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
                } else {
                    c[k] = (uint32_t)ct_e4m3x2_code(x[4 * k], x[4 * k + 1], idi) |
                           ((uint32_t)ct_e4m3x2_code(x[4 * k + 2], x[4 * k + 3], idi) << 16);
                }
            }
        }
        *reinterpret_cast<uint2 *>(static_cast<uint8_t *>(pool) + row * D + u * 8) = make_uint2(c[0], c[1]);
        if (u == 0) scales[row] = di;
    }
}

/* Eight stored values (w: 16 bytes of bf16, or 8 codes in x and y) in fp32. */
template <int DT> CT_DEV void values8(const uint4 &w, float sc, float *x) {
    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
    #pragma unroll
    for (int i = 0; i < 8; i += 2) {
        if (DT == CT_KV_BF16) {
            x[i] = __uint_as_float(ws[i >> 1] << 16);
            x[i + 1] = __uint_as_float(ws[i >> 1] & 0xFFFF0000u);
        } else {
            const uint32_t c = ws[i >> 2] >> (8 * (i & 3));
            if (DT == CT_KV_INT8) {
                x[i] = __fmul_rn((float)(int8_t)(uint8_t)c, sc);
                x[i + 1] = __fmul_rn((float)(int8_t)(uint8_t)(c >> 8), sc);
            } else {
                const float2 f = ct_e4m3x2_to_f32x2((uint16_t)c);
                x[i] = __fmul_rn(f.x, sc);
                x[i + 1] = __fmul_rn(f.y, sc);
            }
        }
    }
}
template <int D, int DT> CT_DEV uint4 load8(const void *pool, size_t row, uint32_t u) {
    if (DT == CT_KV_BF16) return *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(pool) + row * D + u * 8);
    const uint2 a = *reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(pool) + row * D + u * 8);
    return make_uint4(a.x, a.y, 0u, 0u);
}

template <int D, int DT, bool F32, int T>
__global__ void __launch_bounds__(kThreads) k_gqa_read(const void *pool, const float *scales, const int32_t *slots, uint32_t n,
                                                       uint32_t n_kv_heads, uint32_t page_tokens, uint32_t page_magic, uint32_t n_pages, void *ko,
                                                       void *vo, size_t k_stride, size_t v_stride) {
    constexpr int L = lanes_of(D), U = D / 8, R = kThreads / L;
    const uint32_t u = threadIdx.x % L, place = blockIdx.y;
    ct_gqa_enter();
    const bool is_v = place >= n_kv_heads;
    const uint32_t t0 = blockIdx.x * (R * T) + threadIdx.x / L;
    const size_t col = (size_t)(is_v ? place - n_kv_heads : place) * D + u * 8, stride = is_v ? v_stride : k_stride;
    void *to = is_v ? vo : ko;
    uint4 w[T];
    float sc[T];
    bool ok[T];
    const uint32_t own = t0 + (u & (T - 1)) * R;             /* as in the write */
    const size_t mine = pool_row(own < n ? slots[own] : -1, place, n_kv_heads, page_tokens, page_magic, n_pages);
    #pragma unroll
    for (int i = 0; i < T; i++) {
        const size_t row = T == 1 ? mine : shfl_row(mine, (threadIdx.x & (32 - L)) | (i & (L - 1)));
        ok[i] = row != kNoRow && u < U;
        sc[i] = 1.0f;
        if (!ok[i]) continue;
        w[i] = load8<D, DT>(pool, row, u);
        if (DT != CT_KV_BF16) sc[i] = scales[row];
    }
    #pragma unroll
    for (int i = 0; i < T; i++) {
        if (!ok[i]) continue;
        float x[8];
        values8<DT>(w[i], sc[i], x);
        const size_t at = (size_t)(t0 + i * R) * stride + col;
        if (F32) {
            float4 *p = reinterpret_cast<float4 *>(static_cast<float *>(to) + at);
            __stcs(p, make_float4(x[0], x[1], x[2], x[3]));
            __stcs(p + 1, make_float4(x[4], x[5], x[6], x[7]));
        } else {
            const uint4 y = DT == CT_KV_BF16 ? w[i] : make_uint4(pack2_bf16(x[0], x[1]), pack2_bf16(x[2], x[3]),
                                                                 pack2_bf16(x[4], x[5]), pack2_bf16(x[6], x[7]));
            __stcs(reinterpret_cast<uint4 *>(static_cast<uint16_t *>(to) + at), y);
        }
    }
}

/* Running maxima and minima of a thread's 8 values, over rows w (as load8
 * gives them) with scales sc, and whether any row held a NaN or an infinity.
 * bf16 stays packed: a maximum of bf16 values is one of them. */
template <int DT> struct Range8 {
    float hi[8], lo[8];
    bool bad;
    CT_DEV void start() {
        bad = false;
        #pragma unroll
        for (int e = 0; e < 8; e++) { hi[e] = -INFINITY; lo[e] = INFINITY; }
    }
    /* Two rows: 8-bit values in fp32, products and sums two an instruction,
     * extremes of three. */
    CT_DEV static void row(const uint4 &w, float sc, uint64_t *x) {
        const uint32_t ws[2] = {w.x, w.y};
        #pragma unroll
        for (int i = 0; i < 4; i++) {
            float2 f;
            if (DT == CT_KV_INT8) {                          /* byte + 128 under the exponent of 2^23, minus 2^23 + 128 */
                const uint32_t b = ws[i >> 1] ^ 0x80808080u;
                f.x = __uint_as_float(__byte_perm(b, 0x4B000000u, 0x7540 | (2 * i & 3)));
                f.y = __uint_as_float(__byte_perm(b, 0x4B000000u, 0x7540 | ((2 * i & 3) + 1)));
                asm("{ .reg .b64 m; mov.b64 m, {%3, %3}; mov.b64 %0, {%1, %2}; add.rn.f32x2 %0, %0, m; }"
                    : "=l"(x[i]) : "f"(f.x), "f"(f.y), "f"(-8388736.0f));
            } else {
                f = ct_e4m3x2_to_f32x2((uint16_t)(ws[i >> 1] >> (16 * (i & 1))));
                asm("mov.b64 %0, {%1, %2};" : "=l"(x[i]) : "f"(f.x), "f"(f.y));
            }
            asm("{ .reg .b64 m; mov.b64 m, {%1, %1}; mul.rn.f32x2 %0, %0, m; }" : "+l"(x[i]) : "f"(sc));
        }
    }
    CT_DEV void take(const uint4 &w0, const uint4 &w1, float sc0, float sc1) {
        bad = bad || !(fabsf(sc0) < INFINITY) || !(fabsf(sc1) < INFINITY);
        if (DT == CT_KV_E4M3)                                /* a byte of seven ones is NaN (this cache stores none) */
            bad = bad || ((((w0.x & 0x7F7F7F7Fu) + 0x01010101u) | ((w0.y & 0x7F7F7F7Fu) + 0x01010101u) |
                           ((w1.x & 0x7F7F7F7Fu) + 0x01010101u) | ((w1.y & 0x7F7F7F7Fu) + 0x01010101u)) & 0x80808080u) != 0;
        uint64_t x[4], y[4];
        row(w0, sc0, x);
        row(w1, sc1, y);
        #pragma unroll
        for (int i = 0; i < 4; i++)
            asm("{ .reg .f32 a, b, c, d; mov.b64 {a, b}, %4; mov.b64 {c, d}, %5;\n\t"
                "max.f32 %0, %0, a, c; min.f32 %1, %1, a, c; max.f32 %2, %2, b, d; min.f32 %3, %3, b, d; }"
                : "+f"(hi[2 * i]), "+f"(lo[2 * i]), "+f"(hi[2 * i + 1]), "+f"(lo[2 * i + 1]) : "l"(x[i]), "l"(y[i]));
    }
    CT_DEV void finish() {}
};
template <> struct Range8<CT_KV_BF16> {
    float hi[8], lo[8];
    bool bad;
    __nv_bfloat162 ph[4], pl[4];
    uint32_t top;
    CT_DEV void start() {
        top = 0;
        #pragma unroll
        for (int e = 0; e < 4; e++) {
            ph[e] = __nv_bfloat162(__nv_bfloat162_raw{0xFF80, 0xFF80});
            pl[e] = __nv_bfloat162(__nv_bfloat162_raw{0x7F80, 0x7F80});
        }
    }
    CT_DEV void one(const uint4 &w) {
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
        #pragma unroll
        for (int e = 0; e < 4; e++) {
            const __nv_bfloat162 v = *reinterpret_cast<const __nv_bfloat162 *>(&ws[e]);
            ph[e] = __hmax2(ph[e], v);
            pl[e] = __hmin2(pl[e], v);
        }
        top = __vimax3_u16x2(top, ws[0] & 0x7FFF7FFFu, ws[1] & 0x7FFF7FFFu);
        top = __vimax3_u16x2(top, ws[2] & 0x7FFF7FFFu, ws[3] & 0x7FFF7FFFu);
    }
    CT_DEV void take(const uint4 &w0, const uint4 &w1, float, float) {
        one(w0);
        one(w1);
    }
    CT_DEV void finish() {
        bad = max(top & 0xFFFFu, top >> 16) >= 0x7F80u;
        #pragma unroll
        for (int e = 0; e < 4; e++) {
            const float2 h = __bfloat1622float2(ph[e]), l = __bfloat1622float2(pl[e]);
            hi[2 * e] = h.x; hi[2 * e + 1] = h.y;
            lo[2 * e] = l.x; lo[2 * e + 1] = l.y;
        }
    }
};

/* Bounds of a page's keys, one CTA per (listed page, head):
 *   hi_d = max_t k_td, lo_d = min_t k_td over the page's first `count` tokens,
 *   s = max_d max(|hi_d|, |lo_d|) / 127, codes ceil(hi / s) and floor(lo / s).
 * Maxima and minima have no order, so a page's bounds are the same whichever
 * way its tokens came.  A NaN or an infinity among the keys: scale NaN.
 * Bound by instructions when many pages are new (their keys are still in L2):
 * see Range8; by latency when few are.  256 pages of 64 tokens, 8 heads of
 * 128, int8: 8 us; 1024 of 16 tokens, 8 heads of 64: 14. */
constexpr int kBoundThreads = 128;
template <int D, int DT>
__global__ void __launch_bounds__(kBoundThreads) k_gqa_bounds(const void *pool, const float *scales, uint32_t n_kv_heads,
                                                              uint32_t page_tokens, uint32_t n_pages, const int32_t *pages,
                                                              const int32_t *counts, int8_t *bounds, float *bound_scales) {
    constexpr int U = D / 8, R = kBoundThreads / U, W = kBoundThreads / 32;      /* threads along the row, tokens at a time */
    __shared__ float s_hi[R][D], s_lo[R][D];
    __shared__ float s_top[W];
    ct_gqa_enter();
    const uint32_t i = blockIdx.x / n_kv_heads, head = blockIdx.x - i * n_kv_heads;
    const int32_t page = pages[i], ct = counts[i];
    if (page < 0 || (uint32_t)page >= n_pages) return;
    const uint32_t count = ct < 0 ? 0u : min((uint32_t)ct, page_tokens);
    const uint32_t u = threadIdx.x % U, r = threadIdx.x / U;
    const size_t row0 = ((size_t)page * 2 * n_kv_heads + head) * page_tokens;
    Range8<DT> range;
    range.start();
    /* `n` rows from token t + r on, in flight together; past the end: the last token once more */
    auto rows = [&](uint32_t t, auto n) {
        constexpr int N = decltype(n)::value;
        uint4 w[N];
        float sc[N];
        #pragma unroll
        for (int k = 0; k < N; k++) {
            const size_t row = row0 + min(t + r + k * R, count - 1);
            w[k] = load8<D, DT>(pool, row, u);
            sc[k] = DT == CT_KV_BF16 ? 1.0f : scales[row];
        }
        #pragma unroll
        for (int k = 0; k < N; k += 2) range.take(w[k], w[k + 1], sc[k], sc[k + 1]);
    };
    if (r < R) {
        #pragma unroll 1
        for (uint32_t t = 0; t < count;) {
            if (count - t > 2 * R) {
                rows(t, std::integral_constant<int, 8>());
                t += 8 * R;
            } else {
                rows(t, std::integral_constant<int, 2>());
                t += 2 * R;
            }
        }
    }
    range.finish();
    if (r < R) {
        #pragma unroll
        for (int e = 0; e < 8; e += 4) {
            *reinterpret_cast<float4 *>(&s_hi[r][u * 8 + e]) = make_float4(range.hi[e], range.hi[e + 1], range.hi[e + 2], range.hi[e + 3]);
            *reinterpret_cast<float4 *>(&s_lo[r][u * 8 + e]) = make_float4(range.lo[e], range.lo[e + 1], range.lo[e + 2], range.lo[e + 3]);
        }
    }
    float top = 0.0f;
    #pragma unroll
    for (int e = 0; e < 8; e++) top = fmaxf(top, fmaxf(fabsf(range.hi[e]), fabsf(range.lo[e])));
    if (r >= R || count <= r) top = 0.0f;                    /* a thread without tokens */
    top = ct_warp_max(top);
    if ((threadIdx.x & 31) == 0) s_top[threadIdx.x >> 5] = top;
    const bool fine = !__syncthreads_or(r < R && range.bad);
    #pragma unroll
    for (int k = 0; k < W; k++) top = fmaxf(top, s_top[k]);
    const float s = __fdiv_rn(top, 127.0f);
    const size_t out = (size_t)page * n_kv_heads + head;
    /* a bound a thread at a time: the upper ones, then the lower ones */
    #pragma unroll 1
    for (uint32_t c = threadIdx.x; c < 2 * D; c += kBoundThreads) {
        const bool lower = c >= D;
        const float *from = lower ? &s_lo[0][c - D] : &s_hi[0][c];
        float b = from[0];
        #pragma unroll 8
        for (int k = 1; k < R; k++) b = lower ? fminf(b, from[k * D]) : fmaxf(b, from[k * D]);
        int code = 0;
        if (fine && s > 0.0f) {
            const float y = __fdiv_rn(b, s);
            code = max(-127, min(127, lower ? __float2int_rd(y) : __float2int_ru(y)));
        }
        bounds[out * 2 * D + c] = (int8_t)code;
    }
    if (threadIdx.x == 0) bound_scales[out] = fine ? s : __uint_as_float(0x7FC00000u);
}

#define CT_BY_DIM(call)                            \
    switch (dim) {                                 \
        case 32: { constexpr int D = 32; call; }   \
        case 64: { constexpr int D = 64; call; }   \
        case 96: { constexpr int D = 96; call; }   \
        case 128: { constexpr int D = 128; call; } \
        case 192: { constexpr int D = 192; call; } \
        case 256: { constexpr int D = 256; call; } \
        default: return CT_ERR_UNSUPPORTED;        \
    }

/* Tokens a thread moves: 4 when the call fills the GPU with them, else 1.
 * Write, read back in us, in ones and in fours: 8 heads of 128, bf16 -> int8,
 * 64 tokens 1.4, 1.5 and 1.9, 1.8; 2048 4.2, 3.4 and 4.2, 3.3; 4096 7.1, 5.7
 * and 6.1, 4.5; 16384 24.7, 24.1 and 18.2, 18.4; 5 heads of 96, fp32 <-> e4m3,
 * 2560 tokens 3.6, 3.4 and 3.6, 4.7; 4096 5.4, 4.7 and 5.2, 6.3; 16384 16.7,
 * 18.8 and 15.0, 17.0.  The limit lies between 4096 x 5 and 4096 x 8. */
inline bool many(uint32_t n, uint32_t heads) { return (uint64_t)n * heads >= 24576; }

struct WriteCall {
    void *pool; float *scales; const void *k, *v; size_t ks, vs; const int32_t *slots;
    uint32_t n, heads, pt, np; cudaStream_t st;
    template <int D, int DT, bool F32> int go() const {
        constexpr uint32_t R = kThreads / lanes_of(D);
        ct__count_launches(1);
        return ct__cuda_status(many(n, heads) ? launch(k_gqa_write<D, DT, F32, 4>, 4 * R) : launch(k_gqa_write<D, DT, F32, 1>, R),
                               "gqa write");
    }
    template <class K> cudaError_t launch(K k_, uint32_t tokens) const {
        return ct_gqa_launch(k_, dim3((n + tokens - 1) / tokens, 2 * heads), dim3(kThreads), 0, st, 1, pool, scales, k, v, ks, vs,
                             slots, n, heads, pt, ct_gqa_page_magic(pt), np);
    }
};

struct ReadCall {
    const void *pool; const float *scales; const int32_t *slots; uint32_t n, heads, pt, np; void *k, *v; size_t ks, vs;
    cudaStream_t st;
    template <int D, int DT, bool F32> int go() const {
        constexpr uint32_t R = kThreads / lanes_of(D);
        ct__count_launches(1);
        return ct__cuda_status(many(n, heads) ? launch(k_gqa_read<D, DT, F32, 4>, 4 * R) : launch(k_gqa_read<D, DT, F32, 1>, R),
                               "gqa read");
    }
    template <class K> cudaError_t launch(K k_, uint32_t tokens) const {
        return ct_gqa_launch(k_, dim3((n + tokens - 1) / tokens, 2 * heads), dim3(kThreads), 0, st, 1, pool, scales, slots, n, heads,
                             pt, ct_gqa_page_magic(pt), np, k, v, ks, vs);
    }
};

template <int D, class Call> int by_type(const Call &c, uint32_t dtype, int f32) {
    switch (dtype) {
        case CT_KV_BF16: return f32 ? c.template go<D, CT_KV_BF16, true>() : c.template go<D, CT_KV_BF16, false>();
        case CT_KV_INT8: return f32 ? c.template go<D, CT_KV_INT8, true>() : c.template go<D, CT_KV_INT8, false>();
        case CT_KV_E4M3: return f32 ? c.template go<D, CT_KV_E4M3, true>() : c.template go<D, CT_KV_E4M3, false>();
        default: return CT_ERR_UNSUPPORTED;
    }
}

template <int D>
int bounds_of(const void *pool, const float *scales, uint32_t dtype, uint32_t heads, uint32_t pt, uint32_t np, const int32_t *pages,
              const int32_t *counts, uint32_t n, int8_t *bounds, float *bs, cudaStream_t st) {
    auto kernel = dtype == CT_KV_BF16 ? k_gqa_bounds<D, CT_KV_BF16> : dtype == CT_KV_INT8 ? k_gqa_bounds<D, CT_KV_INT8>
                                                                                     : k_gqa_bounds<D, CT_KV_E4M3>;
    ct__count_launches(1);
    return ct__cuda_status(ct_gqa_launch(kernel, dim3(n * heads), dim3(kBoundThreads), 0, st, 1, pool, scales, heads, pt, np, pages,
                                         counts, bounds, bs), "gqa bounds");
}

}  // namespace

extern "C" int ct__launch_gqa_write(void *pool, float *scales, uint32_t dtype, uint32_t n_kv_heads, uint32_t dim, uint32_t page_tokens,
                                    uint32_t n_pages, const void *k, const void *v, size_t k_stride, size_t v_stride, int src_f32,
                                    const int32_t *slots, uint32_t n, void *stream) {
    const WriteCall c = {pool, scales, k, v, k_stride, v_stride, slots, n, n_kv_heads, page_tokens, n_pages, (cudaStream_t)stream};
    CT_BY_DIM(return by_type<D>(c, dtype, src_f32));
}

extern "C" int ct__launch_gqa_read(const void *pool, const float *scales, uint32_t dtype, uint32_t n_kv_heads, uint32_t dim,
                                   uint32_t page_tokens, uint32_t n_pages, const int32_t *slots, uint32_t n, void *k, void *v,
                                   size_t k_stride, size_t v_stride, int out_f32, void *stream) {
    const ReadCall c = {pool, scales, slots, n, n_kv_heads, page_tokens, n_pages, k, v, k_stride, v_stride, (cudaStream_t)stream};
    CT_BY_DIM(return by_type<D>(c, dtype, out_f32));
}

extern "C" int ct__launch_gqa_bounds(const void *pool, const float *scales, uint32_t dtype, uint32_t n_kv_heads, uint32_t dim,
                                     uint32_t page_tokens, uint32_t n_pages, const int32_t *pages, const int32_t *counts, uint32_t n,
                                     int8_t *bounds, float *bound_scales, void *stream) {
    CT_BY_DIM(return bounds_of<D>(pool, scales, dtype, n_kv_heads, page_tokens, n_pages, pages, counts, n, bounds, bound_scales,
                                  (cudaStream_t)stream));
}
