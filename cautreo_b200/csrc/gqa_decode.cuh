/*
 * gqa_decode.cuh -- decode attention of one new token per sequence over a
 * paged cache with K and V per head (pool [page][K, V][kv head][slot][dim]),
 * over every page of the window or over the pages listed for each kv head.
 *
 * Math (sequence s, query head h of kv head c, tokens t that the mask keeps):
 *   x_t = scale * q_h . k_t,  out_h = sum_t softmax(x)_t v_t,  lse_h = ln sum_t exp x_t
 * as one pass over the tokens with a running maximum and sum in the log2
 * domain; a maximum is only followed when it grows by more than 2^8, so the
 * accumulators are rescaled a few times per sequence.
 *
 * Bound: HBM.  A token of a head is 4 D bytes (bf16) for 4 G D flops, G <= 16
 * query heads sharing it: 16 flops a byte at most, a fourteenth of the
 * ridge of the tensor cores, so K and V go through cp.async into shared
 * memory and ldmatrix into mma.sync m16n8k16 with the query heads of the
 * group as the 16 rows (more heads run as further items, whose K and V come
 * from L2).  Codes (int8, e4m3) are widened to bf16 between ldmatrix and the
 * MMA; both widenings are exact, see widen().
 *
 * Split: the steps (TS tokens of an item = sequence x kv head x group of 16
 * heads) of the whole batch lie end to end, and each CTA takes an equal
 * range, found from the device lengths at entry, so no planning launch
 * precedes the kernel.  The warps of a CTA take the steps of a segment in
 * turn, each with its own cp.async ring and its own (max, sum, out), joined
 * through shared memory at the segment's end; an item cut between CTAs
 * leaves fp32 partials that the CTA finishing last joins in index order.
 */
#pragma once
#include <math.h>

#include "../../include/kv_cache.h"
#include "ct_internal.h"
#include "gqa_internal.h"

namespace ct_gqa {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kGrow = 8.0f;           /* log2 growth of a maximum that is followed */

/* Tokens of a warp's step and steps in flight: about 8 KB a step, so that 2
 * CTAs of 4 warps keep ~128 KB in flight on an SM. */
template <int D, int DT> struct Cfg {
    static constexpr int kElt = DT == CT_KV_BF16 ? 2 : 1;
    static constexpr int TS = DT == CT_KV_BF16 ? (D <= 64 ? 32 : 16) : (D <= 128 ? 32 : 16);
    static constexpr int kStages = 3;
    static constexpr int kRow = D * kElt;
    static constexpr int kPitch = kRow + 16;                  /* odd number of 16-B units: conflict-free ldmatrix */
    static constexpr int kScaleBytes = DT == CT_KV_BF16 ? 0 : TS * 8;
    static constexpr int kStage = 2 * TS * kPitch + kScaleBytes;
    static constexpr int kRing = kWarps * kStages * kStage;
};

CT_DEV uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
CT_DEV void cp_async16(uint32_t dst, const void *src, uint32_t bytes) {       /* bytes 16 or 0 (zero fill) */
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
CT_DEV void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> CT_DEV void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

CT_DEV void ldsm4(uint32_t a, uint32_t *r) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
CT_DEV void ldsm4t(uint32_t a, uint32_t *r) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
CT_DEV void mma16816(float *c, const uint32_t *a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
CT_DEV float ex2(float x) {
    float y;
    asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
/* Two floats -> packed bf16 (lo in the low half), round to nearest even. */
CT_DEV uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
CT_DEV uint32_t sub_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

/* Four codes (a 32-bit word) -> bf16 pairs of the even and the odd bytes.
 * int8: 128 + (b & 127) minus 128 or 256, all exact in bf16.
 * e4m3: sign, exponent and mantissa moved to bf16's places, which gives the
 * value times 2^-120 (subnormal codes land on bf16 subnormals of the same
 * ratio); the factor is taken back on the query rows and on the output.
 * 0x7f, NaN in e4m3, is never stored (a row holding NaN has scale NaN). */
template <int DT> CT_DEV void widen(uint32_t w, uint32_t &even, uint32_t &odd) {
    if (DT == CT_KV_INT8) {
        const uint32_t h = w >> 8;
        even = sub_bf16x2((w & 0x007F007Fu) | 0x43004300u, (w & 0x00800080u) | 0x43004300u);
        odd = sub_bf16x2((h & 0x007F007Fu) | 0x43004300u, (h & 0x00800080u) | 0x43004300u);
    } else {
        even = ((w << 8) & 0x80008000u) | ((w << 4) & 0x07F007F0u);
        odd = (w & 0x80008000u) | ((w >> 4) & 0x07F007F0u);
    }
}

/* Steps of a sequence: every item (kv head, group) of it has the same. */
template <int TS>
CT_DEV uint32_t seq_steps(const ct_gqa_args_t &a, uint32_t s, uint32_t &len, uint32_t &start, uint32_t &n_list) {
    const int32_t n = a.seq_lens[s];
    const uint32_t cap = a.max_pages * a.page_tokens;
    len = n < 0 ? 0u : ((uint32_t)n > cap ? cap : (uint32_t)n);
    start = a.window && len > a.window ? len - a.window : 0u;
    uint32_t v;                                              /* tokens to step over */
    n_list = 0;
    if (a.picked) {                                          /* listed pages: those the window has, at most */
        const uint32_t have = len ? (len - 1) / a.page_tokens - start / a.page_tokens + 1 : 0u;
        n_list = have < a.n_pick ? have : a.n_pick;
        v = n_list * a.page_tokens;
    } else {
        v = len - (start & ~15u);
    }
    const uint32_t st = (v + TS - 1) / TS;
    return st ? st : 1u;                                     /* an empty item still writes its zeros */
}

template <int D, int DT>
__global__ void __launch_bounds__(kThreads) k_gqa_decode(const ct_gqa_args_t a) {
    using C = Cfg<D, DT>;
    constexpr int TS = C::TS, NT = TS / 8, GR = TS / 16, kPitch = C::kPitch;
    constexpr bool kQ8 = DT != CT_KV_BF16;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint32_t s_scan[kWarps];
    __shared__ uint32_t s_find[2];                           /* sequence, its first step (low, per head) */
    __shared__ uint64_t s_first;
    __shared__ float s_ml[kWarps][16][2];
    __shared__ uint32_t s_last;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, j = lane & 3;
    const uint32_t HV = a.n_kv_heads * a.n_tiles;

    /* ---- this CTA's range of steps ---- */
    const uint32_t per = (a.n_seq + kThreads - 1) / kThreads;
    uint32_t sum = 0;
    for (uint32_t i = 0; i < per; i++) {
        const uint32_t s = tid * per + i;
        uint32_t len, start, n_list;
        if (s < a.n_seq) sum += seq_steps<TS>(a, s, len, start, n_list);
    }
    uint32_t incl = sum;
    #pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, incl, o);
        if (lane >= (uint32_t)o) incl += y;
    }
    if (lane == 31) s_scan[warp] = incl;
    __syncthreads();
    uint32_t total_seq = 0, before = 0;
    #pragma unroll
    for (int w = 0; w < kWarps; w++) {
        if (w < (int)warp) before += s_scan[w];
        total_seq += s_scan[w];
    }
    const uint32_t excl = before + incl - sum;
    const uint64_t total = (uint64_t)total_seq * HV;
    uint64_t Q = (total + gridDim.x - 1) / gridDim.x;
    if (Q < a.min_steps) Q = a.min_steps;
    const uint64_t x0 = (uint64_t)blockIdx.x * Q;
    if (x0 >= total) return;
    const uint64_t x1 = x0 + Q < total ? x0 + Q : total;
    if (x0 >= (uint64_t)excl * HV && x0 < (uint64_t)(excl + sum) * HV) {
        uint32_t at = excl, s = tid * per, len, start, n_list;
        for (;; s++) {
            const uint32_t st = seq_steps<TS>(a, s, len, start, n_list);
            if (x0 < (uint64_t)(at + st) * HV) break;
            at += st;
        }
        s_find[0] = s;
        s_first = (uint64_t)at * HV;
    }
    __syncthreads();
    uint32_t seq = s_find[0];
    uint64_t seq_x = s_first;                                /* first step of the sequence's first item */

    uint8_t *ring = smem + warp * (C::kStages * C::kStage);
    const uint32_t ring_a = smem_u32(ring);
    /* a segment's end: each warp leaves its [rows][D] sums over its own ring */
    static_assert(16 * D * 4 <= C::kStages * C::kStage, "sums of a warp fit its ring");
    auto join = [&](uint32_t w) { return reinterpret_cast<float *>(smem + w * (C::kStages * C::kStage)); };
    const size_t head_bytes = (size_t)a.page_tokens * C::kRow;
    const size_t v_off = (size_t)a.n_kv_heads * head_bytes;
    /* ldmatrix lane offsets inside a stage */
    const uint32_t mi = lane >> 3, mr = lane & 7;
    const uint32_t k_lane = ((mi >> 1) * 8 + mr) * kPitch + (mi & 1) * 16;
    const uint32_t v_lane = ((mi & 1) * 8 + mr) * kPitch + (mi >> 1) * 16;

    uint64_t x = x0;
    while (x < x1) {
        uint32_t len, start, n_list;
        uint32_t steps = seq_steps<TS>(a, seq, len, start, n_list);
        while (x >= seq_x + (uint64_t)steps * HV) {
            seq_x += (uint64_t)steps * HV;
            seq++;
            steps = seq_steps<TS>(a, seq, len, start, n_list);
        }
        const uint32_t item = (uint32_t)((x - seq_x) / steps);
        const uint32_t tile = item % a.n_tiles, head = item / a.n_tiles;
        const uint64_t item_x = seq_x + (uint64_t)item * steps, item_end = item_x + steps;
        const uint32_t sb = (uint32_t)(x - item_x);
        const uint32_t se = (uint32_t)((x1 < item_end ? x1 : item_end) - item_x);
        const uint32_t rows = a.group - tile * 16 < 16 ? a.group - tile * 16 : 16;
        const uint32_t v_begin = a.picked ? 0u : (start & ~15u);
        const int32_t *table = a.block_table + (size_t)seq * a.max_pages;
        const int32_t *list = a.picked ? a.picked + ((size_t)seq * a.n_kv_heads + head) * a.n_pick : nullptr;

        /* ---- queries as A fragments; rows past the group are zero ---- */
        uint32_t qa[D / 16][4];
        float sc[2];                                         /* log2 scale of rows g, g + 8 */
        #pragma unroll
        for (int h2 = 0; h2 < 2; h2++) {
            const uint32_t r = g + 8 * h2;
            const uint32_t in_group = tile * 16 + r;
            const uint32_t qh = a.blocked ? head * a.group + in_group : in_group * a.n_kv_heads + head;
            const uint16_t *qp = a.q + (size_t)seq * a.q_stride + (size_t)qh * D;
            sc[h2] = a.scale_log2;
            uint2 w[D / 16];
            #pragma unroll
            for (int b = 0; b < D / 16; b++) {
                if (kQ8) {                                   /* values 4j .. 4j+3 of the block */
                    w[b] = r < rows ? __ldg(reinterpret_cast<const uint2 *>(qp + b * 16 + 4 * j)) : make_uint2(0u, 0u);
                } else {
                    w[b].x = r < rows ? __ldg(reinterpret_cast<const uint32_t *>(qp + b * 16 + 2 * j)) : 0u;
                    w[b].y = r < rows ? __ldg(reinterpret_cast<const uint32_t *>(qp + b * 16 + 8 + 2 * j)) : 0u;
                }
            }
            if (kQ8) {
                #pragma unroll
                for (int b = 0; b < D / 16; b++)
                    w[b] = make_uint2(__byte_perm(w[b].x, w[b].y, 0x5410), __byte_perm(w[b].x, w[b].y, 0x7632));
            }
            if (DT == CT_KV_E4M3) {
                /* The keys come 2^-120 too small: the row is multiplied by a
                 * power of two that brings its largest value to [2^119, 2^120)
                 * (exact in bf16), and the scores' factor takes it back. */
                float top = 0.0f;
                #pragma unroll
                for (int b = 0; b < D / 16; b++) {
                    top = fmaxf(fmaxf(top, fabsf(__uint_as_float(w[b].x << 16))), fabsf(__uint_as_float(w[b].x & 0xFFFF0000u)));
                    top = fmaxf(fmaxf(top, fabsf(__uint_as_float(w[b].y << 16))), fabsf(__uint_as_float(w[b].y & 0xFFFF0000u)));
                }
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
                int e = (int)(__float_as_uint(top) >> 23) - 127;      /* floor(log2(top)); Inf: 128 */
                if (e < -8) e = -8;
                if (e > 127) e = 127;
                const float f = __uint_as_float((uint32_t)(119 - e + 127) << 23);
                #pragma unroll
                for (int b = 0; b < D / 16; b++) {
                    w[b].x = pack_bf16(__uint_as_float(w[b].x << 16) * f, __uint_as_float(w[b].x & 0xFFFF0000u) * f);
                    w[b].y = pack_bf16(__uint_as_float(w[b].y << 16) * f, __uint_as_float(w[b].y & 0xFFFF0000u) * f);
                }
                sc[h2] = ldexpf(a.scale_log2, e + 1);
            }
            #pragma unroll
            for (int b = 0; b < D / 16; b++) { qa[b][h2] = w[b].x; qa[b][2 + h2] = w[b].y; }
        }

        float o[D / 8][4];
        #pragma unroll
        for (int i = 0; i < D / 8; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

        /* Physical page of lane's 16-token group of step i: the first GR lanes
         * hold one each; -1 where nothing is to be read. */
        auto lookup = [&](uint32_t i) -> int3 {              /* (physical page, position of its first token, slot) */
            int3 r = make_int3(-1, 0, 0);
            if (i < se && lane < GR) {
                const uint32_t v = v_begin + i * TS + lane * 16;
                const uint32_t e = v / a.page_tokens, off = v - e * a.page_tokens;
                uint32_t lp = e;
                if (list) lp = e < n_list ? (uint32_t)__ldg(list + e) : 0xFFFFFFFFu;
                if (lp < a.max_pages && lp * a.page_tokens < len) {
                    r.x = __ldg(table + lp);
                    r.y = (int)(lp * a.page_tokens + off);
                    r.z = (int)off;
                }
            }
            return r;
        };
        /* Starts the copies of a step into ring slot st; whether it has every
         * one of its tokens. */
        auto fetch = [&](uint32_t st, int3 page) -> bool {
            const uint32_t dst = ring_a + st * C::kStage;
            bool whole = true;
            #pragma unroll
            for (int gr = 0; gr < GR; gr++) {
                const int32_t ph = __shfl_sync(0xFFFFFFFFu, page.x, gr);
                const uint32_t pos = (uint32_t)__shfl_sync(0xFFFFFFFFu, page.y, gr);
                const bool ok = (uint32_t)ph < a.n_pages;
                const uint32_t off = (uint32_t)__shfl_sync(0xFFFFFFFFu, page.z, gr);
                const uint32_t lo = pos < start ? start - pos : 0u;      /* tokens [lo, hi) of the group are kept */
                const uint32_t hi = !ok || pos >= len ? 0u : (len - pos < 16u ? len - pos : 16u);
                whole = whole && lo == 0u && hi == 16u;
                const size_t row0 = (((size_t)(ok ? ph : 0) * 2) * a.n_kv_heads + head) * a.page_tokens + off;
                const uint8_t *k = static_cast<const uint8_t *>(a.pool) + row0 * C::kRow;
                constexpr int CPR = C::kRow / 16, N = 16 * CPR;          /* 16-byte chunks of a row, of the group */
                #pragma unroll
                for (int c0 = 0; c0 < N; c0 += 32) {
                    const uint32_t c = c0 + lane;
                    if (N % 32 != 0 && c >= (uint32_t)N) continue;
                    const uint32_t row = c / CPR, col = c % CPR;
                    const uint32_t bytes = row >= lo && row < hi ? 16u : 0u;
                    const uint32_t d = dst + (gr * 16 + row) * kPitch + col * 16;
                    cp_async16(d, k + c * 16, bytes);
                    cp_async16(d + TS * kPitch, k + v_off + c * 16, bytes);
                }
                if (kQ8 && lane < 8) {                                   /* 16 scales of K, 16 of V */
                    const uint32_t t = (lane & 3) * 4;
                    const uint32_t n = hi > t ? (hi - t < 4u ? hi - t : 4u) : 0u;
                    const float *sp = a.scales + row0 + (lane >> 2) * (size_t)a.n_kv_heads * a.page_tokens + t;
                    cp_async16(dst + 2 * TS * kPitch + ((lane >> 2) * TS + gr * 16 + t) * 4, sp, n * 4);
                }
            }
            return whole;
        };

        uint32_t fi = sb + warp;                             /* next step to fetch */
        int3 page = lookup(fi);
        uint32_t whole_slots = 0;                            /* bit per ring slot */
        #pragma unroll
        for (int st = 0; st < C::kStages - 1; st++) {
            const int3 next = lookup(fi + kWarps);
            if (fi < se && fetch(st, page)) whole_slots |= 1u << st;
            cp_commit();
            page = next;
            fi += kWarps;
        }
        uint32_t slot = 0;
        for (uint32_t i = sb + warp; i < se; i += kWarps) {
            {   /* refill the slot that the previous step freed */
                const int3 next = lookup(fi + kWarps);
                const uint32_t fs = slot == 0 ? C::kStages - 1 : slot - 1;
                whole_slots &= ~(1u << fs);
                if (fi < se && fetch(fs, page)) whole_slots |= 1u << fs;
                cp_commit();
                page = next;
                fi += kWarps;
            }
            cp_wait<C::kStages - 1>();
            __syncwarp();
            const uint32_t stage = ring_a + slot * C::kStage;

            float s[NT][4];
            #pragma unroll
            for (int n = 0; n < NT; n++) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
            #pragma unroll
            for (int gr = 0; gr < GR; gr++) {
                #pragma unroll
                for (int b = 0; b < C::kRow / 32; b++) {
                    uint32_t r[4];
                    ldsm4(stage + k_lane + gr * 16 * kPitch + b * 32, r);
                    if (kQ8) {
                        #pragma unroll
                        for (int h = 0; h < 4; h++) {
                            uint32_t e, od;
                            widen<DT>(r[h], e, od);
                            mma16816(s[2 * gr + (h >> 1)], qa[2 * b + (h & 1)], e, od);
                        }
                    } else {
                        mma16816(s[2 * gr], qa[b], r[0], r[1]);
                        mma16816(s[2 * gr + 1], qa[b], r[2], r[3]);
                    }
                }
            }
            /* scale, mask */
            const float *scp = reinterpret_cast<const float *>(ring + slot * C::kStage + 2 * TS * kPitch);
            float mx[2] = {-INFINITY, -INFINITY};
            #pragma unroll
            for (int n = 0; n < NT; n++) {
                float2 ks = make_float2(1.0f, 1.0f);
                if (kQ8) ks = *reinterpret_cast<const float2 *>(scp + n * 8 + 2 * j);
                s[n][0] *= ks.x * sc[0]; s[n][1] *= ks.y * sc[0];
                s[n][2] *= ks.x * sc[1]; s[n][3] *= ks.y * sc[1];
            }
            const bool whole = (whole_slots >> slot) & 1u;
            if (!whole) {
                #pragma unroll
                for (int gr = 0; gr < GR; gr++) {
                    const uint32_t v = v_begin + i * TS + gr * 16;
                    const uint32_t e = v / a.page_tokens;
                    uint32_t lp = e;
                    if (list) lp = e < n_list ? (uint32_t)__ldg(list + e) : 0xFFFFFFFFu;
                    const bool in = lp < a.max_pages && lp * a.page_tokens < len && (uint32_t)__ldg(table + lp) < a.n_pages;
                    const uint32_t pos = in ? lp * a.page_tokens + (v - e * a.page_tokens) : 0u;
                    #pragma unroll
                    for (int n = 2 * gr; n < 2 * gr + 2; n++) {
                        #pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const uint32_t t = pos + (n & 1) * 8 + 2 * j + h;
                            if (!in || t >= len || t < start) { s[n][h] = -INFINITY; s[n][2 + h] = -INFINITY; }
                        }
                    }
                }
            }
            #pragma unroll
            for (int n = 0; n < NT; n++) {
                mx[0] = fmaxf(mx[0], fmaxf(s[n][0], s[n][1]));
                mx[1] = fmaxf(mx[1], fmaxf(s[n][2], s[n][3]));
            }
            bool grow = false;
            #pragma unroll
            for (int h = 0; h < 2; h++) {
                mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xFFFFFFFFu, mx[h], 1));
                mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xFFFFFFFFu, mx[h], 2));
                grow = grow || mx[h] > m[h] + kGrow;
            }
            if (__any_sync(0xFFFFFFFFu, grow)) {
                #pragma unroll
                for (int h = 0; h < 2; h++) {
                    const float mn = fmaxf(m[h], mx[h]);
                    const float f = mn == -INFINITY ? 1.0f : ex2(m[h] - mn);
                    m[h] = mn;
                    l[h] *= f;
                    #pragma unroll
                    for (int n = 0; n < D / 8; n++) { o[n][2 * h] *= f; o[n][2 * h + 1] *= f; }
                }
            }
            const float mz[2] = {m[0] == -INFINITY ? 0.0f : m[0], m[1] == -INFINITY ? 0.0f : m[1]};
            #pragma unroll
            for (int n = 0; n < NT; n++) {
                #pragma unroll
                for (int h = 0; h < 4; h++) {
                    s[n][h] = ex2(s[n][h] - mz[h >> 1]);
                    l[h >> 1] += s[n][h];
                }
            }
            if (kQ8) {
                #pragma unroll
                for (int n = 0; n < NT; n++) {
                    float2 vs = *reinterpret_cast<const float2 *>(scp + TS + n * 8 + 2 * j);
                    if (DT == CT_KV_E4M3) { vs.x *= 0x1p60f; vs.y *= 0x1p60f; }
                    #pragma unroll
                    for (int h = 0; h < 4; h++) {            /* a masked token's scale may be NaN */
                        const float y = s[n][h] * (h & 1 ? vs.y : vs.x);
                        s[n][h] = !whole && s[n][h] == 0.0f ? 0.0f : y;
                    }
                }
            }
            /* The probabilities as two bf16 digits (16 bits in all): one digit
             * would add an error as large as the rounding of the output. */
            #pragma unroll
            for (int gr = 0; gr < GR; gr++) {
                uint32_t ph[4], pl[4];
                #pragma unroll
                for (int h = 0; h < 4; h++) {
                    const float x0f = s[2 * gr + (h >> 1)][2 * (h & 1)], x1f = s[2 * gr + (h >> 1)][2 * (h & 1) + 1];
                    ph[h] = pack_bf16(x0f, x1f);
                    pl[h] = pack_bf16(x0f - __uint_as_float(ph[h] << 16), x1f - __uint_as_float(ph[h] & 0xFFFF0000u));
                }
                #pragma unroll
                for (int b = 0; b < C::kRow / 32; b++) {
                    uint32_t r[4];
                    ldsm4t(stage + TS * kPitch + v_lane + gr * 16 * kPitch + b * 32, r);
                    if (kQ8) {
                        #pragma unroll
                        for (int h = 0; h < 2; h++) {
                            uint32_t e0, o0, e1, o1;
                            widen<DT>(r[2 * h], e0, o0);
                            widen<DT>(r[2 * h + 1], e1, o1);
                            float *oe = o[4 * b + 2 * h], *oo = o[4 * b + 2 * h + 1];
                            mma16816(oe, ph, e0, e1);
                            mma16816(oo, ph, o0, o1);
                            mma16816(oe, pl, e0, e1);
                            mma16816(oo, pl, o0, o1);
                        }
                    } else {
                        mma16816(o[2 * b], ph, r[0], r[1]);
                        mma16816(o[2 * b + 1], ph, r[2], r[3]);
                        mma16816(o[2 * b], pl, r[0], r[1]);
                        mma16816(o[2 * b + 1], pl, r[2], r[3]);
                    }
                }
            }
            __syncwarp();                                    /* the slot may be refilled */
            slot = slot + 1 == C::kStages ? 0 : slot + 1;
        }
        cp_wait<0>();
        __syncwarp();

        /* ---- join the warps ---- */
        #pragma unroll
        for (int h = 0; h < 2; h++) {
            l[h] += __shfl_xor_sync(0xFFFFFFFFu, l[h], 1);
            l[h] += __shfl_xor_sync(0xFFFFFFFFu, l[h], 2);
            if (j == 0) { s_ml[warp][g + 8 * h][0] = m[h]; s_ml[warp][g + 8 * h][1] = l[h]; }
            if (g + 8 * h < rows) {
                float *dst = join(warp) + (g + 8 * h) * D;
                #pragma unroll
                for (int b = 0; b < D / 16; b++) {
                    if (kQ8) {                               /* the block's values 4j .. 4j+3 */
                        constexpr float f = DT == CT_KV_E4M3 ? 0x1p60f : 1.0f;
                        *reinterpret_cast<float4 *>(dst + b * 16 + 4 * j) =
                            make_float4(o[2 * b][2 * h] * f, o[2 * b + 1][2 * h] * f, o[2 * b][2 * h + 1] * f,
                                        o[2 * b + 1][2 * h + 1] * f);
                    } else {
                        *reinterpret_cast<float2 *>(dst + b * 16 + 2 * j) = make_float2(o[2 * b][2 * h], o[2 * b][2 * h + 1]);
                        *reinterpret_cast<float2 *>(dst + b * 16 + 8 + 2 * j) =
                            make_float2(o[2 * b + 1][2 * h], o[2 * b + 1][2 * h + 1]);
                    }
                }
            }
        }
        __syncthreads();
        const bool cut = sb > 0 || se < steps;
        const uint32_t part = 2 * blockIdx.x + (sb > 0 ? 0u : 1u);
        float *po = a.part_o + (size_t)part * 16 * D;
        float *pml = a.part_ml + (size_t)part * 32;
        auto out_head = [&](uint32_t r) -> uint32_t {
            const uint32_t in_group = tile * 16 + r;
            return a.blocked ? head * a.group + in_group : in_group * a.n_kv_heads + head;
        };
        for (uint32_t c = tid; c < rows * (D / 4); c += kThreads) {
            const uint32_t r = c / (D / 4), d = (c % (D / 4)) * 4;
            float M = s_ml[0][r][0];
            #pragma unroll
            for (int w = 1; w < kWarps; w++) M = fmaxf(M, s_ml[w][r][0]);
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            float L = 0.0f;
            #pragma unroll
            for (int w = 0; w < kWarps; w++) {
                const float f = s_ml[w][r][0] == -INFINITY && !(s_ml[w][r][1] != s_ml[w][r][1]) ? 0.0f : ex2(s_ml[w][r][0] - M);
                const float4 v = *reinterpret_cast<const float4 *>(join(w) + r * D + d);
                L += s_ml[w][r][1] * f;
                acc.x += v.x * f; acc.y += v.y * f; acc.z += v.z * f; acc.w += v.w * f;
            }
            if (cut) {
                __stcg(reinterpret_cast<float4 *>(po + r * D + d), acc);
                if (d == 0) __stcg(reinterpret_cast<float2 *>(pml + 2 * r), make_float2(M, L));
            } else {
                const float inv = L == 0.0f ? 0.0f : 1.0f / L;
                const uint32_t qh = out_head(r);
                uint2 w2;
                w2.x = pack_bf16(acc.x * inv, acc.y * inv);
                w2.y = pack_bf16(acc.z * inv, acc.w * inv);
                *reinterpret_cast<uint2 *>(a.out + ((size_t)seq * a.n_q_heads + qh) * D + d) = w2;
                if (a.lse && d == 0) a.lse[(size_t)seq * a.n_q_heads + qh] = (M + log2f(L)) * kLn2;
            }
        }
        if (cut) {
            /* The CTA that finishes an item last joins its parts, in order. */
            const uint32_t first = (uint32_t)(item_x / Q), last = (uint32_t)((item_end - 1) / Q);
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                const uint32_t n = atomicAdd(a.counters + first, 1u);
                s_last = n == last - first ? 1u : 0u;
                if (s_last) { a.counters[first] = 0u; __threadfence(); }
            }
            __syncthreads();
            if (s_last) {
                for (uint32_t c = tid; c < rows * (D / 4); c += kThreads) {
                    const uint32_t r = c / (D / 4), d = (c % (D / 4)) * 4;
                    float M = -INFINITY;
                    for (uint32_t w = first; w <= last; w++) {
                        const uint32_t p = 2 * w + (w == first ? 1u : 0u);
                        M = fmaxf(M, __ldcg(a.part_ml + (size_t)p * 32 + 2 * r));
                    }
                    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    float L = 0.0f;
                    #pragma unroll 4
                    for (uint32_t w = first; w <= last; w++) {
                        const uint32_t p = 2 * w + (w == first ? 1u : 0u);
                        const float2 ml = __ldcg(reinterpret_cast<const float2 *>(a.part_ml + (size_t)p * 32 + 2 * r));
                        const float4 v = __ldcg(reinterpret_cast<const float4 *>(a.part_o + ((size_t)p * 16 + r) * D + d));
                        const float f = ml.x == -INFINITY && !(ml.y != ml.y) ? 0.0f : ex2(ml.x - M);
                        L += ml.y * f;
                        acc.x += v.x * f; acc.y += v.y * f; acc.z += v.z * f; acc.w += v.w * f;
                    }
                    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
                    const uint32_t qh = out_head(r);
                    uint2 w2;
                    w2.x = pack_bf16(acc.x * inv, acc.y * inv);
                    w2.y = pack_bf16(acc.z * inv, acc.w * inv);
                    *reinterpret_cast<uint2 *>(a.out + ((size_t)seq * a.n_q_heads + qh) * D + d) = w2;
                    if (a.lse && d == 0) a.lse[(size_t)seq * a.n_q_heads + qh] = (M + log2f(L)) * kLn2;
                }
            }
        }
        __syncthreads();                                     /* join and s_ml are free again */
        x = item_x + se;
    }
}

}  // namespace ct_gqa
