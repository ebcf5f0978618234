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
 * ridge of the tensor cores.  So K and V go through cp.async into shared
 * memory and ldmatrix into mma.sync m16n8k16 with 16 tokens (for the scores)
 * or 16 values of a head (for the output) as the rows and 8 query heads of
 * the group as the columns: a group of up to 8 heads wastes nothing on rows,
 * 9 to 16 take two column tiles over the same K and V fragments, more run as
 * further items.  Scores come out as [token][head] and are needed as
 * [token][head] operands: two movmatrix per 16 tokens.
 *
 * bf16 pools: probabilities enter as two bf16 digits (one would add an error
 * as large as the rounding of the output).  8-bit pools: codes are widened to
 * fp16 (exact), queries are brought to fp16 by a power of two a head (exact
 * down to 2^-29 of the head's largest value), and probability x V scale is
 * one fp16 digit (11 bits) of a running power-of-two unit; see `unit`.
 *
 * Split: the steps (TS tokens of an item = sequence x kv head x group of 16
 * heads) of the whole batch lie end to end, each item with kItemCost steps of
 * overhead, and each CTA takes an equal range, found from the device lengths
 * at entry, so no planning launch precedes the kernel.  An item of at most
 * kSolo steps is one warp's; the warps of a CTA share longer ones, each with
 * its own cp.async ring and its own (max, sum, out), joined through shared
 * memory; an item cut between CTAs leaves fp32 partials that the CTA
 * finishing last joins in index order.
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
constexpr uint32_t kItemCost = 4;       /* steps that an item's start and end are counted as */
constexpr uint32_t kSolo = 8;           /* steps up to which an item is one warp's */

/* Tokens of a warp's step (2 to 17 KB of K and V) and steps in the ring. */
template <int D, int DT> struct Cfg {
    static constexpr int kElt = DT == CT_KV_BF16 ? 2 : 1;
    static constexpr int kRow = D * kElt;
    static constexpr int TS = kRow <= 64 ? 32 : 16;
    static constexpr int kStages = 3;
    static constexpr int kPitch = kRow + 16;                  /* odd number of 16-B units: conflict-free ldmatrix */
    static constexpr int kScaleBytes = DT == CT_KV_BF16 ? 0 : TS * 8;
    static constexpr int kStage = 2 * TS * kPitch + kScaleBytes;
    static constexpr int kRing = kWarps * kStages * kStage;
};

CT_DEV uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
CT_DEV void cp_async16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
CT_DEV void cp_async16_part(uint32_t dst, const void *src, uint32_t bytes) {  /* the rest of the 16 bytes: zeros */
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
CT_DEV uint32_t transpose8(uint32_t x) {                      /* an 8 x 8 matrix of 16-bit values over the warp */
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
template <bool F16> CT_DEV void mma16816(float *c, const uint32_t *a, uint32_t b0, uint32_t b1) {
    if (F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                     "{%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
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
/* Two floats -> packed (lo in the low half), round to nearest even. */
CT_DEV uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
CT_DEV uint32_t pack_f16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
CT_DEV float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
CT_DEV float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
CT_DEV float pow2f(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   /* -126 <= e <= 127 */

/* Four codes (a 32-bit word) -> two fp16 pairs, exact: bytes (0, 1), (2, 3),
 * or with Even (0, 2), (1, 3).  int8: the byte + 128 under the exponent of
 * 1024, minus 1152. */
template <int DT, bool Even> CT_DEV void widen(uint32_t w, uint32_t &a, uint32_t &b) {
    if (DT == CT_KV_INT8) {
        const uint32_t u = w ^ 0x80808080u;
        a = __byte_perm(u, 0x64646464u, Even ? 0x4240 : 0x4140);
        b = __byte_perm(u, 0x64646464u, Even ? 0x4341 : 0x4342);
        asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(a) : "r"(0x64806480u));
        asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(b) : "r"(0x64806480u));
    } else {
        const uint32_t u = Even ? __byte_perm(w, 0u, 0x3120) : w;
        asm("{ .reg .b16 lo, hi; mov.b32 {lo, hi}, %2; cvt.rn.f16x2.e4m3x2 %0, lo; cvt.rn.f16x2.e4m3x2 %1, hi; }"
            : "=r"(a), "=r"(b) : "r"(u));
    }
}

/* Steps of a sequence: every item (kv head, group) of it has the same. */
struct Seq {
    uint32_t len, start;                                     /* tokens [start, len) are attended */
    uint32_t n_list;                                         /* listed pages stepped over */
    uint32_t steps;
};
template <int TS> CT_DEV Seq sequence(const ct_gqa_args_t &a, uint32_t s) {
    Seq r;
    const int32_t n = __ldg(a.seq_lens + s);
    const uint32_t cap = a.max_pages * a.page_tokens;
    r.len = n < 0 ? 0u : ((uint32_t)n > cap ? cap : (uint32_t)n);
    r.start = a.window && r.len > a.window ? r.len - a.window : 0u;
    r.n_list = 0;
    uint32_t v;                                              /* tokens to step over */
    if (a.picked) {                                          /* listed pages: as many as the window has, at most */
        const uint32_t have = r.len ? a.page_of(r.len - 1) - a.page_of(r.start) + 1 : 0u;
        r.n_list = have < a.n_pick ? have : a.n_pick;
        v = r.n_list * a.page_tokens;
    } else {
        v = r.len - (r.start & ~15u);
    }
    const uint32_t st = (v + TS - 1) / TS;
    r.steps = st ? st : 1u;                                  /* an empty item still writes its zeros */
    return r;
}

/* HT: column tiles of 8 query heads. */
template <int D, int DT, int HT>
__global__ void __launch_bounds__(kThreads) k_gqa_decode(const ct_gqa_args_t a) {
    using C = Cfg<D, DT>;
    constexpr int TS = C::TS, GR = TS / 16, kPitch = C::kPitch, KB = D / 16;
    constexpr int kHeads = 8 * HT, kJoin = D + 4;            /* pitch of a head's sums: lanes' writes in distinct banks */
    constexpr bool kQ8 = DT != CT_KV_BF16;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint32_t s_scan[kWarps];
    __shared__ uint32_t s_seq;
    __shared__ uint64_t s_first;
    __shared__ float s_ml[kWarps][kHeads][2];
    __shared__ uint32_t s_last;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, j = lane & 3;
    const uint32_t HV = a.n_kv_heads * a.n_tiles;

    /* ---- this CTA's range of steps ---- */
    const uint32_t per = (a.n_seq + kThreads - 1) / kThreads;
    uint32_t sum = 0;
    for (uint32_t i = 0; i < per; i++) {
        const uint32_t s = tid * per + i;
        if (s < a.n_seq) sum += sequence<TS>(a, s).steps + kItemCost;
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
    uint64_t x = (uint64_t)blockIdx.x * Q;
    if (x >= total) return;
    const uint64_t x1 = x + Q < total ? x + Q : total;
    if (x >= (uint64_t)excl * HV && x < (uint64_t)(excl + sum) * HV) {
        uint32_t at = excl, s = tid * per;
        for (;; s++) {
            const uint32_t c = sequence<TS>(a, s).steps + kItemCost;
            if (x < (uint64_t)(at + c) * HV) break;
            at += c;
        }
        s_seq = s;
        s_first = (uint64_t)at * HV;
    }
    __syncthreads();
    uint32_t seq = s_seq;
    uint64_t seq_x = s_first;                                /* where the sequence's first item begins */
    Seq sq = sequence<TS>(a, seq);

    uint8_t *ring = smem + warp * (C::kStages * C::kStage);
    const uint32_t ring_a = smem_u32(ring);
    /* a segment's end: each warp leaves its [head][D] sums over its own ring */
    static_assert(kHeads * kJoin * 4 <= C::kStages * C::kStage, "sums of a warp fit its ring");
    auto join = [&](uint32_t w) { return reinterpret_cast<float *>(smem + w * (C::kStages * C::kStage)); };
    const size_t v_off = (size_t)a.n_kv_heads * a.page_tokens * C::kRow;
    /* ldmatrix lane offsets inside a stage */
    const uint32_t mi = lane >> 3, mr = lane & 7;
    const uint32_t k_lane = ((mi & 1) * 8 + mr) * kPitch + (mi >> 1) * 16;
    const uint32_t v_lane = kQ8 ? k_lane : ((mi >> 1) * 8 + mr) * kPitch + (mi & 1) * 16;
    uint32_t turn = 0;                                       /* short items so far: whose turn it is */

    while (x < x1) {
        uint64_t seq_end = seq_x + (uint64_t)(sq.steps + kItemCost) * HV;
        while (x >= seq_end) {
            seq_x = seq_end;
            seq++;
            sq = sequence<TS>(a, seq);
            seq_end = seq_x + (uint64_t)(sq.steps + kItemCost) * HV;
        }
        const uint32_t width = sq.steps + kItemCost;
        const uint32_t item = (uint32_t)(x - seq_x) / width;             /* both below 2^32: see the plan */
        const uint64_t item_x = seq_x + (uint64_t)item * width, item_end = item_x + width;
        const uint64_t end = x1 < item_end ? x1 : item_end;
        const uint32_t sb = x > item_x + kItemCost ? (uint32_t)(x - item_x) - kItemCost : 0u;
        const uint32_t se = end > item_x + kItemCost ? (uint32_t)(end - item_x) - kItemCost : 0u;
        x = end;
        if (se <= sb) continue;                              /* only overhead fell into this range */
        const bool cut = sb > 0 || se < sq.steps;
        const bool solo = !cut && sq.steps <= kSolo;
        if (solo && (turn++ & (kWarps - 1)) != warp) continue;

        const uint32_t tile = item % a.n_tiles, head = item / a.n_tiles;
        const uint32_t rows = a.group - tile * 16 < 16 ? a.group - tile * 16 : 16;
        const uint32_t v_begin = a.picked ? 0u : (sq.start & ~15u);
        const int32_t *table = a.block_table + (size_t)seq * a.max_pages;
        const int32_t *list = a.picked ? a.picked + ((size_t)seq * a.n_kv_heads + head) * a.n_pick : nullptr;
        const uint32_t stride = solo ? 1u : (uint32_t)kWarps;
        auto query_head = [&](uint32_t r) -> uint32_t {
            const uint32_t in_group = tile * 16 + r;
            return a.blocked ? head * a.group + in_group : in_group * a.n_kv_heads + head;
        };

        /* Logical page of 16-token group gr of step i (0xFFFFFFFF: none). */
        auto entry = [&](uint32_t i, int gr) -> uint32_t {
            const uint32_t e = a.page_of(v_begin + i * TS + gr * 16);
            if (!list) return i < se ? e : 0xFFFFFFFFu;
            return i < se && e < sq.n_list ? (uint32_t)__ldg(list + e) : 0xFFFFFFFFu;
        };
        /* Its physical page (>= n_pages: nothing to read). */
        auto mapped = [&](uint32_t lp) -> uint32_t {
            return lp < a.max_pages && lp * a.page_tokens < sq.len ? (uint32_t)__ldg(table + lp) : 0xFFFFFFFFu;
        };
        /* Position of the group's first token in its sequence. */
        auto position = [&](uint32_t i, int gr, uint32_t lp) -> uint32_t {
            const uint32_t v = v_begin + i * TS + gr * 16;
            return lp * a.page_tokens + (v - a.page_of(v) * a.page_tokens);
        };
        /* Starts the copies of step i into ring slot st; whether the step has
         * every one of its tokens.  Tokens that the mask drops become zeros. */
        auto fetch = [&](uint32_t st, uint32_t i, const uint32_t *lp, const uint32_t *ph) -> bool {
            const uint32_t dst = ring_a + st * C::kStage;
            constexpr int CPR = C::kRow / 16, N = 16 * CPR;              /* 16-byte chunks of a row, of the group */
            bool whole = true;
            #pragma unroll
            for (int gr = 0; gr < GR; gr++) {
                const bool ok = ph[gr] < a.n_pages;
                const uint32_t pos = ok ? position(i, gr, lp[gr]) : 0u;
                const uint32_t off = ok ? pos - lp[gr] * a.page_tokens : 0u;
                const bool all = ok && pos >= sq.start && pos + 16 <= sq.len;
                whole = whole && all;
                const size_t row0 = (((size_t)(ok ? ph[gr] : 0u) * 2) * a.n_kv_heads + head) * a.page_tokens + off;
                const uint8_t *k = static_cast<const uint8_t *>(a.pool) + row0 * C::kRow + lane * 16;
                const uint8_t *v = k + v_off;
                const uint32_t to = dst + gr * 16 * kPitch;
                if (all) {
                    #pragma unroll
                    for (int c0 = 0; c0 < N; c0 += 32) {
                        const uint32_t c = c0 + lane;
                        if (N % 32 != 0 && c >= (uint32_t)N) continue;
                        const uint32_t d = to + (c / CPR) * kPitch + (c % CPR) * 16;
                        cp_async16(d, k + c0 * 16);
                        cp_async16(d + TS * kPitch, v + c0 * 16);
                    }
                    if (kQ8 && lane < 8) {                               /* 16 scales of K, 16 of V */
                        const float *sp = a.scales + row0 + (lane >> 2) * (size_t)a.n_kv_heads * a.page_tokens + (lane & 3) * 4;
                        cp_async16(dst + 2 * TS * kPitch + ((lane >> 2) * TS + gr * 16 + (lane & 3) * 4) * 4, sp);
                    }
                } else {
                    const uint32_t lo = pos < sq.start ? sq.start - pos : 0u;    /* tokens [lo, hi) of the group are kept */
                    const uint32_t hi = !ok || pos >= sq.len ? 0u : (sq.len - pos < 16u ? sq.len - pos : 16u);
                    #pragma unroll 1
                    for (uint32_t c = lane; c < (uint32_t)N; c += 32) {
                        const uint32_t row = c / CPR, d = to + row * kPitch + (c % CPR) * 16;
                        const uint32_t bytes = row >= lo && row < hi ? 16u : 0u;
                        cp_async16_part(d, k + (c - lane) * 16, bytes);
                        cp_async16_part(d + TS * kPitch, v + (c - lane) * 16, bytes);
                    }
                    if (kQ8 && lane < 8) {
                        const uint32_t tk = (lane & 3) * 4;
                        const uint32_t n = hi > tk ? (hi - tk < 4u ? hi - tk : 4u) : 0u;
                        const float *sp = a.scales + row0 + (lane >> 2) * (size_t)a.n_kv_heads * a.page_tokens + tk;
                        cp_async16_part(dst + 2 * TS * kPitch + ((lane >> 2) * TS + gr * 16 + tk) * 4, sp, n * 4);
                    }
                }
            }
            return whole;
        };

        /* The copies run kStages - 1 steps ahead, the pages they need a step
         * and the list entries two steps ahead of that. */
        uint32_t fi = sb + (solo ? 0u : warp);               /* next step to fetch */
        uint32_t lpA[GR], phA[GR], lpB[GR];
        #pragma unroll
        for (int gr = 0; gr < GR; gr++) { lpA[gr] = entry(fi, gr); lpB[gr] = entry(fi + stride, gr); }
        #pragma unroll
        for (int gr = 0; gr < GR; gr++) phA[gr] = mapped(lpA[gr]);
        uint32_t whole_slots = 0;                            /* bit per ring slot */
        auto advance = [&](uint32_t st) {
            uint32_t lpC[GR], phB[GR];
            #pragma unroll
            for (int gr = 0; gr < GR; gr++) { lpC[gr] = entry(fi + 2 * stride, gr); phB[gr] = mapped(lpB[gr]); }
            whole_slots &= ~(1u << st);
            if (fi < se && fetch(st, fi, lpA, phA)) whole_slots |= 1u << st;
            cp_commit();
            #pragma unroll
            for (int gr = 0; gr < GR; gr++) { lpA[gr] = lpB[gr]; phA[gr] = phB[gr]; lpB[gr] = lpC[gr]; }
            fi += stride;
        };
        #pragma unroll
        for (int st = 0; st < C::kStages - 1; st++) advance(st);

        /* ---- queries: B operands (8 heads a tile); heads past the group are zero ---- */
        uint32_t qb[HT][KB][2];
        float sc[HT][2];                                     /* log2 scale of heads 2j, 2j + 1 */
        #pragma unroll
        for (int t = 0; t < HT; t++) {
            const uint32_t r = t * 8 + g;
            const uint16_t *qp = a.q + (size_t)seq * a.q_stride + (size_t)query_head(r < rows ? r : 0u) * D;
            #pragma unroll
            for (int b = 0; b < KB; b++) {
                if (kQ8) {                                   /* values 4j .. 4j+3 of the block */
                    const uint2 w = r < rows ? __ldg(reinterpret_cast<const uint2 *>(qp + b * 16 + 4 * j)) : make_uint2(0u, 0u);
                    qb[t][b][0] = w.x; qb[t][b][1] = w.y;
                } else {
                    qb[t][b][0] = r < rows ? __ldg(reinterpret_cast<const uint32_t *>(qp + b * 16 + 2 * j)) : 0u;
                    qb[t][b][1] = r < rows ? __ldg(reinterpret_cast<const uint32_t *>(qp + b * 16 + 8 + 2 * j)) : 0u;
                }
            }
            sc[t][0] = sc[t][1] = a.scale_log2;
            if (kQ8) {
                /* to fp16 by a power of two that brings the head's largest
                 * value to [2^14, 2^15); the scores' factor takes it back */
                float top = 0.0f;
                #pragma unroll
                for (int b = 0; b < KB; b++) {
                    #pragma unroll
                    for (int h = 0; h < 2; h++) top = fmaxf(top, fmaxf(fabsf(bf16_lo(qb[t][b][h])), fabsf(bf16_hi(qb[t][b][h]))));
                }
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
                int e = (int)(__float_as_uint(top) >> 23) - 127;      /* floor(log2(top)); Inf: 128 */
                e = e < -100 ? -100 : e > 127 ? 127 : e;
                const float f = pow2f(14 - e);
                #pragma unroll
                for (int b = 0; b < KB; b++) {
                    #pragma unroll
                    for (int h = 0; h < 2; h++) qb[t][b][h] = pack_f16(bf16_lo(qb[t][b][h]) * f, bf16_hi(qb[t][b][h]) * f);
                }
                const float back = a.scale_log2 * pow2f(e - 14);
                sc[t][0] = __shfl_sync(0xFFFFFFFFu, back, 8 * j);
                sc[t][1] = __shfl_sync(0xFFFFFFFFu, back, 8 * j + 4);
            }
        }

        float o[KB][HT][4];
        #pragma unroll
        for (int b = 0; b < KB; b++)
            #pragma unroll
            for (int t = 0; t < HT; t++) o[b][t][0] = o[b][t][1] = o[b][t][2] = o[b][t][3] = 0.0f;
        float m[HT][2], l[HT][2];
        /* 8-bit pools: the fp16 weights are probability x V scale x unit.  The
         * unit is a power of two that brought the largest weight of some step
         * to [2^7, 2^8); it falls when a weight would pass 2^15 (`lim`) and is
         * set anew when a maximum grows, so a weight keeps its 11 bits down to
         * 2^-22 of the largest one that still counts. */
        float unit[HT][2], lim[HT][2];
        #pragma unroll
        for (int t = 0; t < HT; t++)
            #pragma unroll
            for (int h = 0; h < 2; h++) { m[t][h] = -INFINITY; l[t][h] = 0.0f; unit[t][h] = 1.0f; lim[t][h] = 0.0f; }

        uint32_t slot = 0;
        for (uint32_t i = sb + (solo ? 0u : warp); i < se; i += stride) {
            advance(slot == 0 ? C::kStages - 1 : slot - 1);              /* refill the slot that the last step freed */
            cp_wait<C::kStages - 1>();
            __syncwarp();
            const uint32_t stage = ring_a + slot * C::kStage;
            const float *scp = reinterpret_cast<const float *>(ring + slot * C::kStage + 2 * TS * kPitch);
            const bool whole = (whole_slots >> slot) & 1u;

            /* scores: rows = tokens g, g + 8 of a group, columns = heads 2j, 2j + 1 */
            float s[GR][HT][4];
            #pragma unroll
            for (int gr = 0; gr < GR; gr++) {
                #pragma unroll
                for (int t = 0; t < HT; t++) s[gr][t][0] = s[gr][t][1] = s[gr][t][2] = s[gr][t][3] = 0.0f;
                #pragma unroll
                for (int b = 0; b < C::kRow / 32; b++) {
                    uint32_t r[4];
                    ldsm4(stage + k_lane + gr * 16 * kPitch + b * 32, r);
                    if (kQ8) {
                        #pragma unroll
                        for (int h = 0; h < 2; h++) {
                            uint32_t f[4];
                            widen<DT, false>(r[2 * h], f[0], f[2]);
                            widen<DT, false>(r[2 * h + 1], f[1], f[3]);
                            #pragma unroll
                            for (int t = 0; t < HT; t++) mma16816<true>(s[gr][t], f, qb[t][2 * b + h][0], qb[t][2 * b + h][1]);
                        }
                    } else {
                        #pragma unroll
                        for (int t = 0; t < HT; t++) mma16816<false>(s[gr][t], r, qb[t][b][0], qb[t][b][1]);
                    }
                }
            }
            bool grow = false;
            #pragma unroll
            for (int gr = 0; gr < GR; gr++) {
                float ks0 = 1.0f, ks1 = 1.0f;
                if (kQ8) { ks0 = scp[gr * 16 + g]; ks1 = scp[gr * 16 + 8 + g]; }
                #pragma unroll
                for (int t = 0; t < HT; t++) {
                    s[gr][t][0] *= ks0 * sc[t][0]; s[gr][t][1] *= ks0 * sc[t][1];
                    s[gr][t][2] *= ks1 * sc[t][0]; s[gr][t][3] *= ks1 * sc[t][1];
                }
                if (!whole) {
                    const uint32_t lp = entry(i, gr);
                    const bool in = mapped(lp) < a.n_pages;
                    const uint32_t pos = in ? position(i, gr, lp) + g : 0u;
                    #pragma unroll
                    for (int t = 0; t < HT; t++) {
                        if (!in || pos >= sq.len || pos < sq.start) s[gr][t][0] = s[gr][t][1] = -INFINITY;
                        if (!in || pos + 8 >= sq.len || pos + 8 < sq.start) s[gr][t][2] = s[gr][t][3] = -INFINITY;
                    }
                }
                #pragma unroll
                for (int t = 0; t < HT; t++)
                    #pragma unroll
                    for (int h = 0; h < 2; h++) grow = grow || fmaxf(s[gr][t][h], s[gr][t][2 + h]) > m[t][h] + kGrow;
            }
            if (__any_sync(0xFFFFFFFFu, grow)) {
                #pragma unroll
                for (int t = 0; t < HT; t++) {
                    #pragma unroll
                    for (int h = 0; h < 2; h++) {
                        float mx = m[t][h];
                        #pragma unroll
                        for (int gr = 0; gr < GR; gr++) mx = fmaxf(mx, fmaxf(s[gr][t][h], s[gr][t][2 + h]));
                        #pragma unroll
                        for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, d));
                        const float f = mx == -INFINITY ? 1.0f : ex2(m[t][h] - mx);
                        m[t][h] = mx;
                        l[t][h] *= f;
                        lim[t][h] = 0.0f;
                        #pragma unroll
                        for (int b = 0; b < KB; b++) { o[b][t][h] *= f; o[b][t][2 + h] *= f; }
                    }
                }
            }
            #pragma unroll
            for (int t = 0; t < HT; t++) {
                #pragma unroll
                for (int h = 0; h < 2; h++) {
                    const float mz = m[t][h] == -INFINITY ? 0.0f : m[t][h];
                    #pragma unroll
                    for (int gr = 0; gr < GR; gr++) {
                        s[gr][t][h] = ex2(s[gr][t][h] - mz);
                        s[gr][t][2 + h] = ex2(s[gr][t][2 + h] - mz);
                        l[t][h] += s[gr][t][h] + s[gr][t][2 + h];
                    }
                }
            }
            if (kQ8) {
                bool over = false;
                #pragma unroll
                for (int gr = 0; gr < GR; gr++) {
                    const float vs0 = scp[TS + gr * 16 + g], vs1 = scp[TS + gr * 16 + 8 + g];
                    #pragma unroll
                    for (int t = 0; t < HT; t++) {
                        #pragma unroll
                        for (int h = 0; h < 4; h++) {        /* a masked token's scale may be NaN */
                            const float w = s[gr][t][h] * (h < 2 ? vs0 : vs1);
                            s[gr][t][h] = !whole && s[gr][t][h] == 0.0f ? 0.0f : w;
                            over = over || s[gr][t][h] > lim[t][h & 1];
                        }
                    }
                }
                if (__any_sync(0xFFFFFFFFu, over)) {
                    #pragma unroll
                    for (int t = 0; t < HT; t++) {
                        #pragma unroll
                        for (int h = 0; h < 2; h++) {
                            float top = 0.0f;
                            #pragma unroll
                            for (int gr = 0; gr < GR; gr++) top = fmaxf(top, fmaxf(s[gr][t][h], s[gr][t][2 + h]));
                            #pragma unroll
                            for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
                            if (top > lim[t][h]) {
                                int e = (int)(__float_as_uint(top) >> 23) - 127;
                                e = e < -119 ? -119 : e > 119 ? 119 : e;
                                const float nu = pow2f(7 - e), f = nu / unit[t][h];
                                unit[t][h] = nu;
                                lim[t][h] = pow2f(e + 8);
                                #pragma unroll
                                for (int b = 0; b < KB; b++) { o[b][t][h] *= f; o[b][t][2 + h] *= f; }
                            }
                        }
                    }
                }
            }
            #pragma unroll
            for (int gr = 0; gr < GR; gr++) {
                uint32_t p0[HT], p1[HT], q0[HT], q1[HT];     /* weights as B operands; bf16: low digits in q */
                #pragma unroll
                for (int t = 0; t < HT; t++) {
                    const float *w = s[gr][t];
                    if (kQ8) {
                        p0[t] = transpose8(pack_f16(w[0] * unit[t][0], w[1] * unit[t][1]));
                        p1[t] = transpose8(pack_f16(w[2] * unit[t][0], w[3] * unit[t][1]));
                    } else {
                        const uint32_t h0 = pack_bf16(w[0], w[1]), h1 = pack_bf16(w[2], w[3]);
                        p0[t] = transpose8(h0);
                        p1[t] = transpose8(h1);
                        q0[t] = transpose8(pack_bf16(w[0] - bf16_lo(h0), w[1] - bf16_hi(h0)));
                        q1[t] = transpose8(pack_bf16(w[2] - bf16_lo(h1), w[3] - bf16_hi(h1)));
                    }
                }
                #pragma unroll
                for (int b = 0; b < C::kRow / 32; b++) {
                    uint32_t r[4];
                    ldsm4t(stage + TS * kPitch + v_lane + gr * 16 * kPitch + b * 32, r);
                    if (kQ8) {
                        #pragma unroll
                        for (int h = 0; h < 2; h++) {
                            uint32_t f[4];
                            widen<DT, true>(r[2 * h], f[0], f[1]);
                            widen<DT, true>(r[2 * h + 1], f[2], f[3]);
                            #pragma unroll
                            for (int t = 0; t < HT; t++) mma16816<true>(o[2 * b + h][t], f, p0[t], p1[t]);
                        }
                    } else {
                        #pragma unroll
                        for (int t = 0; t < HT; t++) {
                            mma16816<false>(o[b][t], r, p0[t], p1[t]);
                            mma16816<false>(o[b][t], r, q0[t], q1[t]);
                        }
                    }
                }
            }
            __syncwarp();                                    /* the slot may be refilled */
            slot = slot + 1 == C::kStages ? 0 : slot + 1;
        }
        cp_wait<0>();
        __syncwarp();

        /* ---- join the warps (a short item has one) ---- */
        #pragma unroll
        for (int t = 0; t < HT; t++) {
            #pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint32_t r = t * 8 + 2 * j + h;
                #pragma unroll
                for (int d = 4; d < 32; d <<= 1) l[t][h] += __shfl_xor_sync(0xFFFFFFFFu, l[t][h], d);
                if (g == 0) { s_ml[warp][r][0] = m[t][h]; s_ml[warp][r][1] = l[t][h]; }
                float *dst = join(warp) + r * kJoin;
                const float back = kQ8 ? 1.0f / unit[t][h] : 1.0f;
                if (r < rows) {
                    #pragma unroll
                    for (int b = 0; b < KB; b++) {
                        if (kQ8) {                           /* values 2g, 2g + 1 of the block */
                            *reinterpret_cast<float2 *>(dst + b * 16 + 2 * g) = make_float2(o[b][t][h] * back, o[b][t][2 + h] * back);
                        } else {                             /* g, g + 8 */
                            dst[b * 16 + g] = o[b][t][h];
                            dst[b * 16 + 8 + g] = o[b][t][2 + h];
                        }
                    }
                }
            }
        }
        if (solo) __syncwarp(); else __syncthreads();
        const uint32_t w0 = solo ? warp : 0u, w1 = solo ? warp + 1 : (uint32_t)kWarps;
        const uint32_t part = 2 * blockIdx.x + (sb > 0 ? 0u : 1u);
        float *po = a.part_o + (size_t)part * 16 * D;
        float *pml = a.part_ml + (size_t)part * 32;
        auto finish = [&](uint32_t r, uint32_t d, float M, float L, const float4 &acc) {
            const float inv = L == 0.0f ? 0.0f : 1.0f / L;
            const size_t row = (size_t)seq * a.n_q_heads + query_head(r);
            *reinterpret_cast<uint2 *>(a.out + row * D + d) =
                make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
            if (a.lse && d == 0) a.lse[row] = (M + log2f(L)) * kLn2;
        };
        /* weight of a part with maximum pm and sum pl; a part without tokens has none */
        auto weight = [&](float pm, float pl, float M) -> float { return pm == -INFINITY && pl == 0.0f ? 0.0f : ex2(pm - M); };
        for (uint32_t c = solo ? lane : tid; c < rows * (D / 4); c += solo ? 32u : (uint32_t)kThreads) {
            const uint32_t r = c / (D / 4), d = (c % (D / 4)) * 4;
            float M = -INFINITY;
            for (uint32_t w = w0; w < w1; w++) M = fmaxf(M, s_ml[w][r][0]);
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            float L = 0.0f;
            for (uint32_t w = w0; w < w1; w++) {
                const float f = weight(s_ml[w][r][0], s_ml[w][r][1], M);
                const float4 v = *reinterpret_cast<const float4 *>(join(w) + r * kJoin + d);
                L += s_ml[w][r][1] * f;
                acc.x += v.x * f; acc.y += v.y * f; acc.z += v.z * f; acc.w += v.w * f;
            }
            if (cut) {
                __stcg(reinterpret_cast<float4 *>(po + r * D + d), acc);
                if (d == 0) __stcg(reinterpret_cast<float2 *>(pml + 2 * r), make_float2(M, L));
            } else {
                finish(r, d, M, L, acc);
            }
        }
        if (solo) { __syncwarp(); continue; }
        if (cut) {
            /* The CTA that finishes an item last joins its parts, in order. */
            const uint32_t first = (uint32_t)((item_x + kItemCost) / Q), last = (uint32_t)((item_end - 1) / Q);
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
                        const float f = weight(ml.x, ml.y, M);
                        L += ml.y * f;
                        acc.x += v.x * f; acc.y += v.y * f; acc.z += v.z * f; acc.w += v.w * f;
                    }
                    finish(r, d, M, L, acc);
                }
            }
        }
        __syncthreads();                                     /* the rings and s_ml are free again */
    }
}

}  // namespace ct_gqa
