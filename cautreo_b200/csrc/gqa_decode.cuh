/*
 * gqa_decode.cuh -- decode attention of one new token per sequence over a
 * paged cache with K and V per head (pool [page][K, V][kv head][slot][dim]),
 * over every page of the window or over the pages listed for each kv head.
 *
 * Math (sequence s, query head h of kv head c, tokens t that the mask keeps):
 *   x_t = scale * q_h . k_t,  out_h = sum_t softmax(x)_t v_t,  lse_h = ln sum_t exp x_t
 * as one pass over the tokens with a running maximum and sum in the log2
 * domain; a maximum is only followed when it grows by more than 2^3, so the
 * accumulators are rescaled a few times per sequence.
 *
 * Bound: HBM.  A token of a head is 4 D bytes (bf16; 2 (D + 4) in 8 bits) for
 * 4 G D flops, G <= 16 query heads sharing it: at most 16 flops a byte (31 in
 * 8 bits), a sixteenth (an eighth) of the ridge of the tensor cores.  So K and V go through cp.async into shared
 * memory and ldmatrix into mma.sync m16n8k16 with 16 tokens (for the scores)
 * or 16 values of a head (for the output) as the rows and 8 query heads of
 * the group as the columns: a group of up to 8 heads wastes nothing on rows,
 * 9 to 16 take two column tiles over the same K and V fragments, more run as
 * further items.  Scores come out as [token][head] and are needed as
 * [token][head] operands: two movmatrix per 16 tokens.
 * Measured, 8 kv heads of 4 query heads, 128 values: 32 sequences of 4096
 * tokens, bf16 95 us (5.6 TB/s), int8 54 us (5.1 TB/s); 64 of 8192 bf16 350 us
 * (6.1 TB/s), int8 193 (5.7); one of 777 tokens 8.1 us, of 64 (which no two
 * CTAs share) 4.4, of none 4.1.
 *
 * bf16 pools: probabilities enter as two bf16 digits (one would add an error
 * as large as the rounding of the output).  8-bit pools: codes are widened to
 * fp16 (exact), queries are brought to fp16 by a power of two a head (exact
 * down to 2^-29 of the head's largest value), and probability x V scale is
 * one fp16 digit (11 bits) in a running power-of-two unit; see `unit`.
 *
 * Split: an item is a (sequence, kv head, group of 16 heads); a step of it
 * TS tokens.  The steps of the whole batch lie end to end, each item with
 * kItemCost steps of overhead, and each CTA takes an equal range; when there
 * are fewer than half as many items as CTAs, every CTA takes one part of one
 * item instead.  Either is found from the device lengths at entry, so no
 * planning launch precedes the kernel.  An item of a few steps is one warp's;
 * the warps of a CTA share longer ones.  Each warp has its own ring of copies
 * that runs ahead across its items, and its own (max, sum, out), joined
 * through shared memory; an item cut between CTAs leaves fp32 partials that
 * the CTA finishing last joins in index order.
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
constexpr float kGrow = 3.0f;           /* log2 growth of a maximum that is followed */
constexpr float kNoMax = -3.402823466e38f;  /* maximum of no tokens: finite, so that no difference of maxima is NaN */
constexpr uint32_t kItemCost = 4;       /* steps that an item's start and end are counted as */
constexpr uint32_t kWhole = 32;         /* longest item, start and end counted, that is never cut between CTAs: 64
                                         * sequences of 300 tokens, 8 kv heads, bf16 x 128 24.8 -> 20.3 us */
constexpr uint32_t kSoloMost = 16;      /* longest item of one warp: longer ones would leave the others idle at the end */
constexpr uint32_t kSoloCost = 3;       /* start and end of an item, in steps of one warp, */
constexpr uint32_t kShareCost = 10;     /* and of one that the warps share */
constexpr uint32_t kFan = 16;           /* workers whose parts are joined at a time, when an item has more than 2 kFan */

/* Tokens of a warp's step (2 to 17 KB of K and V), steps in its ring, and the
 * CTAs that an SM shall hold.
 * Rows of up to 128 bytes take 32 tokens: the instructions that a step costs
 * whatever its size count half, and a long batch, which runs at the power
 * limit, keeps a higher clock (int8 x 128, 256 sequences of 256 tokens 39.5
 * -> 34.6 us, 64 of 16384 ragged, for a second, 217 -> 209; pages of 16, two
 * a step, 77 -> 79).
 * What bounds a long batch is how evenly the SMs share the memory, and that
 * gets worse with the copies in flight: from 100 to 150 KB an SM hides the
 * latency, more lets the SMs nearest to the memory take more than their part.
 * So rings have two steps, and CTAs that would bring more than kInFlight are
 * kept out (32 sequences of 4096 tokens, 8 kv heads, bf16: x 192 143 -> 135
 * us, x 256 186 -> 181; x 128 208 -> 140 KB, 16 sequences 52.0 -> 51.0).
 * Rows of 64 bytes or fewer are bound by their instructions and gain from a
 * third step (8-bit x 64, 16 x 4096 tokens 24.7 -> 22.2 us) and a third CTA,
 * which limits them to 168 registers. */
constexpr int kInFlight = 156 * 1024;
template <int D, int DT, int HT> struct Cfg {
    static constexpr int kElt = DT == CT_KV_BF16 ? 2 : 1;
    static constexpr int kRow = D * kElt;
    static constexpr int TS = kRow <= 128 ? 32 : 16;
    static constexpr int kStages = kRow <= 64 ? 3 : 2;
    static constexpr int kMinB = HT > 1 || kRow > 128 ? 1 : kRow <= 64 ? 3 : 2;
    static constexpr int kPitch = kRow + 16;                  /* odd number of 16-B units: conflict-free ldmatrix */
    static constexpr int kScaleBytes = DT == CT_KV_BF16 ? 0 : TS * 8;
    static constexpr int kStage = 2 * TS * kPitch + kScaleBytes;
    static constexpr int kRing = kWarps * kStages * kStage;
    /* Queries as operands: in registers, or (2 D / 16 registers a tile would
     * spill) in shared memory behind the ring, a copy for each warp. */
    static constexpr int kQPitch = 2 * D + 16;
    static constexpr int kQBytes = kWarps * HT * 8 * kQPitch;
    static constexpr bool kQueriesInSmem = HT * D >= 192;
    static constexpr int kUsed = kRing + (kQueriesInSmem ? kQBytes : 0);
    static constexpr int kMost = kRow <= 64 ? 32 : kRing < kInFlight ? kInFlight / kRing : 1;
    static constexpr int kShare = 227 * 1024 / (kMost + 1);      /* as much as keeps one CTA more out */
    static constexpr int kSmem = kUsed > kShare ? kUsed : kShare;
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
CT_DEV float rcp(float x) {
    float y;
    asm("rcp.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
CT_DEV float lg2(float x) {
    float y;
    asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
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
CT_DEV float inverse_pow2(float x) { return __uint_as_float(0x7F000000u - __float_as_uint(x)); }
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
    uint32_t pages;                                          /* of the whole sequence, at most max_pages */
    uint32_t steps;
};
template <int TS> CT_DEV Seq sequence(const ct_gqa_args_t &a, uint32_t s) {
    Seq r;
    const int32_t n = a.seq_lens[s];
    const uint32_t cap = a.max_pages * a.page_tokens;
    r.len = n < 0 ? 0u : ((uint32_t)n > cap ? cap : (uint32_t)n);
    r.start = a.window && r.len > a.window ? r.len - a.window : 0u;
    r.n_list = 0;
    r.pages = r.len ? a.page_of(r.len - 1) + 1 : 0u;
    uint32_t v;                                              /* tokens to step over */
    if (a.picked) {                                          /* listed pages: as many as the window has, at most */
        const uint32_t have = r.len ? r.pages - a.page_of(r.start) : 0u;
        r.n_list = have < a.n_pick ? have : a.n_pick;
        v = r.n_list * a.page_tokens;
    } else {
        v = r.len - (r.start & ~(TS - 1u));           /* whole steps: pages of a multiple of TS are not straddled */
    }
    const uint32_t st = (v + TS - 1) / TS;
    r.steps = st ? st : 1u;                                  /* an empty item still writes its zeros */
    return r;
}

/* HT: column tiles of 8 query heads.  FEW: fewer than half as many items as
 * CTAs, each CTA takes a part of one; this form has no more code than that
 * needs, since a call of a few microseconds runs every line of it from a cold
 * instruction cache. */
template <int D, int DT, int HT, bool FEW>
__global__ void __launch_bounds__(kThreads, Cfg<D, DT, HT>::kMinB) k_gqa_decode(const ct_gqa_args_t a) {
    using C = Cfg<D, DT, HT>;
    constexpr int TS = C::TS, GR = TS / 16, kPitch = C::kPitch, KB = D / 16, S = C::kStages;
    constexpr int kHeads = 8 * HT;
    constexpr bool kQ8 = DT != CT_KV_BF16;
    constexpr uint32_t kLeast = 128 / TS;                    /* least steps of a part: one a warp or two */
    /* a segment's end: each warp leaves its [head][value] sums in the ring slot
     * that it consumed last, all values at once or half of them at a time */
    constexpr int kJoinCols = kHeads * (D + 4) * 4 <= C::kStage ? D : D / 2;
    constexpr int kJoin = kJoinCols + 4;                     /* pitch: the lanes' writes fall in distinct banks */
    static_assert(kHeads * kJoin * 4 <= C::kStage && kJoinCols % 16 == 0, "half the sums of a warp fit a slot");
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint32_t s_scan[kWarps];
    /* An end of the CTA's range: an item (and its ordinal in the batch), a step
     * of it, the first and last worker that hold steps of it. */
    struct End { uint32_t seq, head, tile, step, first, last, ordinal; };
    __shared__ End s_end[2];
    __shared__ float s_ml[kWarps][kHeads][2];
    __shared__ uint32_t s_free[kWarps], s_last;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, j = lane & 3;
    const uint32_t HV = a.n_kv_heads * a.n_tiles;
    ct_gqa_enter();

    /* ---- this CTA's range of steps: from s_end[0] to before s_end[1] ---- */
    auto end_at = [&](uint32_t s, uint32_t item, uint32_t step, uint32_t first, uint32_t last) -> End {
        const uint32_t head = item / a.n_tiles;
        return {s, head, item - head * a.n_tiles, step, first, last, s * HV + item};
    };
    if (FEW) {                                               /* each warp for itself; the last barrier shares the result */
        uint32_t sum = 0, before = 0;
        #pragma unroll 1
        for (uint32_t s = lane; s < a.n_seq; s += 32) sum += sequence<TS>(a, s).steps;
        sum = __reduce_add_sync(0xFFFFFFFFu, sum);
        /* Parts of an item: as many as there are CTAs for, but with 9 to 16
         * heads, whose sums are long to join, few where a part would be short:
         * none of up to 256 tokens, else about as many as make a part's steps
         * and the join take equal time (4 kv heads of 16 query heads, bf16 x
         * 256: 4000 tokens 30.4 -> 24.0 us; 30 sequences of 239 tokens, 1 kv
         * head, 14.4 -> 11.9). */
        const uint32_t spare = gridDim.x - a.n_seq * HV;     /* every item's last part may be a short one */
        const uint32_t Q = max(kLeast, (uint32_t)__umul64hi((uint64_t)sum * HV + spare - 1, a.spare_magic));
        #pragma unroll 1
        for (uint32_t s0 = 0; s0 < a.n_seq; s0 += 32) {
            const uint32_t s = s0 + lane, steps = s < a.n_seq ? sequence<TS>(a, s).steps : 0u;
            uint32_t n = min((steps + Q - 1) / Q, a.most_parts);
            if (HT == 2) {
                n = min(n, max(2 * kFan, steps / 8));        /* more are joined in two rounds */
                if (steps <= kLeast * HT) n = min(steps, 1u);
                else if (n <= 2 * kFan) n = min(n, max(1u, (uint32_t)sqrtf((float)steps * (19.0f * TS / (HT * D)))));
            }
            uint32_t incl = n * HV;                          /* parts of the sequence's items */
            #pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, incl, o);
                if (lane >= (uint32_t)o) incl += y;
            }
            const uint32_t x = blockIdx.x - (before + incl - n * HV);
            if (warp == 0 && x < n * HV) {
                const uint32_t item = x / n, part = x - item * n, first = blockIdx.x - part, each = steps / n, over = steps - each * n;
                s_end[0] = end_at(s, item, part * each + min(part, over), first, first + n - 1);
                s_end[1].step = (part + 1) * each + min(part + 1, over);
            }
            before += __shfl_sync(0xFFFFFFFFu, incl, 31);
        }
        if (blockIdx.x >= before) return;
    } else {
        const uint32_t per = (a.n_seq + kThreads - 1) / kThreads;
        uint32_t sum = 0;
        #pragma unroll 1
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
        uint32_t before = 0, all = 0;
        #pragma unroll
        for (int w = 0; w < kWarps; w++) {
            if (w < (int)warp) before += s_scan[w];
            all += s_scan[w];
        }
        const uint64_t total = (uint64_t)all * HV, excl = (uint64_t)(before + incl - sum) * HV, next = excl + (uint64_t)sum * HV;
        const uint32_t Q = max(kLeast, (uint32_t)__umul64hi(total + gridDim.x - 1, a.worker_magic));
        const uint64_t x0 = (uint64_t)blockIdx.x * Q;
        if (x0 >= total) return;
        if (tid == 0 && x0 + Q >= total) s_end[1] = end_at(a.n_seq, 0u, 0u, 0u, 0u);
        #pragma unroll 1
        for (uint32_t b = 0; b < 2; b++) {                   /* where the range begins, where the next one does */
            const uint64_t x = x0 + b * Q;
            if (x < excl || x >= next) continue;
            uint64_t at = excl;
            uint32_t s = tid * per, width;
            #pragma unroll 1
            for (;; s++) {
                width = sequence<TS>(a, s).steps + kItemCost;
                if (x < at + (uint64_t)width * HV) break;
                at += (uint64_t)width * HV;
            }
            const uint32_t rel = (uint32_t)(x - at), item = rel / width;          /* below 2^32: see the plan */
            uint32_t in = rel - item * width;
            /* A short item goes to the later CTA as a whole: cutting it costs
             * both of them a shared start and end, and the join. */
            if (width <= kWhole) in = 0;
            const uint32_t step = in > kItemCost ? in - kItemCost : 0u;
            /* workers that hold steps of the item: from the one of its first
             * step (this one if the item begins here) to that of its last */
            const uint32_t here = blockIdx.x + b;
            s_end[b] = end_at(s, item, step, here - (step + Q - 1) / Q, here + (width - 1 - in) / Q);
        }
    }
    __syncthreads();
    const uint32_t range = FEW ? 1u : s_end[1].ordinal - s_end[0].ordinal + (s_end[1].step ? 1u : 0u);     /* items */
    if (range == 0) return;

    uint8_t *ring = smem + warp * (S * C::kStage);
    const uint32_t ring_a = smem_u32(ring);
    const size_t v_off = (size_t)a.n_kv_heads * a.page_tokens * C::kRow;
    /* ldmatrix lane offsets inside a stage */
    const uint32_t mi = lane >> 3, mr = lane & 7;
    const uint32_t k_lane = ((mi & 1) * 8 + mr) * kPitch + (mi >> 1) * 16;
    const uint32_t v_lane = kQ8 ? k_lane : ((mi >> 1) * 8 + mr) * kPitch + (mi & 1) * 16;

    /* A segment: the part of an item inside the range, and this warp's run of
     * its steps [wb, we). */
    struct Segment {
        uint32_t seq, head, tile;
        Seq sq;
        uint32_t sb, se, wb, we;
        bool solo;
    };
    /* The range's at-th item; called with at = 0, 1, 2, ... */
    auto segment = [&](Segment &z, uint32_t at) {
        bool next = at == 0;
        if (at == 0) {
            z.seq = s_end[0].seq;
            z.head = s_end[0].head;
            z.tile = s_end[0].tile;
        } else if (++z.tile == a.n_tiles) {
            z.tile = 0;
            if (++z.head == a.n_kv_heads) { z.head = 0; z.seq++; next = true; }
        }
        if (next) z.sq = sequence<TS>(a, z.seq);
        z.sb = at == 0 ? s_end[0].step : 0u;
        z.se = at + 1 == range && s_end[1].step ? s_end[1].step : z.sq.steps;
        const uint32_t n = z.se - z.sb;
        z.solo = false;
        if (!FEW) {
            /* A whole item is one warp's if there is nothing to share, or if the
             * range's whole items, handed out one by one, take less of the
             * warps' time so than shared. */
            const uint32_t items = range - (s_end[0].step ? 1u : 0u) - (s_end[1].step ? 1u : 0u), rounds = (items + kWarps - 1) / kWarps;
            z.solo = n == z.sq.steps && (n == 1 || (n <= kSoloMost && items > 1 &&
                                                    kWarps * rounds * (n + kSoloCost) <= items * (n + kShareCost)));
        }
        if (z.solo) {
            z.wb = z.sb;
            z.we = (at & (kWarps - 1)) == warp ? z.se : z.sb;
        } else {                                             /* n below 2^28: four times it fits */
            z.wb = z.sb + n * warp / kWarps;
            z.we = z.sb + n * (warp + 1) / kWarps;
        }
    };
    auto first_token = [&](const Seq &q) -> uint32_t { return a.picked ? 0u : (q.start & ~(TS - 1u)); };
    /* Logical page of the e-th page stepped over (0xFFFFFFFF: none). */
    auto entry = [&](const Segment &z, uint32_t e) -> uint32_t {
        if (!a.picked) return e;
        return e < z.sq.n_list ? (uint32_t)a.picked[((size_t)z.seq * a.n_kv_heads + z.head) * a.n_pick + e] : 0xFFFFFFFFu;
    };
    /* Its physical page (>= n_pages: nothing to read). */
    auto mapped = [&](const Segment &z, uint32_t lp) -> uint32_t {
        return lp < z.sq.pages ? (uint32_t)a.block_table[(size_t)z.seq * a.max_pages + lp] : 0xFFFFFFFFu;
    };

    /* ---- copies: S - 1 steps ahead of the arithmetic ----
     * Cursor of the next tokens to copy: their address, the slot in their page
     * and the page's slots [page_lo, page_hi) that the mask keeps.  Page
     * numbers are loaded 32 at a time, one a lane, 16 pages ahead. */
    Segment z = {}, pz = {};
    if (FEW) { segment(z, 0); pz = z; }
    uint32_t p_at = 0xFFFFFFFFu, left = 0, page_e = 0, off = 0, page_lo = 0, page_hi = 0;
    uint32_t turned = 0, lps = 0, phs = 0, lps_then = 0, phs_then = 0;       /* pages opened; logical, physical numbers */
    const uint8_t *kp = nullptr;
    const float *sp = nullptr;
    bool turn = false, done = false;
    uint32_t whole_slots = 0, fill = 0;                      /* bit per ring slot; slot of the next copies */
    const size_t page_bytes = 2 * v_off, page_rows = (size_t)2 * a.n_kv_heads * a.page_tokens;
    auto turn_page = [&]() {                                 /* opens the next page */
        const uint32_t i = turned & 31;
        if (i == 0 && turned) { lps = lps_then; phs = phs_then; }
        if (i == 16) { lps_then = entry(pz, page_e + 16 + lane); phs_then = mapped(pz, lps_then); }
        const uint32_t lp = __shfl_sync(0xFFFFFFFFu, lps, i), ph = __shfl_sync(0xFFFFFFFFu, phs, i);
        const bool ok = ph < a.n_pages;
        const uint32_t row = pz.head * a.page_tokens + off;  /* of the page */
        kp = static_cast<const uint8_t *>(a.pool) + (ok ? ph : 0u) * page_bytes + (size_t)row * C::kRow + lane * 16;
        if (kQ8)
            sp = a.scales + (ok ? ph : 0u) * page_rows + row + (lane >> 2) * (a.n_kv_heads * a.page_tokens) + (lane & 3) * 4;
        const uint32_t first = lp * a.page_tokens;
        page_lo = pz.sq.start > first ? pz.sq.start - first : 0u;
        page_hi = ok ? min(pz.sq.len - first, a.page_tokens) : 0u;
        page_e++;
        turned++;
        turn = false;
    };
    /* Starts the copies of this warp's next step (tokens that the mask drops
     * become zeros), then, if that was the last of its segment, looks for the
     * next segment and loads the numbers of its first pages. */
    auto advance = [&]() {
        if (left) {
            constexpr int CPR = C::kRow / 16, N = 16 * CPR;  /* 16-byte chunks of a row, of 16 tokens */
            const uint32_t to = ring_a + fill * C::kStage;
            const uint32_t to_s = to + 2 * TS * kPitch + ((lane >> 2) * TS + (lane & 3) * 4) * 4;
            if (turn) turn_page();
            bool whole = off >= page_lo && off + TS <= page_hi;
            if (whole) {
                const uint8_t *vp = kp + v_off;
                #pragma unroll
                for (int c0 = 0; c0 < GR * N; c0 += 32) {
                    const uint32_t c = c0 + lane;
                    if (GR * N % 32 != 0 && c >= (uint32_t)(GR * N)) continue;
                    const uint32_t d = to + (c / CPR) * kPitch + (c % CPR) * 16;
                    cp_async16(d, kp + c0 * 16);
                    cp_async16(d + TS * kPitch, vp + c0 * 16);
                }
                if (kQ8 && lane < 8) {                       /* scales of K, of V */
                    #pragma unroll
                    for (int gr = 0; gr < GR; gr++) cp_async16(to_s + gr * 64, sp + gr * 16);
                }
                off += TS;
                kp += TS * C::kRow;
                if (kQ8) sp += TS;
            } else {                                         /* 16 tokens at a time: across pages, or masked */
                whole = true;
                #pragma unroll 1
                for (uint32_t gr = 0; gr < (uint32_t)GR; gr++) {
                    if (turn || off == a.page_tokens) { if (!turn) off = 0; turn_page(); }
                    const uint32_t lo = page_lo > off ? page_lo - off : 0u;      /* tokens [lo, hi) are kept */
                    const uint32_t hi = page_hi > off ? min(page_hi - off, 16u) : 0u;
                    if (lo == 0 && hi == 16) {
                        #pragma unroll
                        for (int c0 = 0; c0 < N; c0 += 32) {
                            const uint32_t c = c0 + lane;
                            if (N % 32 != 0 && c >= (uint32_t)N) continue;
                            const uint32_t d = to + (gr * 16 + c / CPR) * kPitch + (c % CPR) * 16;
                            cp_async16(d, kp + c0 * 16);
                            cp_async16(d + TS * kPitch, kp + v_off + c0 * 16);
                        }
                        if (kQ8 && lane < 8) cp_async16(to_s + gr * 64, sp);
                    } else {
                        whole = false;
                        #pragma unroll 1
                        for (uint32_t c = lane; c < (uint32_t)N; c += 32) {
                            const uint32_t row = c / CPR, d = to + (gr * 16 + row) * kPitch + (c % CPR) * 16;
                            const uint32_t bytes = row >= lo && row < hi ? 16u : 0u;
                            cp_async16_part(d, kp + (c - lane) * 16, bytes);
                            cp_async16_part(d + TS * kPitch, kp + v_off + (c - lane) * 16, bytes);
                        }
                        if (kQ8 && lane < 8) {
                            const uint32_t tk = (lane & 3) * 4;
                            cp_async16_part(to_s + gr * 64, sp, (hi > tk ? min(hi - tk, 4u) : 0u) * 4);
                        }
                    }
                    off += 16;
                    kp += 16 * C::kRow;
                    if (kQ8) sp += 16;
                }
            }
            if (off == a.page_tokens) { off = 0; turn = true; }
            whole_slots = whole ? whole_slots | (1u << fill) : whole_slots & ~(1u << fill);
            fill = fill + 1 == S ? 0 : fill + 1;
            left--;
        }
        cp_commit();
        if (left == 0 && !done) {
            #pragma unroll 1
            do {
                if (++p_at == range) { done = true; break; }
                if (!FEW) segment(pz, p_at);
                left = pz.we - pz.wb;
            } while (left == 0);
            if (left) {
                const uint32_t v = first_token(pz.sq) + pz.wb * TS;
                page_e = a.page_of(v);
                off = v - page_e * a.page_tokens;
                lps = entry(pz, page_e + lane);
                phs = mapped(pz, lps);
                turned = 0;
                turn = true;
            }
        }
    };
    uint32_t slot = 0;                                       /* slot of the next step; the one before it is free */
    int prime = S;                                           /* the first call looks for a segment, S - 1 fill the ring */

    /* ---- arithmetic ---- */
    #pragma unroll 1
    for (uint32_t at = 0; at < range; at++) {
        if (!FEW) segment(z, at);
        if (z.solo && z.we == z.wb) continue;                /* another warp's */
        const uint32_t seq = z.seq, tile = z.tile, head = z.head;
        const uint32_t rows = a.group - tile * 16 < 16 ? a.group - tile * 16 : 16;
        const bool cut = z.sb > 0 || z.se < z.sq.steps;
        auto query_head = [&](uint32_t r) -> uint32_t {
            const uint32_t in_group = tile * 16 + r;
            return a.blocked ? head * a.group + in_group : in_group * a.n_kv_heads + head;
        };

        /* ---- queries: B operands (8 heads a tile); heads past the group are zero ---- */
        constexpr bool kQS = C::kQueriesInSmem;
        uint32_t qb[kQS ? 1 : HT][KB][2];
        uint8_t *qs = smem + C::kRing + warp * (kHeads * C::kQPitch);
        float sc[HT][2];                                     /* log2 scale of heads 2j, 2j + 1 */
        #pragma unroll
        for (int t = 0; t < HT; t++) {
            uint32_t (&qt)[KB][2] = qb[kQS ? 0 : t];
            const uint32_t r = t * 8 + g;
            const uint16_t *qp = a.q + (size_t)seq * a.q_stride + (size_t)query_head(r < rows ? r : 0u) * D;
            #pragma unroll
            for (int b = 0; b < KB; b++) {
                if (kQ8) {                                   /* values 4j .. 4j+3 of the block */
                    const uint2 w = r < rows ? *reinterpret_cast<const uint2 *>(qp + b * 16 + 4 * j) : make_uint2(0u, 0u);
                    qt[b][0] = w.x; qt[b][1] = w.y;
                } else {
                    qt[b][0] = r < rows ? *reinterpret_cast<const uint32_t *>(qp + b * 16 + 2 * j) : 0u;
                    qt[b][1] = r < rows ? *reinterpret_cast<const uint32_t *>(qp + b * 16 + 8 + 2 * j) : 0u;
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
                    for (int h = 0; h < 2; h++) top = fmaxf(top, fmaxf(fabsf(bf16_lo(qt[b][h])), fabsf(bf16_hi(qt[b][h]))));
                }
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
                int e = (int)(__float_as_uint(top) >> 23) - 127;      /* floor(log2(top)); Inf: 128 */
                e = e < -100 ? -100 : e > 127 ? 127 : e;
                const float f = pow2f(14 - e);
                #pragma unroll
                for (int b = 0; b < KB; b++) {
                    #pragma unroll
                    for (int h = 0; h < 2; h++) qt[b][h] = pack_f16(bf16_lo(qt[b][h]) * f, bf16_hi(qt[b][h]) * f);
                }
                const float back = a.scale_log2 * pow2f(e - 14);
                sc[t][0] = __shfl_sync(0xFFFFFFFFu, back, 8 * j);
                sc[t][1] = __shfl_sync(0xFFFFFFFFu, back, 8 * j + 4);
            }
            if (kQS) {
                #pragma unroll
                for (int b = 0; b < KB; b++) {
                    uint32_t *to = reinterpret_cast<uint32_t *>(qs + r * C::kQPitch + b * 32) + j;
                    to[0] = qt[b][0];
                    to[4] = qt[b][1];
                }
            }
        }
        if (kQS) __syncwarp();
        const uint32_t qs_a = smem_u32(qs) + mr * C::kQPitch + mi * 16;

        float o[KB][HT][4];
        #pragma unroll
        for (int b = 0; b < KB; b++)
            #pragma unroll
            for (int t = 0; t < HT; t++) o[b][t][0] = o[b][t][1] = o[b][t][2] = o[b][t][3] = 0.0f;
        float m[HT][2], l[HT][2];
        /* 8-bit pools: the fp16 weights are probability (at most 2^kGrow) x V
         * scale x unit, a power of two that brought the largest V scale of
         * some step to [2^11, 2^12) and falls when one would pass that; so a
         * weight is below 2^15, and keeps its 11 bits where its V scale is
         * 2^-25 of the largest or more. */
        float unit = 1.0f;
        bool blank = true, renew = true;                     /* blank: some head has seen no token yet, */
        uint32_t seen = 0;                                   /* bits of those that have */
        #pragma unroll
        for (int t = 0; t < HT; t++)
            #pragma unroll
            for (int h = 0; h < 2; h++) m[t][h] = l[t][h] = 0.0f;

        #pragma unroll 1
        for (uint32_t i = z.wb; i < z.we;) {
            advance();                                       /* refill the slot that the last step freed */
            if (prime) { prime--; continue; }
            cp_wait<S - 1>();
            __syncwarp();
            const uint32_t stage = ring_a + slot * C::kStage;
            const float *scp = reinterpret_cast<const float *>(ring + slot * C::kStage + 2 * TS * kPitch);

            /* scores: rows = tokens g, g + 8 of a group, columns = heads 2j, 2j + 1 */
            float s[GR][HT][4];
            #pragma unroll
            for (int gr = 0; gr < GR; gr++) {
                constexpr bool kTwo = KB > 4;                /* every other block apart: two chains of MMAs */
                float s2[HT][4];
                #pragma unroll
                for (int t = 0; t < HT; t++)
                    #pragma unroll
                    for (int h = 0; h < 4; h++) s[gr][t][h] = s2[t][h] = 0.0f;
                #pragma unroll
                for (int b = 0; b < KB; b += 2) {
                    uint32_t r[4], f[2][4], q[HT][4];
                    ldsm4(stage + k_lane + gr * 16 * kPitch + b * 16 * C::kElt, r);
                    if (kQ8) {
                        #pragma unroll
                        for (int h = 0; h < 2; h++) {
                            widen<DT, false>(r[2 * h], f[h][0], f[h][2]);
                            widen<DT, false>(r[2 * h + 1], f[h][1], f[h][3]);
                        }
                    } else {
                        #pragma unroll
                        for (int h = 0; h < 4; h++) f[0][h] = r[h];
                        ldsm4(stage + k_lane + gr * 16 * kPitch + (b + 1) * 32, f[1]);
                    }
                    #pragma unroll
                    for (int t = 0; t < HT; t++) {
                        if (kQS) {
                            ldsm4(qs_a + t * 8 * C::kQPitch + b * 32, q[t]);
                        } else {
                            q[t][0] = qb[kQS ? 0 : t][b][0]; q[t][1] = qb[kQS ? 0 : t][b][1];
                            q[t][2] = qb[kQS ? 0 : t][b + 1][0]; q[t][3] = qb[kQS ? 0 : t][b + 1][1];
                        }
                        mma16816<kQ8>(s[gr][t], f[0], q[t][0], q[t][1]);
                        mma16816<kQ8>(kTwo ? s2[t] : s[gr][t], f[1], q[t][2], q[t][3]);
                    }
                }
                #pragma unroll
                for (int t = 0; t < HT; t++)
                    #pragma unroll
                    for (int h = 0; h < 4; h++)
                        if (kTwo) s[gr][t][h] += s2[t][h];
            }
            /* log2 of the probabilities, up to the running maxima */
            float vs[GR][2];                                 /* V scales of tokens g, g + 8 */
            #pragma unroll
            for (int gr = 0; gr < GR; gr++) {
                if (kQ8) {
                    const float ks[2] = {scp[gr * 16 + g], scp[gr * 16 + 8 + g]};
                    vs[gr][0] = scp[TS + gr * 16 + g]; vs[gr][1] = scp[TS + gr * 16 + 8 + g];
                    #pragma unroll
                    for (int t = 0; t < HT; t++)
                        #pragma unroll
                        for (int h = 0; h < 4; h++) s[gr][t][h] *= ks[h >> 1];
                }
                #pragma unroll
                for (int t = 0; t < HT; t++)
                    #pragma unroll
                    for (int h = 0; h < 4; h++) s[gr][t][h] = fmaf(s[gr][t][h], sc[t][h & 1], -m[t][h & 1]);
            }
            if (!((whole_slots >> slot) & 1u)) {             /* some tokens are not to be attended */
                #pragma unroll
                for (int gr = 0; gr < GR; gr++) {
                    const uint32_t v = first_token(z.sq) + i * TS + gr * 16;
                    const uint32_t e = a.page_of(v), lp = entry(z, e);
                    const bool in = mapped(z, lp) < a.n_pages;
                    const uint32_t t0 = in ? lp * a.page_tokens + (v - e * a.page_tokens) + g : 0u;
                    #pragma unroll
                    for (int h = 0; h < 2; h++) {
                        if (in && t0 + 8 * h < z.sq.len && t0 + 8 * h >= z.sq.start) continue;
                        vs[gr][h] = 0.0f;                    /* it may be NaN */
                        #pragma unroll
                        for (int t = 0; t < HT; t++) s[gr][t][2 * h] = s[gr][t][2 * h + 1] = -INFINITY;
                    }
                }
            }
            float top = kNoMax;
            #pragma unroll
            for (int gr = 0; gr < GR; gr++)
                #pragma unroll
                for (int t = 0; t < HT; t++)
                    #pragma unroll
                    for (int h = 0; h < 4; h++) top = fmaxf(top, s[gr][t][h]);
            if (__any_sync(0xFFFFFFFFu, blank || top > kGrow)) {
                float by[HT][2];                             /* how far the maxima move */
                #pragma unroll
                for (int t = 0; t < HT; t++)
                    #pragma unroll
                    for (int h = 0; h < 2; h++) {
                        by[t][h] = (seen >> (2 * t + h)) & 1u ? 0.0f : -INFINITY;
                        #pragma unroll
                        for (int gr = 0; gr < GR; gr++) by[t][h] = fmaxf(by[t][h], fmaxf(s[gr][t][h], s[gr][t][2 + h]));
                    }
                #pragma unroll
                for (int d = 4; d < 32; d <<= 1)
                    #pragma unroll
                    for (int t = 0; t < HT; t++)
                        #pragma unroll
                        for (int h = 0; h < 2; h++) by[t][h] = fmaxf(by[t][h], __shfl_xor_sync(0xFFFFFFFFu, by[t][h], d));
                const uint32_t was = seen;
                blank = false;
                #pragma unroll
                for (int t = 0; t < HT; t++)
                    #pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const bool none = by[t][h] == -INFINITY;         /* still no token */
                        blank = blank || none;
                        by[t][h] = none ? 0.0f : by[t][h];
                        seen |= none ? 0u : 1u << (2 * t + h);
                        m[t][h] += by[t][h];
                        #pragma unroll
                        for (int gr = 0; gr < GR; gr++) { s[gr][t][h] -= by[t][h]; s[gr][t][2 + h] -= by[t][h]; }
                    }
                if (was) {                                   /* a head without tokens has no sums */
                    #pragma unroll
                    for (int t = 0; t < HT; t++)
                        #pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const float f = (was >> (2 * t + h)) & 1u ? ex2(-by[t][h]) : 1.0f;
                            l[t][h] *= f;
                            #pragma unroll
                            for (int b = 0; b < KB; b++) { o[b][t][h] *= f; o[b][t][2 + h] *= f; }
                        }
                }
            }
            #pragma unroll
            for (int gr = 0; gr < GR; gr++)
                #pragma unroll
                for (int t = 0; t < HT; t++)
                    #pragma unroll
                    for (int h = 0; h < 4; h++) {
                        s[gr][t][h] = ex2(s[gr][t][h]);
                        l[t][h & 1] += s[gr][t][h];
                    }
            if (kQ8) {
                float vm = 0.0f;
                #pragma unroll
                for (int gr = 0; gr < GR; gr++) vm = fmaxf(vm, fmaxf(vs[gr][0], vs[gr][1]));
                if (__any_sync(0xFFFFFFFFu, vm * unit >= 4096.0f || (renew && vm > 0.0f))) {
                    #pragma unroll
                    for (int d = 4; d < 32; d <<= 1) vm = fmaxf(vm, __shfl_xor_sync(0xFFFFFFFFu, vm, d));
                    int to = 11 - ((int)(__float_as_uint(vm) >> 23) - 127);
                    to = to < -120 ? -120 : to > 100 ? 100 : to;
                    const float f = pow2f(to) * inverse_pow2(unit);
                    unit = pow2f(to);
                    if (!renew) {
                        #pragma unroll
                        for (int t = 0; t < HT; t++)
                            #pragma unroll
                            for (int b = 0; b < KB; b++) { o[b][t][0] *= f; o[b][t][1] *= f; o[b][t][2] *= f; o[b][t][3] *= f; }
                    }
                    renew = false;
                }
                #pragma unroll
                for (int gr = 0; gr < GR; gr++) {
                    const float w0 = vs[gr][0] * unit, w1 = vs[gr][1] * unit;
                    #pragma unroll
                    for (int t = 0; t < HT; t++)
                        #pragma unroll
                        for (int h = 0; h < 4; h++) s[gr][t][h] *= h < 2 ? w0 : w1;
                }
            }
            #pragma unroll
            for (int gr = 0; gr < GR; gr++) {
                uint32_t p0[HT], p1[HT], q0[HT], q1[HT];     /* weights as B operands; bf16: low digits in q */
                #pragma unroll
                for (int t = 0; t < HT; t++) {
                    const float *w = s[gr][t];
                    if (kQ8) {
                        p0[t] = transpose8(pack_f16(w[0], w[1]));
                        p1[t] = transpose8(pack_f16(w[2], w[3]));
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
            slot = slot + 1 == S ? 0 : slot + 1;
            i++;
        }

        /* ---- join the warps (a short item has one) ---- */
        const uint32_t part = 2 * blockIdx.x + (z.sb > 0 ? 0u : 1u);
        float *po = a.part_o + (size_t)part * 16 * D;
        float *pml = a.part_ml + (size_t)part * 32;
        auto write = [&](uint32_t r, uint32_t d, float f, const float4 &v) {
            *reinterpret_cast<uint2 *>(a.out + ((size_t)seq * a.n_q_heads + query_head(r)) * D + d) =
                make_uint2(pack_bf16(v.x * f, v.y * f), pack_bf16(v.z * f, v.w * f));
        };
        const uint32_t freed = slot == 0 ? S - 1 : slot - 1;
        float *mine = reinterpret_cast<float *>(ring + freed * C::kStage);
        if (lane == 0) s_free[warp] = warp * (S * C::kStage) + freed * C::kStage;
        #pragma unroll
        for (int t = 0; t < HT; t++)
            #pragma unroll
            for (int h = 0; h < 2; h++) {
                #pragma unroll
                for (int d = 4; d < 32; d <<= 1) l[t][h] += __shfl_xor_sync(0xFFFFFFFFu, l[t][h], d);
                if (g == 0) { s_ml[warp][t * 8 + 2 * j + h][0] = (seen >> (2 * t + h)) & 1u ? m[t][h] : kNoMax; s_ml[warp][t * 8 + 2 * j + h][1] = l[t][h]; }
            }
        #pragma unroll
        for (int d0 = 0; d0 < D; d0 += kJoinCols) {
            #pragma unroll
            for (int t = 0; t < HT; t++) {
                #pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint32_t r = t * 8 + 2 * j + h;
                    float *dst = mine + r * kJoin;
                    const float back = kQ8 ? inverse_pow2(unit) : 1.0f;
                    if (r < rows) {
                        #pragma unroll
                        for (int b = 0; b < kJoinCols / 16; b++) {
                            const float *ob = o[d0 / 16 + b][t];
                            if (kQ8) {                       /* values 2g, 2g + 1 of the block */
                                *reinterpret_cast<float2 *>(dst + b * 16 + 2 * g) = make_float2(ob[h] * back, ob[2 + h] * back);
                            } else {                         /* g, g + 8 */
                                dst[b * 16 + g] = ob[h];
                                dst[b * 16 + 8 + g] = ob[2 + h];
                            }
                        }
                    }
                }
            }
            if (z.solo) __syncwarp(); else __syncthreads();
            #pragma unroll 1
            for (uint32_t c = z.solo ? lane : tid; c < rows * (kJoinCols / 4); c += z.solo ? 32u : (uint32_t)kThreads) {
                const uint32_t r = c / (kJoinCols / 4), dj = (c % (kJoinCols / 4)) * 4, d = d0 + dj;
                float M = s_ml[warp][r][0], L = s_ml[warp][r][1];
                float4 acc = *reinterpret_cast<const float4 *>(smem + s_free[warp] + (r * kJoin + dj) * 4);
                if (!z.solo) {
                    M = kNoMax;
                    #pragma unroll
                    for (int w = 0; w < kWarps; w++) M = fmaxf(M, s_ml[w][r][0]);
                    acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    L = 0.0f;
                    #pragma unroll
                    for (int w = 0; w < kWarps; w++) {
                        const float f = ex2(s_ml[w][r][0] - M);
                        const float4 v = *reinterpret_cast<const float4 *>(smem + s_free[w] + (r * kJoin + dj) * 4);
                        L += s_ml[w][r][1] * f;
                        acc.x += v.x * f; acc.y += v.y * f; acc.z += v.z * f; acc.w += v.w * f;
                    }
                }
                if (cut) {
                    __stcg(reinterpret_cast<float4 *>(po + r * D + d), acc);
                    if (d == 0) __stcg(reinterpret_cast<float2 *>(pml + 2 * r), make_float2(M, L));
                } else {
                    write(r, d, L == 0.0f ? 0.0f : rcp(L), acc);
                    if (a.lse && d == 0) a.lse[(size_t)seq * a.n_q_heads + query_head(r)] = (M + lg2(L)) * kLn2;
                }
            }
            if (z.solo) __syncwarp(); else __syncthreads();              /* the slots and s_ml are free again */
        }
        if (cut) {
            /* The CTA that finishes an item last joins its parts, in order.
             * An item of more than 2 kFan workers (few items in the batch)
             * is joined in two rounds: each aligned run of kFan workers by
             * its last one, into the run's first part, then the runs. */
            const End &end = s_end[FEW || z.sb > 0 ? 0 : 1];
            const uint32_t first = end.first, last = end.last;
            const bool tree = last - first >= 2 * kFan;
            uint32_t lo = first, hi = last, by = 1;
            if (tree) {
                lo = blockIdx.x & ~(kFan - 1);
                hi = min(lo + kFan - 1, last);
                lo = max(lo, first);
            }
            bool last_here = true;
            #pragma unroll 1
            for (int round = 0; last_here && round < (tree ? 2 : 1); round++) {
                /* three sets of counters: an item's, by its first worker; a
                 * run's, by its first worker, apart for the run that an item
                 * begins in (an earlier item may end in the same worker) */
                const uint32_t set = !tree || round ? 0u : lo == first ? 1u : 2u;
                uint32_t *counter = a.counters + set * gridDim.x + (set == 2 ? lo : first);
                const uint32_t n = by == 1 ? hi - lo + 1 : (last / kFan) - (first / kFan) + 1;
                __syncthreads();                             /* this CTA's part (or its run's) is written */
                if (tid == 0) {
                    __threadfence();
                    const uint32_t before = atomicAdd(counter, 1u);
                    s_last = before == n - 1 ? 1u : 0u;
                    if (s_last) { *counter = 0u; __threadfence(); }
                }
                __syncthreads();
                last_here = s_last != 0;
                if (!last_here) break;
                /* part k of the join: of worker lo + k, or of the k-th run of
                 * workers, in its first slot (in the item's first worker: its
                 * second) */
                const uint32_t from = by == 1 ? lo : first / kFan * kFan, to = by == 1 && lo != first ? 2 * lo : 2 * first + 1;
                auto slot_of = [&](uint32_t k) -> uint32_t { return k ? 2 * (from + k * by) : to; };
                const bool more = tree && round == 0;
                /* weights of the parts (at most 65), a row a warp, in the
                 * warps' free slots; 1 / sum in place of the warps' maxima */
                auto s_weight = [&](uint32_t r, uint32_t k) -> float & {
                    return reinterpret_cast<float *>(smem + s_free[r & (kWarps - 1)])[r / kWarps * n + k];
                };
                #pragma unroll 1
                for (uint32_t r = warp; r < rows; r += kWarps) {
                    float M = kNoMax, L = 0.0f;
                    float2 ml[3];
                    #pragma unroll
                    for (int i = 0; i < 3; i++) {
                        const uint32_t k = lane + 32 * i;
                        ml[i] = make_float2(kNoMax, 0.0f);
                        if (k < n) ml[i] = ct_gqa_load_l2(reinterpret_cast<const float2 *>(a.part_ml + slot_of(k) * 32) + r);
                        M = fmaxf(M, ml[i].x);
                    }
                    #pragma unroll
                    for (int d = 1; d < 32; d <<= 1) M = fmaxf(M, __shfl_xor_sync(0xFFFFFFFFu, M, d));
                    #pragma unroll
                    for (int i = 0; i < 3; i++) {
                        const float f = ex2(ml[i].x - M);
                        L += ml[i].y * f;
                        if (lane + 32 * i < n) s_weight(r, lane + 32 * i) = f;
                    }
                    #pragma unroll
                    for (int d = 1; d < 32; d <<= 1) L += __shfl_xor_sync(0xFFFFFFFFu, L, d);
                    if (lane == 0) {
                        s_ml[0][r][0] = more ? 1.0f : L == 0.0f ? 0.0f : rcp(L);
                        if (more) __stcg(reinterpret_cast<float2 *>(a.part_ml + (size_t)to * 32) + r, make_float2(M, L));
                        else if (a.lse) a.lse[(size_t)seq * a.n_q_heads + query_head(r)] = (M + lg2(L)) * kLn2;
                    }
                }
                __syncthreads();
                /* Loads in flight: 8 of a thread, 16 in the form that has the
                 * registers (one sequence of 8000 tokens 13.8 -> 13.2 us),
                 * spread over the columns that a thread has with 9 to 16 heads
                 * (one sequence of 500 tokens, 4 kv heads of 16 query heads,
                 * 128 values: 12.2 -> 11.6). */
                constexpr int kCols = HT == 1 ? 1 : D >= 96 ? 4 : 2, kParts = (FEW ? 16 : 8) / kCols;
                const uint32_t cols = rows * (D / 4);
                #pragma unroll 1
                for (uint32_t c0 = tid; c0 < cols; c0 += kCols * kThreads) {
                    float4 acc[kCols];
                    #pragma unroll
                    for (int x = 0; x < kCols; x++) acc[x] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    #pragma unroll 1
                    for (uint32_t k0 = 0; k0 < n; k0 += kParts) {
                        float4 v[kCols][kParts];
                        #pragma unroll
                        for (int k = 0; k < kParts; k++) {   /* 32-bit offsets: the parts are a few MB */
                            const float4 *from = reinterpret_cast<const float4 *>(a.part_o + slot_of(k0 + k) * (16 * D));
                            #pragma unroll
                            for (int x = 0; x < kCols; x++)
                                if (k0 + k < n && c0 + x * kThreads < cols) v[x][k] = ct_gqa_load_l2(from + c0 + x * kThreads);
                        }
                        #pragma unroll
                        for (int k = 0; k < kParts; k++) {
                            if (k0 + k >= n) break;
                            #pragma unroll
                            for (int x = 0; x < kCols; x++) {
                                if (c0 + x * kThreads >= cols) break;
                                const float f = s_weight((c0 + x * kThreads) / (D / 4), k0 + k);
                                acc[x].x += v[x][k].x * f; acc[x].y += v[x][k].y * f;
                                acc[x].z += v[x][k].z * f; acc[x].w += v[x][k].w * f;
                            }
                        }
                    }
                    #pragma unroll
                    for (int x = 0; x < kCols; x++) {
                        const uint32_t c = c0 + x * kThreads, r = c / (D / 4), d = (c % (D / 4)) * 4;
                        if (c >= cols) break;
                        if (more) __stcg(reinterpret_cast<float4 *>(a.part_o + (size_t)to * (16 * D)) + c, acc[x]);
                        else write(r, d, s_ml[0][r][0], acc[x]);
                    }
                }
                by = kFan;
            }
            __syncthreads();                                 /* the free slots may be refilled */
        }
    }
}

}  // namespace ct_gqa
