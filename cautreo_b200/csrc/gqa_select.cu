/*
 * gqa_select.cu -- the pages that a query is likely to attend, chosen by a
 * cheap score for each (sequence, kv head).
 *
 * Math: a query head of the group is rounded to whole numbers, e = max|q|/127,
 * c = rint(q / e).  With a page's bounds (upper and lower codes hi, lo and
 * their scale s), the largest dot product that any key inside the bounds has
 * is sum_d max(c_d, 0) hi_d + min(c_d, 0) lo_d, a dot product of length 2 D
 * in int8 with an int32 sum; score = max over heads of (sum * e), times s.
 * Whole-number sums are exact in every order, and the two products are
 * single fp32 roundings, so the chosen pages do not depend on how the sums
 * are split (ties go to the lowest page).
 *
 * Bound: HBM, 2 D + 4 bytes a page and head, while the scores are made, and
 * latency of the launch, the rounding and the select: 64 sequences of 16 to
 * 1024 pages, 8 heads of 128, take 27 us, 10.7 of them for the bytes, 3 what a
 * call costs that has nothing to choose, 6 for rows of unequal length (21 us
 * for as many pages in rows of 512).  A CTA per
 * (sequence, kv head), or a cluster of up to 8 when the batch has few: its
 * warps take 16 pages at a time, as the rows of mma.sync m16n8k32 (int8), 8
 * heads of the group being the columns, with the next pages' numbers loaded
 * ahead.  The scores become ordered 32-bit keys in the first CTA's shared
 * memory; a radix select over the bits that differ finds the key of the last
 * page chosen, and a scan writes the pages in ascending order.
 */
#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <math.h>

#include "../../include/hal.h"
#include "../../include/kv_cache.h"
#include "ct_internal.h"
#include "gqa_internal.h"

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr uint32_t kMaxPages = 49152;                        /* keys in shared memory: 192 KB */
constexpr int kTiles = 2;                                    /* runs of 8 pages a warp takes at a time: the rows of an MMA */
constexpr uint32_t kKeyInf = 0xFF800000u, kKeyForced = 0xFFFFFFFFu;

CT_DEV void mma_s8(int *c, const uint32_t *a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

/* Ordered key of a score: larger score, larger key; 0 is kept for "never". */
CT_DEV uint32_t key_of(float x) {
    if (x != x) return kKeyInf;
    const uint32_t u = __float_as_uint(x + 0.0f);            /* -0 and +0 tie */
    return (u >> 31) ? ~u : u | 0x80000000u;
}

/* CTAs an SM holds; four leave 64 registers a thread, which spills 32 bytes at
 * D = 128 (8 at 96, 4 at 64). */
template <int D> constexpr uint32_t kResident = D <= 128 ? 4 : 2;

template <int D>
__global__ void __launch_bounds__(kThreads, kResident<D>) k_gqa_select(const ct_gqa_select_args_t a) {
    extern __shared__ __align__(16) uint32_t keys[];
    constexpr int kPitch = 2 * D + 64;                       /* rows g, g + 1 in different halves of the banks */
    __shared__ __align__(16) int8_t s_q[16][kPitch];         /* (positive, negative) parts of 16 heads' codes */
    __shared__ float s_e[16];
    __shared__ uint32_t s_bad, s_hist[256], s_scan[2][kWarps], s_thr, s_left, s_most, s_nz, s_all, s_any;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, j = lane & 3;
    const cg::cluster_group cluster = cg::this_cluster();
    const uint32_t ranks = cluster.num_blocks(), rank = cluster.block_rank();
    const uint32_t pair = blockIdx.x / ranks;                /* (sequence, kv head) */
    const uint32_t seq = pair / a.n_kv_heads, head = pair % a.n_kv_heads;
    int32_t *out = a.picked + (size_t)pair * a.n_pick;
    uint32_t *lead = ranks > 1 ? cluster.map_shared_rank(keys, 0) : keys;
    ct_gqa_enter();
    const int32_t n = a.seq_lens[seq];
    const uint32_t cap = a.max_pages * a.page_tokens;
    const uint32_t len = n < 0 ? 0u : ((uint32_t)n > cap ? cap : (uint32_t)n);
    const uint32_t start = a.window && len > a.window ? len - a.window : 0u;
    const uint32_t first = start / a.page_tokens;
    const uint32_t have = len ? (len - 1) / a.page_tokens - first + 1 : 0u;
    const int32_t *table = a.block_table + (size_t)seq * a.max_pages + first;
    const bool choose = have > a.n_pick;
    if (!choose && rank) return;                             /* the whole cluster decides alike: no barrier is missed */
    if (choose && ranks > 1) cluster.sync();                 /* the first CTA runs: its shared memory may be written */
    if (tid == 0) { s_bad = 0; s_nz = 0; s_all = 0xFFFFFFFFu; s_any = 0; }
    __syncthreads();

    constexpr uint32_t kStep = kTiles * 8;
    const uint32_t pb = (uint32_t)((uint64_t)have * rank / ranks), pe = (uint32_t)((uint64_t)have * (rank + 1) / ranks);
    int32_t ph[kTiles];
    auto numbers = [&](uint32_t p0) {                        /* of the pages that a warp takes from p0 on */
        #pragma unroll
        for (int t = 0; t < kTiles; t++) {
            const uint32_t p = p0 + t * 8 + g;
            ph[t] = p < pe ? table[p] : -1;
        }
    };
    const uint32_t n_tiles = (a.group + 15) / 16;
    if (choose) numbers(pb + warp * kStep);                  /* on their way while the queries are rounded */
    for (uint32_t tile = 0; choose && tile < n_tiles; tile++) {
        /* the tile's heads as whole numbers: two rows a warp */
        for (uint32_t r = warp; r < 16; r += kWarps) {
            const uint32_t in_group = tile * 16 + r;
            const bool live = in_group < a.group;
            const uint32_t qh = a.blocked ? head * a.group + in_group : in_group * a.n_kv_heads + head;
            const uint16_t *qp = a.q + (size_t)seq * a.q_stride + (size_t)qh * D;
            float x[D / 32];
            uint32_t top = 0;
            #pragma unroll
            for (int i = 0; i < D / 32; i++) {
                x[i] = live ? ct_bf16_to_f32(qp[lane + 32 * i]) : 0.0f;
                top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
            }
            #pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
            const float e = __fdiv_rn(__uint_as_float(top), 127.0f);
            #pragma unroll
            for (int i = 0; i < D / 32; i++) {
                int c = 0;
                if (top < 0x7F800000u && e > 0.0f) c = __float2int_rn(__fdiv_rn(x[i], e));
                c = max(-127, min(127, c));
                s_q[r][lane + 32 * i] = (int8_t)max(c, 0);
                s_q[r][D + lane + 32 * i] = (int8_t)min(c, 0);
            }
            if (lane == 0) {
                s_e[r] = live ? e : -1.0f;
                if (top >= 0x7F800000u) s_bad = 1;
            }
        }
        __syncthreads();
        const uint32_t rows = a.group - tile * 16 < 16 ? a.group - tile * 16 : 16;
        const bool bad = s_bad != 0;
        if (tile) numbers(pb + warp * kStep);
        for (uint32_t p0 = pb + warp * kStep; p0 < pe; p0 += kWarps * kStep) {
            uint4 w[kTiles][D / 32];
            float ps[kTiles];
            bool ok[kTiles];
            #pragma unroll
            for (int t = 0; t < kTiles; t++) {
                ok[t] = (uint32_t)ph[t] < a.n_pages;
                const size_t at = (size_t)(ok[t] ? ph[t] : 0) * a.n_kv_heads + head;
                const uint4 *src = reinterpret_cast<const uint4 *>(a.bounds + at * 2 * D) + j;
                #pragma unroll
                for (int b = 0; b < D / 32; b++) w[t][b] = ok[t] ? src[b * 4] : make_uint4(0u, 0u, 0u, 0u);
                ps[t] = ok[t] ? a.bound_scales[at] : 0.0f;
            }
            numbers(p0 + kWarps * kStep);
            /* rows = pages p0 + g and p0 + 8 + g, columns = heads 2j, 2j + 1 of a
             * tile; lane j owns bytes 16 j .. 16 j + 15 of each 64 */
            float m[2] = {-INFINITY, -INFINITY};
            #pragma unroll
            for (int ht = 0; ht < 2; ht++) {
                if (8 * ht >= (int)rows) break;
                int c[4] = {0, 0, 0, 0};
                #pragma unroll
                for (int b = 0; b < D / 32; b++) {
                    const uint4 q = *reinterpret_cast<const uint4 *>(&s_q[8 * ht + g][b * 64 + 16 * j]);
                    const uint32_t a0[4] = {w[0][b].x, w[1][b].x, w[0][b].y, w[1][b].y};
                    const uint32_t a1[4] = {w[0][b].z, w[1][b].z, w[0][b].w, w[1][b].w};
                    mma_s8(c, a0, q.x, q.y);
                    mma_s8(c, a1, q.z, q.w);
                }
                #pragma unroll
                for (int h = 0; h < 2; h++) {                /* heads past the group have e = -1 */
                    const float e = s_e[8 * ht + 2 * j + h];
                    #pragma unroll
                    for (int t = 0; t < 2; t++) m[t] = fmaxf(m[t], e < 0.0f ? -INFINITY : __fmul_rn((float)c[2 * t + h], e));
                }
            }
            #pragma unroll
            for (int t = 0; t < kTiles; t++) {
                m[t] = fmaxf(m[t], __shfl_xor_sync(0xFFFFFFFFu, m[t], 1));
                m[t] = fmaxf(m[t], __shfl_xor_sync(0xFFFFFFFFu, m[t], 2));
                const uint32_t pp = p0 + t * 8 + g;
                if (j == 0 && pp < pe) {
                    uint32_t key = bad ? kKeyInf : key_of(__fmul_rn(m[t], ps[t]));
                    if (pp < a.n_first || pp + a.n_last >= have) key = kKeyForced;
                    if (!ok[t]) key = 0;
                    lead[pp] = tile ? max(lead[pp], key) : key;
                }
            }
        }
        __syncthreads();
    }
    if (choose && ranks > 1) {
        cluster.sync();                                      /* every rank's keys have reached the first CTA */
        if (rank) return;
    }
    if (!choose)
        for (uint32_t p = tid; p < have; p += kThreads) keys[p] = (uint32_t)table[p] < a.n_pages ? 1u : 0u;
    __syncthreads();

    /* ---- the key of the last page chosen ---- */
    uint32_t thr = 0, left = 0;                              /* keys above thr, and the first `left` equal to it, are chosen */
    if (choose) {
        /* mapped pages, forced ones apart, and the bits in which the other keys differ */
        uint32_t nz = 0, all = 0xFFFFFFFFu, any = 0;
        for (uint32_t p = tid; p < have; p += kThreads) {
            const uint32_t k = keys[p];
            nz += (k != 0) + ((k == kKeyForced) << 16);
            if (k != 0 && k != kKeyForced) { all &= k; any |= k; }
        }
        /* at most 49152 pages: both counts fit 16 bits of the sum */
        nz = __reduce_add_sync(0xFFFFFFFFu, nz);
        all = __reduce_and_sync(0xFFFFFFFFu, all);
        any = __reduce_or_sync(0xFFFFFFFFu, any);
        if (lane == 0) { atomicAdd(&s_nz, nz); atomicAnd(&s_all, all); atomicOr(&s_any, any); }
        s_hist[tid] = 0;
        __syncthreads();
        if ((s_nz & 0xFFFFu) > a.n_pick) {
            uint32_t want = a.n_pick - (s_nz >> 16);         /* forced pages come first */
            if (want == 0) {
                thr = kKeyForced - 1;
            } else {
                const uint32_t differ = s_all ^ s_any;
                int shift = differ ? 24 - __clz(differ) : 0; /* lowest bit of the first pass's digit */
                uint32_t prefix = s_all;                     /* the bits above the digits are the same in all */
                uint32_t known = shift >= 24 ? 0u : 0xFFFFFFFFu << (shift < 0 ? 8 : shift + 8);
                for (;;) {
                    const int lo = shift < 0 ? 0 : shift;
                    for (uint32_t p = tid; p < have; p += kThreads) {
                        const uint32_t k = keys[p];
                        if (k != 0 && k != kKeyForced && ((k ^ prefix) & known) == 0) atomicAdd(&s_hist[(k >> lo) & 255u], 1u);
                    }
                    __syncthreads();
                    /* suffix counts over 256 bins; thread t looks at bin 255 - t */
                    const uint32_t cnt = s_hist[255 - tid];
                    uint32_t inc = cnt;
                    #pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, inc, o);
                        if (lane >= (uint32_t)o) inc += y;
                    }
                    if (lane == 31) s_scan[0][warp] = inc;
                    __syncthreads();
                    s_hist[tid] = 0;
                    for (uint32_t w = 0; w < warp; w++) inc += s_scan[0][w];
                    if (inc >= want && inc - cnt < want) { s_thr = 255 - tid; s_left = want - (inc - cnt); s_most = cnt; }
                    __syncthreads();
                    known = 0xFFFFFFFFu << lo;
                    prefix = (prefix & ~(255u << lo)) | (s_thr << lo);
                    want = s_left;
                    /* nothing to tell apart below this digit if all of its keys are chosen */
                    if (lo == 0 || (want == s_most && (prefix & known))) break;
                    shift -= 8;
                }
                const bool all_of = shift > 0;
                thr = all_of ? (prefix & known) - 1 : prefix;
                left = all_of ? 0u : want;
            }
        }
    }
    /* ---- ascending pages: thread t owns a run of them ---- */
    const uint32_t per = (have + kThreads - 1) / kThreads;
    const uint32_t b0 = min(tid * per, have), b1 = min(b0 + per, have);
    uint32_t gt = 0, eq = 0;
    for (uint32_t p = b0; p < b1; p++) { gt += keys[p] > thr; eq += keys[p] == thr; }
    uint32_t ig = gt, ie = eq;
    #pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t yg = __shfl_up_sync(0xFFFFFFFFu, ig, o), ye = __shfl_up_sync(0xFFFFFFFFu, ie, o);
        if (lane >= (uint32_t)o) { ig += yg; ie += ye; }
    }
    if (lane == 31) { s_scan[0][warp] = ig; s_scan[1][warp] = ie; }
    __syncthreads();
    uint32_t all_gt = 0;
    for (uint32_t w = 0; w < kWarps; w++) {
        if (w < warp) { ig += s_scan[0][w]; ie += s_scan[1][w]; }
        all_gt += s_scan[0][w];
    }
    uint32_t ng = ig - gt, ne = ie - eq;
    for (uint32_t p = b0; p < b1; p++) {
        const uint32_t k = keys[p];
        const bool take = k > thr || (k == thr && thr != 0 && ne < left);
        if (take) out[ng + min(ne, left)] = (int32_t)(first + p);
        ng += k > thr;
        ne += k == thr;
    }
    for (uint32_t i = all_gt + left + tid; i < a.n_pick; i += kThreads) out[i] = -1;
}

template <int D> int prepare() {
    return ct__cuda_status(cudaFuncSetAttribute(k_gqa_select<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxPages * 4),
                           "gqa select");
}

template <int D> int run(const ct_gqa_select_args_t *a, cudaStream_t st) {
    /* CTAs for each (sequence, kv head): more than one when the batch leaves
     * SMs idle and its rows are long enough to share; as many as the SMs hold
     * where they are longer (16 sequences of 2048 pages, 8 heads: 35.6 -> 24.3
     * us; of 512 pages, which stay whole, 11.3, shared 12.6). */
    const uint32_t slots = a->n_sms * (4 * a->max_pages <= 48 * 1024 ? kResident<D> : 1u);       /* four keys arrays fit an SM */
    const uint64_t rows = (uint64_t)a->n_seq * a->n_kv_heads, work = (uint64_t)a->max_pages * ((a->group + 15) / 16);
    uint32_t ranks = 1;
    while (ranks < 8 && ((2 * ranks * rows <= a->n_sms && a->max_pages >= 256 * ranks) ||
                         (2 * ranks * rows <= slots && work > 512 * ranks)))
        ranks *= 2;
    ct__count_launches(1);
    return ct__cuda_status(ct_gqa_launch(k_gqa_select<D>, dim3(a->n_seq * a->n_kv_heads * ranks), dim3(kThreads),
                                         (size_t)a->max_pages * 4, st, ranks, *a),
                           "gqa select");
}

}  // namespace

extern "C" uint32_t ct__gqa_select_max_pages(void) { return kMaxPages; }

extern "C" int ct__gqa_select_prepare(void) {
    int rc = prepare<32>();
    if (!rc) rc = prepare<64>();
    if (!rc) rc = prepare<96>();
    if (!rc) rc = prepare<128>();
    if (!rc) rc = prepare<192>();
    if (!rc) rc = prepare<256>();
    return rc;
}

extern "C" int ct__launch_gqa_select(const ct_gqa_select_args_t *a, void *stream) {
    cudaStream_t st = (cudaStream_t)stream;
    switch (a->dim) {
        case 32: return run<32>(a, st);
        case 64: return run<64>(a, st);
        case 96: return run<96>(a, st);
        case 128: return run<128>(a, st);
        case 192: return run<192>(a, st);
        case 256: return run<256>(a, st);
        default: return CT_ERR_UNSUPPORTED;
    }
}
