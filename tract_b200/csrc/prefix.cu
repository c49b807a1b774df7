// b200kv_attend_shared: decode attention of a batch whose sequences begin with the same pages (b200kv_fork_shared).
//
// b200kv_attend streams the pages of every sequence for that sequence alone, so the beginning that n sequences share is read
// n times.  Here the rows of all of them -- sequence x query head of the kv head's group -- meet each shared page once:
//   m, l, O  of a row over the shared pages     prefix_tc_kernel (tcgen05) or prefix_simt_kernel, split along the pages
//   m, l, O  of a row over its own pages        the decode kernels, starting behind the shared pages
//   out = sum_k e^(m_k - m) O_k / sum_k e^(m_k - m) l_k,   m = max m_k      combine_shared_kernel
// Semantics of each row: transformers/src/ops/flash_sdpa.rs:239-341 with one query.  The reference has no counterpart of the
// sharing itself: its states are cloned whole (gpu/src/ops/dyn_kv_cache.rs:136-168).
#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>
#include <vector>

#include "attn_convert.cuh"
#include "decode_common.h"
#include "f32x2.cuh"
#include "q40_common.cuh"

namespace cg = cooperative_groups;

namespace b200kv {

struct PrefixParams {
    DecodeParams d;  // q, rotary embedding, pool, table, workspace: as the decode kernels get them
    int32_t chunk_bytes;
    float skip_fraction;
};

constexpr int XM = 128;            // rows of a tile
constexpr int X_SM_THREADS = 128;  // softmax threads per tile: one per row
constexpr int X_XCHG = 8;          // per tile and page parity: one flag per softmax warp (does the page need its remainder product)
// f16 weights skip the remainder product of a page once sqrt(64) x the largest weight of the page is below this fraction of
// the running sum, for every row of the tile (see prefill_tc.cu)
constexpr float X_SKIP_FRACTION = 0.125f;
// Weights are 2^(s sl2 - m) with one rounding, while m is a rounded s sl2: at the maximum the exponent is off 0 by half a step
// of m.  From this |m| on (a step of 2) the products are rounded first, as m was: otherwise the weights of a page leave the range
// of f16 from 2^27 on, that of bf16 from 2^31 on.
constexpr float X_FAR = 16777216.f;
enum { PSRC_PAGES16 = 0, PSRC_Q8 = 1, PSRC_Q4 = 2 };

constexpr int X_CLUSTER = 2;  // CTAs that join their runs before a partial leaves the chip

// ALT: one tile of 128 rows, whose pages two pipelines take in turn; otherwise two tiles, which read every staged page twice.
template <bool ALT, int D, int SRC>
struct XGeo {
    static constexpr bool RAW = SRC != PSRC_PAGES16;   // block-quantised pages: converter warps rebuild the operand tiles
    static constexpr int FT = RAW ? 256 : 0;           // converter threads, beside the copy warp
    static constexpr int ROWS = ALT ? XM : 2 * XM;     // rows of a CTA
    static constexpr int USERS = ALT ? 1 : 2;          // pipelines that read a staged page
    static constexpr int PLANES = D / 64;
    static constexpr int CHUNK = PAGE_TOKENS * D * 2;  // one operand tile: 64 keys
    static constexpr int QBYTES = XM * D * 2;
    static constexpr int KPARTS = RAW ? 2 : 1;         // K as value + remainder where it was rounded
    static constexpr int KSTAGE = KPARTS * CHUNK;
    static constexpr int NK = RAW ? 2 : 4;
    static constexpr int NV = RAW ? (ALT ? 4 : 3) : 5;
    static constexpr int NR = RAW ? (ALT ? 3 : 2) : 1;
    static constexpr int RAW_STAGE = RAW ? 2 * (PAGE_TOKENS * D + PAGE_TOKENS * (D / 32) * 2) : 0;
    static constexpr int THREADS = 2 * X_SM_THREADS + 64 + 32 + FT;
    static constexpr int N_BARS = 2 * NK + 2 * NV + 12 + 2 * NR;
    static constexpr uint32_t COL_S = D, COLS_PER_TILE = 256;  // TMEM: O in columns 0 .. D-1, the two S buffers behind it
    static constexpr int PARTS = (ALT ? 2 : 1) * X_CLUSTER;    // partials of a row in a cluster
    static constexpr int ML_BYTES = PARTS * ROWS * 8;
    // what the other parts send of the columns that a CTA joins: over the operand rings, which are done with by then
    static constexpr size_t JOIN = (size_t)(PARTS - 1) * ROWS * (D / X_CLUSTER) * 4 + (size_t)ROWS * (D / X_CLUSTER / 4 + 1) * 16;
    static constexpr size_t RINGS = (size_t)NK * KSTAGE + (size_t)NV * CHUNK + (size_t)NR * RAW_STAGE;
    static constexpr int UNIT_BYTES = RAW ? ROWS * 4 : 0;
    static constexpr size_t SMEM = (size_t)ROWS * D * 2 + RINGS + N_BARS * 8 + 32 + 4 * X_XCHG * 4 + ML_BYTES + UNIT_BYTES;
    static_assert(COL_S + 128 <= COLS_PER_TILE && JOIN <= RINGS && SMEM <= 227 * 1024, "TMEM columns and shared memory of an SM");
};

// The shared pages against every row that sees them, on the 5th-generation tensor cores.
//   S = Q K^T   M = 128 rows (sequence, head of the group), N = 64 keys of a page, operands in shared memory
//   P = 2^(scale log2e S - m)   one thread per row, m raised only when exceeded by 2^8, l = sum P
//   O += P V    A = P from TMEM, B = V as it lies in the page
// The pipeline -- S double-buffered in TMEM, P over the S it came from, rings of K and V tiles, bounded waits -- is the one
// of prefill_tc.cu and attn_tc.cu; there are no masks (every row sees every shared page whole) and the rows come from different
// sequences.  The result is a run's partial (m, l, O) in f32 for the combine pass.
// Bound: a page and kv head is 32 KB of f16, 1340 cycles of an SM's share of HBM at the copy rate; its products for 128 rows
// take 640 to 900 cycles of the tensor pipe, but one pipeline needs 2200 cycles from a page to the next (product, softmax,
// product, each waiting for the one before; 3500 over int8 pages, whose converter warps share the issue slots with the softmax).
// Two pipelines per CTA therefore: up to 128 rows they take the pages in turn, one every 1100 (1750) cycles; above that they are two
// tiles, each of which meets every page, at the pace of one pipeline.  Measured without own pages, 8 heads, from 16384 to 32768
// tokens: 0.83 us a page and CTA with one tile (the copy rate), 1.24 with two; int8 0.92 and 1.61.
// Measured: 128 rows per kv head, 8 of them, after 32768 tokens: f16 27 us for this kernel (134 MB, 5.0 TB/s), 43 for the call;
// int8 35 and 51, of which the conversion is 9.  4 us go before the first page (TMEM, barriers, query tiles), 5 after the last.
// A CTA has a run of pages; the two CTAs of a cluster have neighbouring runs and join (m, l, O) through distributed shared
// memory, each for half of the channels, before a partial is written: half of the partials' traffic and workspace, which
// otherwise limits the runs to fewer than the GPU has SMs.
template <bool ALT, int D, int SRC>
__global__ void __launch_bounds__(XGeo<ALT, D, SRC>::THREADS, 1) __cluster_dims__(X_CLUSTER, 1, 1)
    prefix_tc_kernel(const __grid_constant__ PrefixParams p, const __grid_constant__ PrefixBatch pb) {
    using GEO = XGeo<ALT, D, SRC>;
    constexpr int NK = GEO::NK, NV = GEO::NV, NR = GEO::NR, CHUNK = GEO::CHUNK, QBYTES = GEO::QBYTES, PLANES = GEO::PLANES;
    constexpr int KSTAGE = GEO::KSTAGE, KPARTS = GEO::KPARTS, FT = GEO::FT, ROWS = GEO::ROWS, PARTS = GEO::PARTS;
    constexpr bool RAW = GEO::RAW;  // converted pages: f16 operands whatever the query type
    constexpr uint32_t COL_O = 0, COL_S = GEO::COL_S, COLS_PER_TILE = GEO::COLS_PER_TILE;
    constexpr int FILL_ARRIVALS = RAW ? FT / 32 : 1;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* q_s = smem;                                    // [ROWS / 128][PLANES][128 rows][128 B], swizzled
    uint8_t* k_ring = smem + ROWS * D * 2;                  // NK K stages of KPARTS tiles
    uint8_t* v_ring = k_ring + NK * KSTAGE;                 // NV V tiles
    uint8_t* raw_ring = v_ring + NV * CHUNK;                // NR raw chunk pairs
    uint64_t* full_k = (uint64_t*)(raw_ring + NR * GEO::RAW_STAGE);  // [NK] the tile is complete
    uint64_t* full_v = full_k + NK;                         // [NV]
    uint64_t* free_k = full_v + NV;                         // [NK] every Q.K^T on the stage has completed
    uint64_t* free_v = free_k + NK;                         // [NV] every P.V on the stage has completed
    uint64_t* bar_s = free_v + NV;                          // [2 pipelines][2] S buffer written
    uint64_t* bar_p = bar_s + 4;                            // [2][2] P written by the softmax warps
    uint64_t* bar_o = bar_p + 4;                            // [2][2] P.V of a pipeline's page i completed, on barrier i & 1
    uint64_t* full_raw = bar_o + 4;                         // [NR] raw bytes landed
    uint64_t* free_raw = full_raw + NR;                     // [NR] every converter warp is done with the raw stage
    uint32_t* tmem_slot = (uint32_t*)(((uintptr_t)(free_raw + NR) + 15) & ~(uintptr_t)15);
    volatile int* fail_s = (volatile int*)(tmem_slot + 1);
    float* xchg = (float*)(tmem_slot + 4);                  // [2][2 parities][X_XCHG]
    float2* ml_s = (float2*)(xchg + 4 * X_XCHG);            // [PARTS][ROWS] (m, l) of every part of the cluster
    float* unit_s = (float*)(ml_s + PARTS * ROWS);          // RAW: [ROWS] what a step of 1 of a bf16 query's f16 operand stands for
    float4* join_s = (float4*)k_ring;                       // [PARTS - 1][D / X_CLUSTER / 4][ROWS]

    const DecodeParams& dp = p.d;
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int kvh = blockIdx.y, rank = (int)cluster.block_rank();
    const PrefixGroup grp = prefix_group_of(pb, blockIdx.x);
    const int at = ((int)blockIdx.x - grp.cta0) / X_CLUSTER, joined = at / grp.tiles, tile = at % grp.tiles;
    int page0, n_pages;
    prefix_run(grp, grp.splits * X_CLUSTER, joined * X_CLUSTER + rank, &page0, &n_pages);
    const int n_rows = grp.n_seqs * dp.G;
    // pages of pipeline t, and the page its i-th one is
    auto pages_of = [&](int t) { return ALT ? (n_pages - t + 1) / 2 : n_pages; };
    auto page_at = [&](int t, int i) { return ALT ? 2 * i + t : i; };

    if (tid == 0) {
        for (int s = 0; s < NK; s++) mbar_init(&full_k[s], FILL_ARRIVALS), mbar_init(&free_k[s], GEO::USERS);
        for (int s = 0; s < NV; s++) mbar_init(&full_v[s], FILL_ARRIVALS), mbar_init(&free_v[s], GEO::USERS);
        for (int i = 0; i < 4; i++) mbar_init(&bar_s[i], 1), mbar_init(&bar_p[i], X_SM_THREADS / 32);
        for (int i = 0; i < 4; i++) mbar_init(&bar_o[i], 1);
        for (int s = 0; s < NR; s++) mbar_init(&full_raw[s], 1), mbar_init(&free_raw[s], FT / 32);
        *fail_s = (smem_u32(smem) & 1023u) ? 1 : 0;  // the swizzled operand tiles need a 1024-byte aligned base
        mbar_fence_init();
    }
    if (warp == 0) tmem_alloc(tmem_slot, COLS_PER_TILE * 2);
    cluster.barrier_arrive();  // every CTA of the cluster runs before one writes into the other's shared memory
    grid_dependency_wait();    // the append before this launch has written its pages, and whoever made q is done

    const int qt = min(tid / X_SM_THREADS, 1), w4 = (tid % X_SM_THREADS) >> 5;  // pipeline, lane quarter
    const int row = w4 * 32 + lane;
    const int cta_row = ALT ? row : qt * XM + row;
    const int my_row = tile * ROWS + cta_row;  // row of the group: sequence my_row / G, head my_row % G
    const bool live = my_row < n_rows;
    const bool is_softmax = tid < 2 * X_SM_THREADS;
    const int is_bf16 = dp.dtype == B200KV_BF16;
    const int mma_bf16 = RAW ? 0 : is_bf16;  // type of the tensor-core operands (Q, K, V, P)

    __syncthreads();  // the barriers are there: the copy warp starts, the others fetch Q meanwhile
    // The next kernel may be scheduled; it waits for this grid before it reads the partials.  Not before the TMEM is allocated: a
    // later kernel that got hold of the SM's columns first would wait for this one, and this one for the columns.
    grid_launch_dependents();
    const int role = warp - 2 * (X_SM_THREADS / 32);  // 0, 1: MMAs of that pipeline; above: copies and conversion; below 0: softmax
    // ---- Q tiles -> shared memory, K-major with the 128-byte swizzle; neighbouring threads fetch neighbouring units of a row ----
    if (is_softmax) {
        constexpr int UNITS = D / 8;
        auto place = [&](int x) -> uint4* {  // unit x % UNITS of row x / UNITS
            const int r = x / UNITS, uu = x % UNITS, in_tile = r % XM;
            return (uint4*)(q_s + (r / XM) * QBYTES + (uu / 8) * (XM * 128) + in_tile * 128 + (((uu % 8) ^ (in_tile & 7)) << 4));
        };
        if (dp.q_cos) {  // the rotated value is rounded to the query's type, as a separate rope kernel would store it
#pragma unroll 1
            for (int x = tid; x < ROWS * UNITS; x += 2 * X_SM_THREADS) {
                const int g_row = tile * ROWS + x / UNITS, b = grp.b0 + g_row / dp.G, head = kvh * dp.G + g_row % dp.G;
                uint32_t w[4] = {0u, 0u, 0u, 0u};
                if (g_row < n_rows)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const float a = load_query(dp, D, b, head, (x % UNITS) * 8 + 2 * j), c = load_query(dp, D, b, head, (x % UNITS) * 8 + 2 * j + 1);
                        if (is_bf16) {
                            const __nv_bfloat162 h = __floats2bfloat162_rn(a, c);
                            w[j] = *(const uint32_t*)&h;
                        } else {
                            const __half2 h = __floats2half2_rn(a, c);
                            w[j] = *(const uint32_t*)&h;
                        }
                    }
                *place(x) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        } else {
            constexpr int BATCH = ROWS * UNITS / (2 * X_SM_THREADS) < 8 ? ROWS * UNITS / (2 * X_SM_THREADS) : 8;
#pragma unroll 1
            for (int x0 = tid; x0 < ROWS * UNITS; x0 += BATCH * 2 * X_SM_THREADS) {
                uint4 w[BATCH];
#pragma unroll
                for (int i = 0; i < BATCH; i++) {  // all of them on their way before the first is stored
                    const int x = x0 + i * 2 * X_SM_THREADS, g_row = tile * ROWS + x / UNITS;
                    const int b = grp.b0 + g_row / dp.G, head = kvh * dp.G + g_row % dp.G;
                    w[i] = make_uint4(0u, 0u, 0u, 0u);
                    if (g_row < n_rows) w[i] = ((const uint4*)((const uint16_t*)dp.q + (int64_t)b * dp.qb + (int64_t)head * dp.qh))[x % UNITS];
                }
#pragma unroll
                for (int i = 0; i < BATCH; i++) *place(x0 + i * 2 * X_SM_THREADS) = w[i];
            }
        }
        // Over converted pages a bf16 row becomes f16 times a power of two that brings its largest magnitude to 2^14 .. 2^15: what
        // lies within 2^28 of that stays exact (bf16 has fewer bits), the rest is off by at most 2^-39 of it.  The scale of the
        // row's scores takes the power back.  A thread has the units that it stored, UNITS neighbouring lanes a row.
        if (RAW && is_bf16) {
#pragma unroll 1
            for (int x = tid; x < ROWS * UNITS; x += 2 * X_SM_THREADS) {
                const uint4 b = *place(x);
                uint32_t w[4] = {b.x, b.y, b.z, b.w};
                float big = 0.f;
#pragma unroll
                for (int j = 0; j < 4; j++) big = fmaxf(big, fmaxf(fabsf(__uint_as_float(w[j] << 16)), fabsf(__uint_as_float(w[j] & 0xffff0000u))));
#pragma unroll
                for (int o = UNITS / 2; o; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
                const int e = max((int)(__float_as_uint(big) >> 23) - 127, -100);  // (both powers stay normal)
                const float up = __uint_as_float((uint32_t)(127 + 14 - e) << 23);
                if (x % UNITS == 0) unit_s[x / UNITS] = __uint_as_float((uint32_t)(127 - 14 + e) << 23);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const __half2 h = __floats2half2_rn(__uint_as_float(w[j] << 16) * up, __uint_as_float(w[j] & 0xffff0000u) * up);
                    w[j] = *(const uint32_t*)&h;
                }
                *place(x) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
        fence_async_proxy();  // generic-proxy writes -> visible to the tensor core
    }
    uint32_t tmem = 0;
    if (role < 2) {
        tc_fence_before();
        asm volatile("bar.sync 1, %0;" ::"n"(2 * X_SM_THREADS + 64) : "memory");  // softmax and MMA warps
        tc_fence_after();
        tmem = *tmem_slot;
    }

    const int32_t* pages = dp.table + (int64_t)grp.trow * dp.max_pages_per_seq + page0;
    const int n_copy = (int)blockIdx.x == dp.stall_item && kvh == 0 ? 0 : n_pages;  // test hook, see DecodeParams
    auto page_src = [&](int32_t pg) {  // a page id outside the pool is reported and replaced, so that the barriers go on
        if (pg < 0 || pg >= dp.n_pages) {
            if (lane == 0) atomicOr(dp.status, STATUS_PAGE_OOB);
            pg = 0;
        }
        return dp.pool + (int64_t)pg * dp.page_bytes + (int64_t)kvh * (2 * p.chunk_bytes);
    };
    const uint32_t lane_base = tmem + qt * COLS_PER_TILE + ((uint32_t)(w4 * 32) << 16);  // softmax threads: this warp's lane quarter
    float m_ref = -INFINITY, l_run = 0.f;

    if (!is_softmax) {
        // Every lane of these warps walks its loop (the values stay warp-uniform); one elected lane issues.
        if (role < 2) {
            const int t = role, n = pages_of(t);
            const uint32_t tm = tmem + t * COLS_PER_TILE;
            const uint32_t idesc_s = instr_desc(mma_bf16, 0, XM, PAGE_TOKENS);
            const uint32_t idesc_o = instr_desc(mma_bf16, 1, XM, D);
            const uint64_t q_desc = smem_desc(smem_u32(q_s) + (ALT ? 0 : t * QBYTES), 0, 1024);
            const uint64_t k_desc = smem_desc(smem_u32(k_ring), 0, 1024);
            // V tile: planes of 64 channels 8192 bytes apart (leading dimension), 8-key groups 1024 bytes apart
            const uint64_t v_desc = smem_desc(smem_u32(v_ring), PAGE_TOKENS * 128, 1024);
            const bool adaptive = !mma_bf16;
            auto issue_qk = [&](int i) {  // S(i) = Q . K^T of the pipeline's i-th page into buffer i & 1
                const int j = page_at(t, i);
                wait_or_fail(&full_k[j % NK], (uint32_t)((j / NK) & 1), fail_s, dp.wait_ns);
                tc_fence_after();
                if (elect_one()) {
                    const uint64_t kd = k_desc + (uint64_t)(((j % NK) * KSTAGE) >> 4);
#pragma unroll
                    for (int pl = 0; pl < PLANES; pl++)
#pragma unroll
                        for (int kk = 0; kk < 4; kk++) {
                            const uint64_t off = (uint64_t)((pl * (XM * 128) + kk * 32) >> 4);
                            const uint64_t koff = (uint64_t)((pl * (PAGE_TOKENS * 128) + kk * 32) >> 4);
                            if constexpr (KPARTS == 2) {
                                tc_mma_ss_a<A_KEEP>(tm + COL_S + 64 * (i & 1), q_desc + off, kd + koff, idesc_s, (pl | kk) ? 1u : 0u);
                                tc_mma_ss_a<A_REUSE_LAST>(tm + COL_S + 64 * (i & 1), q_desc + off, kd + (uint64_t)(CHUNK >> 4) + koff, idesc_s, 1u);
                            } else {
                                tc_mma_ss(tm + COL_S + 64 * (i & 1), q_desc + off, kd + koff, idesc_s, (pl | kk) ? 1u : 0u);
                            }
                        }
                    tc_commit(&bar_s[2 * t + (i & 1)]);
                    tc_commit(&free_k[j % NK]);
                }
                __syncwarp();
            };
            if (n > 0) issue_qk(0);
            if (n > 1) issue_qk(1);
            for (int i = 0; i < n; i++) {
                const int j = page_at(t, i);
                wait_or_fail(&full_v[j % NV], (uint32_t)((j / NV) & 1), fail_s, dp.wait_ns);
                wait_or_fail(&bar_p[2 * t + (i & 1)], (uint32_t)((i >> 1) & 1), fail_s, dp.wait_ns);
                tc_fence_after();
                const int* flags = (const int*)(xchg + (2 * t + (i & 1)) * X_XCHG);
                const bool two = !adaptive || __any_sync(0xffffffffu, flags[lane & 3] != 0);
                if (elect_one()) {
                    const uint64_t vd = v_desc + (uint64_t)(((j % NV) * CHUNK) >> 4);
                    const uint32_t pa = tm + COL_S + 64 * (i & 1);
#pragma unroll
                    for (int kk = 0; kk < 4; kk++) {
                        tc_mma_ts(tm + COL_O, pa + kk * 8, vd + (uint64_t)((kk * 2048) >> 4), idesc_o, (i | kk) ? 1u : 0u);
                        if (two) tc_mma_ts(tm + COL_O, pa + 32 + kk * 8, vd + (uint64_t)((kk * 2048) >> 4), idesc_o, 1u);
                    }
                    tc_commit(&bar_o[2 * t + (i & 1)]);
                    tc_commit(&free_v[j % NV]);
                }
                __syncwarp();
                // S(i + 2) reuses the buffer P(i) sits in: the tensor core runs one thread's MMAs in issue order
                if (i + 2 < n) issue_qk(i + 2);
            }
        } else if constexpr (!RAW) {
            // ================= the chunks of a 16-bit page are the operand tiles =================
            int32_t pg_next = n_pages > 0 ? pages[0] : 0;
            for (int i = 0; i < n_copy; i++) {
                const uint8_t* src = page_src(pg_next);
                if (i + 1 < n_pages) pg_next = pages[i + 1];  // fetched one page ahead of its use
                if (i >= NK) wait_or_fail(&free_k[i % NK], (uint32_t)((i / NK - 1) & 1), fail_s, dp.wait_ns);
                if (elect_one()) {
                    mbar_expect_tx(&full_k[i % NK], CHUNK);
                    bulk_g2s(k_ring + (i % NK) * CHUNK, src, CHUNK, &full_k[i % NK]);
                }
                __syncwarp();
                if (i >= NV) wait_or_fail(&free_v[i % NV], (uint32_t)((i / NV - 1) & 1), fail_s, dp.wait_ns);
                if (elect_one()) {
                    mbar_expect_tx(&full_v[i % NV], CHUNK);
                    bulk_g2s(v_ring + (i % NV) * CHUNK, src + CHUNK, CHUNK, &full_v[i % NV]);
                }
                __syncwarp();
            }
        } else {
            constexpr int FMT = SRC == PSRC_Q8 ? B200KV_FMT_Q8_1 : B200KV_FMT_Q4_0;
            const int ft = tid - (2 * X_SM_THREADS + 64 + 32);
            if (ft < 0) {
                // ================= raw chunk pairs, for the converter warps =================
                int32_t pg_next = n_pages > 0 ? pages[0] : 0;
                for (int i = 0; i < n_copy; i++) {
                    const uint8_t* src = page_src(pg_next);
                    if (i + 1 < n_pages) pg_next = pages[i + 1];
                    if (i >= NR) wait_or_fail(&free_raw[i % NR], (uint32_t)((i / NR - 1) & 1), fail_s, dp.wait_ns);
                    if (elect_one()) {
                        mbar_expect_tx(&full_raw[i % NR], 2 * p.chunk_bytes);
                        bulk_g2s(raw_ring + (i % NR) * GEO::RAW_STAGE, src, 2 * p.chunk_bytes, &full_raw[i % NR]);
                    }
                    __syncwarp();
                }
            } else {
                // ================= converter warps: raw chunk pair -> f16 operand tiles =================
                // No warp waits for another one: each goes on with the next page as soon as its share of this one is written.
                for (int i = 0; i < n_pages; i++) {
                    const uint8_t* raw = raw_ring + (i % NR) * GEO::RAW_STAGE;
                    wait_or_fail(&full_raw[i % NR], (uint32_t)((i / NR) & 1), fail_s, dp.wait_ns);
                    if (i >= NK) wait_or_fail(&free_k[i % NK], (uint32_t)((i / NK - 1) & 1), fail_s, dp.wait_ns);
                    convert_rows<FMT, D, 0, FT, true>(raw, k_ring + (i % NK) * KSTAGE, k_ring + (i % NK) * KSTAGE + CHUNK, PAGE_TOKENS, ft);
                    fence_async_proxy();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&full_k[i % NK]);
                    if (i >= NV) wait_or_fail(&free_v[i % NV], (uint32_t)((i / NV - 1) & 1), fail_s, dp.wait_ns);
                    convert_rows<FMT, D, 1, FT, true>(raw + p.chunk_bytes, v_ring + (i % NV) * CHUNK, nullptr, PAGE_TOKENS, ft);
                    fence_async_proxy();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&full_v[i % NV]), mbar_arrive(&free_raw[i % NR]);
                }
            }
        }
    } else {
        // ================= softmax threads =================
        const bool adaptive = !mma_bf16;
        const float sl2 = dp.scale * 1.4426950408889634f * (RAW && is_bf16 ? unit_s[cta_row] : 1.f);  // scores enter the exponent in log2 units
        float log_thresh = -INFINITY;
        const int n = pages_of(qt);
        for (int i = 0; i < n; i++) {
            const uint32_t sbuf = lane_base + COL_S + 64 * (i & 1);
            wait_or_fail(&bar_s[2 * qt + (i & 1)], (uint32_t)((i >> 1) & 1), fail_s, dp.wait_ns);
            tc_fence_after();
            uint32_t sr[64];
            tmem_ld32(sbuf, sr);
            tmem_ld32(sbuf + 32, sr + 32);
            tmem_ld_wait();
            const float tmax = row_max64(sr) * sl2;
            int* flags = (int*)(xchg + (2 * qt + (i & 1)) * X_XCHG);
            // Three questions per row, one reduction per warp.  Bit 0: the page needs its remainder product (see X_SKIP_FRACTION;
            // the first one always).  Bit 1: the reference maximum is exceeded by more than 2^8 (or was -inf until now): O is rescaled.
            // Bit 2: see X_FAR.
            const bool mine = adaptive && (i == 0 || !(tmax - m_ref + 3.f <= log_thresh));
            const bool raise = tmax > m_ref + 8.f || (m_ref == -INFINITY && tmax > -INFINITY);
            const uint32_t votes = __reduce_or_sync(0xffffffffu, (mine ? 1u : 0u) | (raise && i > 0 ? 2u : 0u) | (fabsf(tmax) > X_FAR ? 4u : 0u));
            const bool two = !adaptive || (votes & 1u);
            if (adaptive && lane == 0) flags[w4] = two ? 1 : 0;
            float alpha = 1.f;
            if (raise) {
                alpha = fast_exp2(m_ref - tmax);
                m_ref = tmax;
                l_run *= alpha;
            }
            if (votes & 6u) {
                if (votes & 2u) {
                    // O must hold every page before this one: see prefill_tc.cu for why the wait on barrier (i - 1) & 1 cannot
                    // mistake the completion of P.V(i - 3) or P.V(i + 1) for that of P.V(i - 1)
                    wait_or_fail(&bar_o[2 * qt + ((i - 1) & 1)], (uint32_t)(((i - 1) >> 1) & 1), fail_s, dp.wait_ns);
                    tc_fence_after();
#pragma unroll
                    for (int cc = 0; cc < D / 16; cc++) {
                        uint32_t orow[16];
                        tmem_ld16(lane_base + COL_O + cc * 16, orow);
                        tmem_ld_wait();
#pragma unroll
                        for (int c = 0; c < 16; c++) orow[c] = __float_as_uint(__uint_as_float(orow[c]) * alpha);
                        tmem_st16(lane_base + COL_O + cc * 16, orow);
                    }
                }
                if (votes & 4u) {  // (through TMEM: 64 products in registers would cost the common page spills)
#pragma unroll 1
                    for (int cc = 0; cc < 4; cc++) {
                        uint32_t x[16];
                        tmem_ld16(sbuf + cc * 16, x);
                        tmem_ld_wait();
#pragma unroll
                        for (int c = 0; c < 16; c++) x[c] = __float_as_uint(__fmul_rn(__uint_as_float(x[c]), sl2));
                        tmem_st16(sbuf + cc * 16, x);
                    }
                    tmem_st_wait();
                    tmem_ld32(sbuf, sr);
                    tmem_ld32(sbuf + 32, sr + 32);
                    tmem_ld_wait();
                }
            }
            const float m_use = m_ref == -INFINITY ? 0.f : m_ref;
            const float unit = (votes & 4u) ? 1.f : sl2;
            uint32_t pr[32], pr2[32];
            float page_sum;
            if (mma_bf16) page_sum = softmax_exps<2>(sr, unit, m_use, pr, pr2);
            else if (two) page_sum = softmax_exps<1>(sr, unit, m_use, pr, pr2);
            else page_sum = softmax_exps<0>(sr, unit, m_use, pr, pr2);
            tmem_st32(sbuf + 32, pr2);
            tmem_st32(sbuf, pr);
            l_run += page_sum;
            log_thresh = fast_log2(p.skip_fraction * l_run);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar_p[2 * qt + (i & 1)]);
        }
        if (n > 0) wait_or_fail(&bar_o[2 * qt + ((n - 1) & 1)], (uint32_t)(((n - 1) >> 1) & 1), fail_s, dp.wait_ns);
        tc_fence_after();
        if (n == 0 || *fail_s) m_ref = -INFINITY, l_run = 0.f;  // no pages, or a CTA that gave up: an empty partial
    }

    // ---- join the parts of the cluster: (m, l) to both CTAs, then each CTA's half of the channels ----
    const int part = ALT ? 2 * rank + qt : rank;
    // A CTA that gave up lets copies and products that may still be in flight end first: its rings take the other CTA's part next.
    // (Whoever gave up has set the flag and waits here; nobody is past the barriers below before.)
    if (*fail_s)
        for (const uint64_t t0 = globaltimer_ns(); globaltimer_ns() - t0 < 200000ull;) __nanosleep(10000);
    cluster.barrier_wait();
    if (is_softmax)
#pragma unroll
        for (int r = 0; r < X_CLUSTER; r++) cluster.map_shared_rank(ml_s, r)[part * ROWS + cta_row] = make_float2(m_ref, l_run);
    cluster.sync();  // every pipeline of both CTAs has ended: the operand rings are free
    constexpr int COLS = D / X_CLUSTER;  // channels a CTA joins: COLS * rank ..
    float M = -INFINITY, total = 0.f, mine = 0.f;
    if (is_softmax) {
#pragma unroll
        for (int q = 0; q < PARTS; q++) M = fmaxf(M, ml_s[q * ROWS + cta_row].x);
#pragma unroll
        for (int q = 0; q < PARTS; q++) {
            const float2 ml = ml_s[q * ROWS + cta_row];
            const float f = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - M);
            total = fmaf(f, ml.y, total);
            if (q == part) mine = f;
        }
#pragma unroll
        for (int r = 0; r < X_CLUSTER; r++) {
            const int home = ALT ? 2 * r : r;  // the part that stays in TMEM until the sum
            if (part == home) continue;
            float4* dst = cluster.map_shared_rank(join_s, r) + (size_t)(part < home ? part : part - 1) * (COLS / 4) * ROWS + cta_row;
#pragma unroll
            for (int cc = 0; cc < COLS / 16; cc++) {
                uint32_t o[16];
                tmem_ld16(lane_base + COL_O + r * COLS + cc * 16, o);
                tmem_ld_wait();
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);  // (an empty part's TMEM holds anything)
                    if (mine > 0.f)
                        v = make_float4(__uint_as_float(o[4 * c]) * mine, __uint_as_float(o[4 * c + 1]) * mine, __uint_as_float(o[4 * c + 2]) * mine,
                                        __uint_as_float(o[4 * c + 3]) * mine);
                    dst[(cc * 4 + c) * ROWS] = v;
                }
            }
        }
    }
    cluster.sync();
    if (is_softmax && (!ALT || qt == 0)) {
        const int64_t rec = (int64_t)grp.base + ((int64_t)joined * dp.Hkv + kvh) * n_rows + my_row;
        float4* out_s = join_s + (size_t)(PARTS - 1) * (COLS / 4) * ROWS;  // [ROWS][COLS / 4 + 1]
#pragma unroll
        for (int cc = 0; cc < COLS / 16; cc++) {
            uint32_t o[16];
            tmem_ld16(lane_base + COL_O + rank * COLS + cc * 16, o);
            tmem_ld_wait();
#pragma unroll
            for (int c = 0; c < 4; c++) {
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                if (mine > 0.f)
                    v = make_float4(__uint_as_float(o[4 * c]) * mine, __uint_as_float(o[4 * c + 1]) * mine, __uint_as_float(o[4 * c + 2]) * mine,
                                    __uint_as_float(o[4 * c + 3]) * mine);
#pragma unroll
                for (int q = 0; q < PARTS - 1; q++) {
                    const float4 x = join_s[((size_t)q * (COLS / 4) + cc * 4 + c) * ROWS + cta_row];
                    v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
                }
                out_s[cta_row * (COLS / 4 + 1) + cc * 4 + c] = v;
            }
        }
        // from rows per thread to neighbouring threads per row
        asm volatile("bar.sync 2, %0;" ::"n"(ROWS) : "memory");
        const int64_t rec0 = (int64_t)grp.base + ((int64_t)joined * dp.Hkv + kvh) * n_rows + tile * ROWS;
        for (int x = cta_row; x < ROWS * (COLS / 4); x += ROWS) {
            const int r = x / (COLS / 4), u = x % (COLS / 4);
            if (tile * ROWS + r < n_rows) ((float4*)(dp.part_o + (rec0 + r) * D + rank * COLS))[u] = out_s[r * (COLS / 4 + 1) + u];
        }
        if (live && rank == 0) *(float2*)(dp.part_ml + rec * 2) = make_float2(M * 0.6931471805599453f, total);  // natural-log units
    }
    tc_fence_before();
    __syncthreads();
    if (*fail_s && tid == 0) atomicOr(dp.status, STATUS_WAIT_EXPIRED);
    if (warp == 0) tmem_dealloc(tmem, COLS_PER_TILE * 2);
}

// ---- the same on the CUDA cores, for f32 pages ---------------------------------------------------------------------------
// A tile is 128 rows, or 64 or 32 for fewer.  Per page S = Q K^T with 4 x 4 scores per thread, the online softmax with expf (4
// threads per row), O += P V with 4 rows x D / 16 channels per thread, all products as packed pairs.  The chunks are used as they
// lie in the page: two bulk copies, each on its way while the other operand's product runs.
// Bound by the FMA pipe -- 4 D flops per row and key -- and the 16-byte shared-memory reads that feed it, which a warp takes two to
// four cycles for: a page takes 17 us for 128 rows (FMA pipe alone: 8.6), 8 for 64, 9.5 for two CTAs of 32.  Scores and outputs of
// 8 x 4 or 8 x 8 a thread read less and left too few warps or registers: the same times.  Measured, D = 128: 16 heads of their own,
// 16 sequences after 8192 tokens 76 us (one tile of 64 rows: 129, regular attention 402); 32 heads over 8, 64 sequences 266 (959).
template <int D, int ROWS>
struct CGeo {
    static constexpr int THREADS = 4 * ROWS, CTAS = ROWS <= 32 ? 2 : 1;  // per SM
    static constexpr int LD = D + 4;             // pitch of the query rows in floats: 16-byte aligned, successive rows 4 banks apart
    static constexpr int PL = PAGE_TOKENS + 16;  // the same of the scores, 16 banks apart
    static constexpr size_t SMEM = (2 * (size_t)PAGE_TOKENS * D + (size_t)ROWS * (LD + PL) + 3 * ROWS) * 4 + 32;
    static_assert(CTAS * (SMEM + 1024) <= 227 * 1024, "shared memory of an SM");
};

template <int D, int ROWS>
__global__ void __launch_bounds__(4 * ROWS, ROWS <= 32 ? 2 : 1) prefix_simt_kernel(const __grid_constant__ PrefixParams p, const __grid_constant__ PrefixBatch pb) {
    using GEO = CGeo<D, ROWS>;
    constexpr int LD = GEO::LD, PL = GEO::PL, CPT = D / 16;
    extern __shared__ __align__(16) float csm[];
    float* k_s = csm;                     // the chunks as they lie in the page: planes of 32 channels, [64 tokens][8 units of 4], the
    float* v_s = k_s + PAGE_TOKENS * D;   //   units of a token in the order unit ^ token % 8
    float* q_s = v_s + PAGE_TOKENS * D;   // [ROWS][LD]
    float* p_s = q_s + ROWS * LD;         // [ROWS][PL] scores, then weights
    float* m_s = p_s + ROWS * PL;         // [ROWS] running maximum
    float* l_s = m_s + ROWS;              // [ROWS] running sum
    float* a_s = l_s + ROWS;              // [ROWS] factor of this page's rescale
    uint64_t* bars = (uint64_t*)(a_s + ROWS);  // K, V have landed
    volatile int* fail_s = (volatile int*)(bars + 2);
    const DecodeParams& dp = p.d;
    const int tid = threadIdx.x;
    const int kvh = blockIdx.y;
    const PrefixGroup grp = prefix_group_of(pb, blockIdx.x);
    const int split = (blockIdx.x - grp.cta0) / grp.tiles, tile = (blockIdx.x - grp.cta0) % grp.tiles;
    int page0, n_pages;
    prefix_run(grp, grp.splits, split, &page0, &n_pages);
    const int n_rows = grp.n_seqs * dp.G, row0 = tile * ROWS;
    const int32_t* pages = dp.table + (int64_t)grp.trow * dp.max_pages_per_seq + page0;
    const int n_copy = (int)blockIdx.x == dp.stall_item && kvh == 0 ? 0 : n_pages;  // test hook, see DecodeParams
    auto fetch = [&](int i, int x) {  // thread 0: K (x = 0) or V of page i of the run
        if (i >= n_copy) return;
        int32_t pg = pages[i];
        if (pg < 0 || pg >= dp.n_pages) {
            atomicOr(dp.status, STATUS_PAGE_OOB);
            pg = 0;
        }
        constexpr uint32_t BYTES = PAGE_TOKENS * D * 4;
        mbar_expect_tx(&bars[x], BYTES);
        bulk_g2s(x ? v_s : k_s, dp.pool + (int64_t)pg * dp.page_bytes + (int64_t)kvh * (2 * p.chunk_bytes) + x * p.chunk_bytes, BYTES, &bars[x]);
    };
    if (tid == 0) {
        mbar_init(&bars[0], 1), mbar_init(&bars[1], 1);
        *fail_s = 0;
        mbar_fence_init();
    }
    grid_dependency_wait();
    grid_launch_dependents();
    if (tid == 0) fetch(0, 0), fetch(0, 1);
    for (int i0 = tid; i0 < ROWS * D; i0 += 8 * GEO::THREADS) {  // eight on their way before the first is stored
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int r = (i0 + j * GEO::THREADS) / D, ch = (i0 + j * GEO::THREADS) % D;
            v[j] = row0 + r < n_rows ? load_query(dp, D, grp.b0 + (row0 + r) / dp.G, kvh * dp.G + (row0 + r) % dp.G, ch) : 0.f;
        }
#pragma unroll
        for (int j = 0; j < 8; j++) q_s[(i0 + j * GEO::THREADS) / D * LD + (i0 + j * GEO::THREADS) % D] = v[j];
    }
    if (tid < ROWS) m_s[tid] = -INFINITY, l_s[tid] = 0.f;
    const int tx = tid & 15, ty = tid >> 4;  // rows ty + (ROWS / 4) {0 .. 3}
    uint64_t acc[4][CPT / 2] = {};           // their outputs, pairs of channels
    __syncthreads();          // the queries are there, and the barriers

    for (int i = 0; i < n_pages; i++) {
        wait_or_fail(&bars[0], i & 1, fail_s, dp.wait_ns);
        {  // scores against keys tx + 16 {0 .. 3}
            uint64_t s[4][4] = {};  // the sums over even and over odd channels
#pragma unroll 2
            for (int c = 0; c < D; c += 4) {
                ulonglong2 qv[4], kv[4];
#pragma unroll
                for (int r = 0; r < 4; r++) qv[r] = *(const ulonglong2*)(q_s + (ty + ROWS / 4 * r) * LD + c);
#pragma unroll
                for (int k = 0; k < 4; k++) kv[k] = *(const ulonglong2*)(k_s + (c >> 5) * (PAGE_TOKENS * 32) + (tx + 16 * k) * 32 + ((c & 31) ^ ((tx & 7) << 2)));
#pragma unroll
                for (int r = 0; r < 4; r++)
#pragma unroll
                    for (int k = 0; k < 4; k++) s[r][k] = f2_fma(qv[r].y, kv[k].y, f2_fma(qv[r].x, kv[k].x, s[r][k]));
            }
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const float2 x = f2_unpack(s[r][k]);
                    p_s[(ty + ROWS / 4 * r) * PL + tx + 16 * k] = (x.x + x.y) * dp.scale;
                }
        }
        __syncthreads();
        if (tid == 0) fetch(i + 1, 0);
        {  // softmax of the page: four neighbouring threads own a row, quads of keys in turn
            const int r = tid >> 2, part = tid & 3;
            float4 x[4];
            float mx = -INFINITY;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                x[e] = *(const float4*)(p_s + r * PL + 4 * (part + 4 * e));
                mx = fmaxf(mx, fmaxf(fmaxf(x[e].x, x[e].y), fmaxf(x[e].z, x[e].w)));
            }
#pragma unroll
            for (int o = 2; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            const float m_old = m_s[r], m_new = fmaxf(m_old, mx), m_use = m_new == -INFINITY ? 0.f : m_new;
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float4 w = make_float4(expf(x[e].x - m_use), expf(x[e].y - m_use), expf(x[e].z - m_use), expf(x[e].w - m_use));
                *(float4*)(p_s + r * PL + 4 * (part + 4 * e)) = w;
                sum += (w.x + w.y) + (w.z + w.w);
            }
#pragma unroll
            for (int o = 2; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            __syncwarp();  // every lane has read the old maximum of its row
            if (part == 0) {
                const float a = expf(m_old - m_use);
                a_s[r] = a, m_s[r] = m_new, l_s[r] = fmaf(l_s[r], a, sum);
            }
        }
        wait_or_fail(&bars[1], i & 1, fail_s, dp.wait_ns);
        __syncthreads();
        {  // values: channels tx * 4 + 64 j .. + 3
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float a = a_s[ty + ROWS / 4 * r];
#pragma unroll
                for (int e = 0; e < CPT / 2; e++) acc[r][e] = f2_mul(acc[r][e], f2_pack(a, a));
            }
#pragma unroll 1
            for (int t = 0; t < PAGE_TOKENS; t += 4) {
                float4 w[4];
#pragma unroll
                for (int r = 0; r < 4; r++) w[r] = *(const float4*)(p_s + (ty + ROWS / 4 * r) * PL + t);
#pragma unroll
                for (int k = 0; k < 4; k++)
#pragma unroll
                    for (int j = 0; j < CPT / 4; j++) {
                        const int c = tx * 4 + 64 * j;
                        const ulonglong2 v = *(const ulonglong2*)(v_s + (c >> 5) * (PAGE_TOKENS * 32) + (t + k) * 32 + ((c & 31) ^ (((t & 4) + k) << 2)));
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            const float x = k == 0 ? w[r].x : k == 1 ? w[r].y : k == 2 ? w[r].z : w[r].w;
                            acc[r][2 * j] = f2_fma(f2_pack(x, x), v.x, acc[r][2 * j]), acc[r][2 * j + 1] = f2_fma(f2_pack(x, x), v.y, acc[r][2 * j + 1]);
                        }
                    }
            }
        }
        __syncthreads();
        if (tid == 0) fetch(i + 1, 1);
    }
    __syncthreads();
    if (*fail_s) {  // an empty partial, once the copies in flight have landed
        if (tid == 0) atomicOr(dp.status, STATUS_WAIT_EXPIRED);
        if (tid < ROWS) m_s[tid] = -INFINITY, l_s[tid] = 0.f;
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int e = 0; e < CPT / 2; e++) acc[r][e] = 0ull;
        __nanosleep(200000);
        __syncthreads();
    }
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const int row = ty + ROWS / 4 * r, my_row = row0 + row;
        if (my_row >= n_rows) continue;
        const int64_t rec = (int64_t)grp.base + ((int64_t)split * dp.Hkv + kvh) * n_rows + my_row;
#pragma unroll
        for (int j = 0; j < CPT / 4; j++) *(ulonglong2*)(dp.part_o + rec * D + tx * 4 + 64 * j) = make_ulonglong2(acc[r][2 * j], acc[r][2 * j + 1]);
        if (tx == 0) *(float2*)(dp.part_ml + rec * 2) = make_float2(m_s[row], l_s[row]);
    }
}

// ---- join the partials of the shared pages and of the sequence's own ------------------------------------------------------
struct SharedBatch {
    int4 pre[INLINE_BATCH];  // per batch entry: {first record of its group, runs of the group, rows of the group, its first row}
};
struct SharedCombineParams {
    const float* part_o;
    const float* part_ml;
    void* out;  // may be null when `act` is given
    int64_t ob, oh;
    int32_t Hkv, G, dtype, n_rows;
    uint8_t* act;  // the result as the quantised activation of a W4A8 GEMM, or null (see combine_kernel of decode.cu)
    int* act_status;
};

// One CTA per (sequence, query head), one thread per channel; at most MAX_SPLITS partials.
template <int D>
__global__ void __launch_bounds__(D) combine_shared_kernel(SharedCombineParams p, const __grid_constant__ InlineBatch ib, const __grid_constant__ SharedBatch sb) {
    __shared__ float m_s[MAX_SPLITS], l_s[MAX_SPLITS], w_s[MAX_SPLITS];
    const int b = blockIdx.x, hq = blockIdx.y, ch = threadIdx.x;
    const int kvh = hq / p.G, g = hq % p.G;
    grid_dependency_wait();
    const int64_t act_nb = (int64_t)p.Hkv * p.G * D / QK, act_blk = (int64_t)hq * (D / QK) + (ch >> 5);
    if (p.act) {  // a warp holds one block of 32 columns of row b
        if (b == 0 && hq == 0 && ch == 0) q40_status_begin(p.act_status);
        if (b >= p.n_rows) {
            q40_quantize_block(0.f, false, p.act, p.n_rows, act_nb, b, act_blk, ch & 31);
            return;
        }
    }
    const int4 own = ib.ent[b], pre = sb.pre[b];
    const int n_own = own.w, n = n_own + pre.y;
    auto record = [&](int k) -> int64_t {
        return k < n_own ? ((int64_t)(own.z + k) * p.Hkv + kvh) * p.G + g
                         : (int64_t)pre.x + ((int64_t)(k - n_own) * p.Hkv + kvh) * pre.z + pre.w + g;
    };
    float v[8];  // the first partial outputs do not depend on the weights: they travel while the weights are made
#pragma unroll
    for (int k = 0; k < 8; k++) v[k] = (k < n) ? p.part_o[record(k) * D + ch] : 0.f;
    if (ch < n) {
        const float2 ml = *(const float2*)(p.part_ml + record(ch) * 2);
        m_s[ch] = ml.x, l_s[ch] = ml.y;
    }
    __syncthreads();
    float M = -INFINITY;
    for (int k = 0; k < n; k++) M = fmaxf(M, m_s[k]);
    if (ch < n) w_s[ch] = expf(m_s[ch] - M);
    __syncthreads();
    float den = 0.f, num = 0.f;
    for (int k = 0; k < n; k++) den = fmaf(w_s[k], l_s[k], den);
#pragma unroll
    for (int k = 0; k < 8; k++) num = fmaf((k < n) ? w_s[k] : 0.f, v[k], num);
#pragma unroll 1
    for (int k0 = 8; k0 < n; k0 += 8) {
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = (k0 + k < n) ? p.part_o[record(k0 + k) * D + ch] : 0.f;
#pragma unroll
        for (int k = 0; k < 8; k++) num = fmaf((k0 + k < n) ? w_s[k0 + k] : 0.f, v[k], num);
    }
    const float res = num / den;
    if (p.out) st_from_f32(p.out, p.dtype, (int64_t)b * p.ob + (int64_t)hq * p.oh + ch, res);
    if (p.act) q40_quantize_block(round_to_dtype(res, p.dtype), true, p.act, p.n_rows, act_nb, b, act_blk, ch & 31);
}

// ---- host side --------------------------------------------------------------------------------------------------------

// Pages that two sequences share at their beginning.  Pages are only ever shared at the same place of a sequence and with
// everything before them (b200kv_fork_shared), so the shared ones come first.  A page that is not full for one of them is its
// last one and never shared for long (an append moves it); it does not count.
static int shared_pages(const SeqState& a, const SeqState& b) {
    if (a.start > 0 || b.start > 0) return 0;  // the front of a trimmed sequence is gone
    int lo = 0, hi = (int)std::min(a.len / PAGE_TOKENS, b.len / PAGE_TOKENS);
    while (lo < hi) {  // pages [0, lo) are the same, page hi (if there is one) is not
        const int mid = (lo + hi) / 2;
        if (a.pages[mid] == b.pages[mid]) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

struct Run {
    int b0, n, pages;
};
// Cuts the batch into runs of neighbours and gives each the pages that all of its sequences share: from the left, always the
// run that saves most page reads, (n - 1) * pages.
static std::vector<Run> shared_runs(const b200kv_cache* c, int32_t n_seqs, const int32_t* seqs) {
    std::vector<int> with_next((size_t)n_seqs, 0);
    for (int i = 0; i + 1 < n_seqs; i++) with_next[i] = shared_pages(c->seqs[seqs[i]], c->seqs[seqs[i + 1]]);
    std::vector<Run> runs;
    for (int i = 0; i < n_seqs;) {
        Run best{i, 1, 0};
        int64_t best_saved = 0;
        int pages = with_next[i];
        for (int j = i + 1; j < n_seqs && pages > 0; j++) {
            if ((int64_t)(j - i) * pages > best_saved) best = {i, j - i + 1, pages}, best_saved = (int64_t)(j - i) * pages;
            pages = std::min(pages, with_next[j]);
        }
        runs.push_back(best);
        i += best.n;
    }
    return runs;
}

template <bool ALT, int D, int SRC>
static cudaError_t launch_prefix_tc_t(const PrefixParams& p, const PrefixBatch& pb, int ctas, cudaStream_t stream) {
    using GEO = XGeo<ALT, D, SRC>;
    cudaError_t e = allow_shared_memory<prefix_tc_kernel<ALT, D, SRC>>(GEO::SMEM);
    if (e != cudaSuccess) return e;
    return launch_after_predecessor(prefix_tc_kernel<ALT, D, SRC>, dim3((unsigned)ctas, (unsigned)p.d.Hkv), dim3(GEO::THREADS), GEO::SMEM, stream, p, pb);
}
template <int D, int SRC>
static cudaError_t launch_prefix_tc_rows(bool one_tile, const PrefixParams& p, const PrefixBatch& pb, int ctas, cudaStream_t stream) {
    return one_tile ? launch_prefix_tc_t<true, D, SRC>(p, pb, ctas, stream) : launch_prefix_tc_t<false, D, SRC>(p, pb, ctas, stream);
}
static cudaError_t launch_prefix_tc(int fmt, int D, bool one, const PrefixParams& p, const PrefixBatch& pb, int ctas, cudaStream_t stream) {
    if (fmt == B200KV_FMT_Q8_1) return D == 128 ? launch_prefix_tc_rows<128, PSRC_Q8>(one, p, pb, ctas, stream) : launch_prefix_tc_rows<64, PSRC_Q8>(one, p, pb, ctas, stream);
    if (fmt == B200KV_FMT_Q4_0) return D == 128 ? launch_prefix_tc_rows<128, PSRC_Q4>(one, p, pb, ctas, stream) : launch_prefix_tc_rows<64, PSRC_Q4>(one, p, pb, ctas, stream);
    return D == 128 ? launch_prefix_tc_rows<128, PSRC_PAGES16>(one, p, pb, ctas, stream) : launch_prefix_tc_rows<64, PSRC_PAGES16>(one, p, pb, ctas, stream);
}
template <int D, int ROWS>
static cudaError_t launch_prefix_simt_t(const PrefixParams& p, const PrefixBatch& pb, int ctas, cudaStream_t stream) {
    using GEO = CGeo<D, ROWS>;
    cudaError_t e = allow_shared_memory<prefix_simt_kernel<D, ROWS>>(GEO::SMEM);
    if (e != cudaSuccess) return e;
    return launch_after_predecessor(prefix_simt_kernel<D, ROWS>, dim3((unsigned)ctas, (unsigned)p.d.Hkv), dim3(GEO::THREADS), GEO::SMEM, stream, p, pb);
}
static cudaError_t launch_prefix_simt(int D, int rows_cta, const PrefixParams& p, const PrefixBatch& pb, int ctas, cudaStream_t stream) {
    if (rows_cta > 64) return D == 128 ? launch_prefix_simt_t<128, 128>(p, pb, ctas, stream) : launch_prefix_simt_t<64, 128>(p, pb, ctas, stream);
    if (rows_cta > 32) return D == 128 ? launch_prefix_simt_t<128, 64>(p, pb, ctas, stream) : launch_prefix_simt_t<64, 64>(p, pb, ctas, stream);
    return D == 128 ? launch_prefix_simt_t<128, 32>(p, pb, ctas, stream) : launch_prefix_simt_t<64, 32>(p, pb, ctas, stream);
}

// The three ways of a call, and what each takes in microseconds, fitted to grids of 2 to 64 sequences after 512 to 16384 tokens
// and to some hundred calls of random sizes.  Of 196 calls, 160 of them of random sizes, the choice is within 10% of the best of the
// three for 186, the median the best itself; at worst 1.5 times (2 f32 sequences of 16 heads of their own after 748 tokens: 17.3, alone 11.4).
//   ALONE      launch_decode: every sequence reads its pages from L2 or HBM, 8 (4) rows at a time.  No more to set up than
//              regular attention, but each page is worked on n times.
//   TOGETHER   one launch of the decode kernel, the shared pages being further work items: rows of several sequences fill the
//              row tiles that a group of few heads leaves half empty, and the own pages need no launch of their own.  Each CTA
//              of rows reads the pages again.
//   APART      the shared pages through the kernels above, every row at once, the own pages beside them.
// 32 heads over 8, f16 D = 128, alone / together / apart: 2 sequences after 1024 tokens 8.8 / 10.4 / 13.5; 8 after 4096
// 18.9 / 16.3 / 17.0; 4 after 16384 28.0 / 22.7 / 24.4; 32 after 16384 176 / 148 / 30.
enum Way { ALONE, TOGETHER, APART };
struct WaySizes {
    int fmt, D, Hkv, G, n_seqs, max_rows;
    bool use_mma, tc;                       // the tensor-core forms of the decode kernel and of the kernel over shared pages
    int64_t alone, together, apart, own;    // pages x row tiles, per kv head: 8 (4) rows of the decode kernels, XM .. of the others
};
// A page against one row tile of a decode kernel, spread over the GPU: tensor cores 2.6 ns; CUDA cores by the page's bytes and the
// work of widening them, a single row three quarters of four.
static double decode_unit(int fmt, int D, int G, bool use_mma) {
    if (use_mma) return 2.6e-3;
    return (fmt == B200KV_FMT_F32 ? 17e-3 : fmt_is_block_quant(fmt) ? 9e-3 : 14e-3) * D / 128 * (G == 1 ? 0.75 : 1.0);
}
static Way shared_way(const b200kv_cache* c, const WaySizes& z) {
    const bool quant = fmt_is_block_quant(z.fmt);
    const double unit = decode_unit(z.fmt, z.D, z.G, z.use_mma);
    const double own = unit * (double)z.own * z.Hkv;
    double alone = 6.5 + unit * (double)z.alone * z.Hkv;
    const int64_t slots = 148 * decode_ctas_per_sm(c, z.use_mma);
    // with more sequences than one CTA each can be resident, 16-bit pages go in several short rounds (44 sequences after 463
    // tokens: 25, 36 of them: 14; 28 after 153, with 16 heads: 14)
    const int64_t own_ctas = (int64_t)z.n_seqs * z.Hkv * ((z.G + (z.use_mma ? 7 : 3)) / (z.use_mma ? 8 : 4));
    if (z.use_mma && !quant && own_ctas > slots) alone += std::min(10.0, 1.2 * (double)z.alone * z.Hkv / (double)own_ctas);
    double together = 8.4 + 1.15 * unit * (double)z.together * z.Hkv + own, apart = 1e30;
    // each sequence's own pages are CTAs of that launch, however few they are: many of them crowd out the shared pages (8 heads
    // without groups after 4096 tokens: 16 sequences take 16, 32 of them 56), until they are too many to be resident together and
    // all CTAs become short (48 sequences after 1024: 20)
    if (own_ctas > slots) together *= 1.6;
    else if (own_ctas > slots / 2) together = 1e30;
    if (z.tc)  // a page for all rows of a CTA, on 148 of them; 2.4 is fitted to whole calls with two tiles of rows (larger query tiles and
               // joins, and pages at 1.5 to 1.75 times the pace of one tile)
        apart = (quant ? 15.0 : 13.0) + (quant ? 1.3 : 0.9) * (z.max_rows <= XM ? 1.0 : 2.4) * (double)z.apart * z.Hkv / 148 + own;
    else if (z.fmt == B200KV_FMT_F32) {  // a page and tile, in whole rounds of the resident CTAs; then the own pages, which find no room beside them
        const int64_t resident = z.max_rows <= 32 ? 2 * 148 : 148;
        apart = 8.0 + (z.max_rows <= 32 ? 9.5 : z.max_rows <= 64 ? 8.0 : 17.0) * (z.D == 128 ? 1.0 : 0.6) * (double)((z.apart * z.Hkv + resident - 1) / resident) +
                7.0 * (double)own_ctas / 148;
    }
    if (apart < together && apart < alone) return APART;
    return together < alone ? TOGETHER : ALONE;
}

// At most INLINE_BATCH sequences; `ends` as launch_decode takes it.
static int launch_shared(b200kv_cache* c, int32_t n_seqs, const int32_t* seqs, int32_t n_q_heads, const void* q, const int64_t* qs, void* out,
                         const int64_t* os, int32_t dtype, float scale, cudaStream_t stream, const QueryRope& ends) {
    const int Hkv = c->L.Hkv, D = c->L.D, G = n_q_heads / Hkv;
    std::vector<Run> runs = shared_runs(c, n_seqs, seqs);
    bool any = false;
    for (const Run& r : runs) any |= r.n > 1 && r.pages > 0;
    if (!any) return launch_decode(c, n_seqs, seqs, n_q_heads, q, qs, out, os, dtype, scale, stream, 0, &ends);

    // ---- the shared pages: which kernel, how many rows to a CTA ----
    const int fmt = c->L.fmt;
    const bool quant = fmt_is_block_quant(fmt);
    const bool q_rows16 = (uintptr_t)q % 16 == 0 && qs[0] % 8 == 0 && qs[1] % 8 == 0;
    const bool tc = dtype != B200KV_F32 && (quant || fmt == dtype) && q_rows16 && !c->force_simt;
    int max_rows = 0, max_pages = 1;
    for (const Run& r : runs)
        if (r.n > 1 && r.pages > 0) max_rows = std::max(max_rows, r.n * G), max_pages = std::max(max_pages, r.pages);
    const bool one_tile = max_rows <= XM;
    const int cluster = tc ? X_CLUSTER : 1;                  // CTAs that write one partial
    int rows_cta = tc ? (one_tile ? XM : 2 * XM) : (max_rows > 64 ? 128 : max_rows > 32 ? 64 : 32);
    int64_t slots = tc ? 148 / X_CLUSTER : rows_cta == 32 ? 2 * 148 : 148;  // resident CTAs, or clusters

    // ---- the own pages of every sequence: as launch_decode cuts them, starting behind the shared ones ----
    const bool use_mma = decode_mma_supported(fmt, D, dtype) && !c->force_simt;
    const int nz = (G + (use_mma ? 7 : 3)) / (use_mma ? 8 : 4);
    std::vector<int64_t> first((size_t)n_seqs), own_pages((size_t)n_seqs);
    std::vector<int> most((size_t)n_seqs, MAX_SPLITS);  // runs of a sequence's own pages: a row joins at most MAX_SPLITS partials
    for (const Run& r : runs)
        for (int i = r.b0; i < r.b0 + r.n; i++) {
            const SeqState& s = c->seqs[seqs[i]];
            first[i] = r.n > 1 && r.pages > 0 ? (int64_t)r.pages * PAGE_TOKENS : s.start;
            if (r.n > 1 && r.pages > 0) most[i] = MAX_SPLITS / 2;
            own_pages[i] = (s.len + PAGE_TOKENS - 1) / PAGE_TOKENS - first[i] / PAGE_TOKENS;
        }
    const int dec_rows = use_mma ? 8 : 4;
    WaySizes z{fmt, D, Hkv, G, n_seqs, max_rows, use_mma, tc, 0, 0, 0, 0};
    for (const Run& r : runs)
        if (r.n > 1 && r.pages > 0) {
            z.alone += (int64_t)r.n * nz * r.pages, z.together += (int64_t)((r.n * G + dec_rows - 1) / dec_rows) * r.pages;
            z.apart += (int64_t)((r.n * G + rows_cta - 1) / rows_cta) * r.pages;
        }
    for (int64_t x : own_pages) z.own += x * nz;
    z.alone += z.own;
    const Way way = c->shared_way == 0 ? shared_way(c, z) : c->shared_way == 2 && (tc || fmt == B200KV_FMT_F32) ? APART : TOGETHER;
    if (way == ALONE) return launch_decode(c, n_seqs, seqs, n_q_heads, q, qs, out, os, dtype, scale, stream, 0, &ends);
    const bool together = way == TOGETHER;
    if (together) rows_cta = nz * dec_rows;
    // The own pages run beside the shared ones, on the SMs that these leave: each gets its share of the work, in microseconds of
    // an SM per page and head: 1.0 to 1.2 for a tile pair; for an own page 0.75 for each 32 KB at the copy rate, or what the decode
    // kernel takes (15 sequences of 7 heads a group with up to 200 own 4-bit tokens of D = 64: 23.2 us when this took the bytes alone, 18.8 now).
    if (tc && !together) {
        int64_t own = 0, shared = 0;
        for (int i = 0; i < n_seqs; i++) own += own_pages[i];
        for (const Run& r : runs)
            if (r.n > 1 && r.pages > 0) shared += (int64_t)((r.n * G + rows_cta - 1) / rows_cta) * r.pages;
        const double page_us = std::max(2.0 * c->L.chunk_bytes / 32768.0 * 0.75, decode_unit(fmt, D, G, use_mma) * 148 * nz);
        const double own_us = (double)own * page_us, shared_us = (double)shared * 1.1;
        slots = std::max<int64_t>(slots / 4, (int64_t)(slots * shared_us / (shared_us + own_us)));
    }
    std::vector<int64_t> all_pages = own_pages;
    if (together)
        for (const Run& r : runs)
            if (r.n > 1 && r.pages > 0) all_pages.insert(all_pages.end(), (size_t)((r.n * G + rows_cta - 1) / rows_cta), r.pages);
    int64_t own_chunk = pages_per_split(c, all_pages.data(), (int)all_pages.size(), use_mma, nz);

    InlineBatch ib{};
    SharedBatch sb{};
    PrefixBatch pb{};
    int n_items = 0, ctas = 0;
    int64_t n_rec = 0, run_pages = 1;
    if (together) run_pages = std::min<int64_t>(own_chunk, max_pages);
    else
        for (;; run_pages++) {  // the shortest runs for which every CTA is resident: a run is `cluster` CTAs' pages
            int64_t n = 0;
            for (const Run& r : runs)
                if (r.n > 1 && r.pages > 0) n += (int64_t)((r.n * G + rows_cta - 1) / rows_cta) * ((r.pages + run_pages - 1) / run_pages);
            if (n * Hkv <= slots || run_pages >= max_pages) break;
        }
    for (;;) {
        ib = InlineBatch{};
        pb = PrefixBatch{};
        n_items = 0, ctas = 0;
        for (int i = 0; i < n_seqs; i++) {
            const int splits = own_pages[i] ? (int)std::min<int64_t>(most[i], (own_pages[i] + own_chunk - 1) / own_chunk) : 0;
            ib.ent[i] = make_int4(seqs[i], (int)c->seqs[seqs[i]].len, n_items, splits);
            ib.first[i] = (int32_t)first[i];
            n_items += splits;
        }
        ib.n = n_seqs;
        n_rec = (int64_t)n_items * Hkv * G;
        if (together) pb.n_own = ctas = n_items;
        for (const Run& r : runs) {
            if (r.n <= 1 || r.pages <= 0) continue;
            const int rows = r.n * G;
            PrefixGroup& g = pb.g[pb.n++];
            g.trow = seqs[r.b0], g.n_pages = r.pages, g.b0 = r.b0, g.n_seqs = r.n;
            g.tiles = (rows + rows_cta - 1) / rows_cta;
            int own_splits = 0;  // a row joins at most MAX_SPLITS partials
            for (int i = r.b0; i < r.b0 + r.n; i++) own_splits = std::max(own_splits, ib.ent[i].w);
            g.splits = (int)std::min<int64_t>(MAX_SPLITS - own_splits, (r.pages + run_pages - 1) / run_pages);
            g.cta0 = ctas, g.base = (int32_t)n_rec;
            for (int i = 0; i < r.n; i++) sb.pre[r.b0 + i] = make_int4(g.base, g.splits, rows, i * G);
            ctas += g.tiles * g.splits * (together ? 1 : cluster);
            n_rec += (int64_t)g.splits * Hkv * rows;
        }
        if ((size_t)n_rec * (D + 2) * sizeof(float) <= c->ws_bytes) break;  // sized once, at create: longer runs where it is small
        bool longest = run_pages >= max_pages;
        for (int i = 0; i < n_seqs; i++) longest &= own_pages[i] <= own_chunk;
        if (longest)  // the partials of the shared pages beside those of the own ones do not fit: regular attention needs half of them
            return launch_decode(c, n_seqs, seqs, n_q_heads, q, qs, out, os, dtype, scale, stream, 0, &ends);
        run_pages += std::max<int64_t>(1, run_pages / 4);
        own_chunk += std::max<int64_t>(1, own_chunk / 4);
    }

    PrefixParams p{};
    DecodeParams& dp = p.d;
    dp.pool = c->pool, dp.table = c->d_table, dp.status = c->d_status;
    dp.q = q, dp.qb = qs[0], dp.qh = qs[1];
    if (ends.cos) dp.q_cos = ends.cos, dp.q_sin = ends.sin, dp.rope_b = ends.stride_b;
    dp.part_o = (float*)c->ws, dp.part_ml = dp.part_o + n_rec * D;
    dp.page_bytes = c->L.page_bytes, dp.n_pages = (int32_t)c->n_pages, dp.max_pages_per_seq = c->max_pages_per_seq;
    dp.Hkv = Hkv, dp.G = G, dp.dtype = dtype, dp.scale = scale, dp.wait_ns = c->wait_ns;
    if (c->stall_next_decode) dp.stall_item = 0, dp.wait_ns = 1000000, c->stall_next_decode = false;  // one call, 1 ms
    p.chunk_bytes = c->L.chunk_bytes, p.skip_fraction = X_SKIP_FRACTION;
    cudaError_t e = cudaSuccess;
    if (!together) {
        ProfScope ps(c, K_PREFIX, stream);
        e = tc ? launch_prefix_tc(fmt, D, one_tile, p, pb, ctas, stream)
               : launch_prefix_simt(D, rows_cta, p, pb, ctas, stream);
    }
    if (e != cudaSuccess) return fail("shared-prefix launch failed: %s", cudaGetErrorString(e));
    if (together || n_items > 0) {
        ProfScope ps(c, K_DECODE, stream);
        dp.beside = !together;
        if (!together) dp.stall_item = -1;  // the launch before took the hook
        const PrefixBatch* with = together ? &pb : nullptr;
        const int more = together ? ctas - n_items : 0;
        if ((use_mma ? launch_decode_mma(fmt, dp, n_items, stream, &ib, with, more) : launch_decode_simt(fmt, D, dp, n_items, stream, &ib, with, more)) != B200KV_OK)
            return B200KV_KO;
    }
    SharedCombineParams cp{};
    cp.part_o = dp.part_o, cp.part_ml = dp.part_ml, cp.out = out, cp.ob = os[0], cp.oh = os[1];
    cp.Hkv = Hkv, cp.G = G, cp.dtype = dtype, cp.n_rows = n_seqs;
    if (ends.act_scratch) cp.act = (uint8_t*)ends.act_scratch + Q_HEADER, cp.act_status = (int*)ends.act_scratch;
    const unsigned rows = cp.act ? (unsigned)((n_seqs + 7) / 8 * 8) : (unsigned)n_seqs;
    {
        ProfScope ps(c, K_COMBINE, stream);
        e = D == 128 ? launch_after_predecessor(combine_shared_kernel<128>, dim3(rows, n_q_heads), dim3(128), 0, stream, cp, ib, sb)
                     : launch_after_predecessor(combine_shared_kernel<64>, dim3(rows, n_q_heads), dim3(64), 0, stream, cp, ib, sb);
    }
    if (e != cudaSuccess) return fail("combine launch failed: %s", cudaGetErrorString(e));
    return B200KV_OK;
}

}  // namespace b200kv

using namespace b200kv;

extern "C" int b200kv_attend_shared(b200kv_cache* c, int32_t n_seqs, const int32_t* seqs, int32_t n_q_heads, const void* q,
                                    const int64_t q_strides[3], const void* cos, const void* sin, int64_t rope_stride, void* out,
                                    const int64_t out_strides[3], void* scratch, int32_t dtype, float scale, void* stream_) {
    if (validate_seqs(c, n_seqs, seqs) != B200KV_OK) return B200KV_KO;
    if (!c->L.has_v) return fail("this cache holds one tensor only: attention needs K and V");
    if (fmt_is_kivi(c->L.fmt)) return fail("the sequences of a KIVI cache share no pages: use b200kv_attend");
    if (!q || !q_strides || (!out && !scratch) || (out && !out_strides)) return fail("null tensor or strides");
    if ((cos == nullptr) != (sin == nullptr)) return fail("cos and sin come together");
    if ((uintptr_t)scratch % 16) return fail("scratch must be 16-byte aligned");
    if (n_q_heads <= 0 || n_q_heads % c->L.Hkv != 0)
        return fail("n_q_heads (%d) must be a positive multiple of n_kv_heads (%d)", n_q_heads, c->L.Hkv);
    if (dtype < B200KV_F32 || dtype > B200KV_BF16) return fail("unknown dtype %d", dtype);
    for (int i = 0; i < n_seqs; i++)
        if (c->seqs[seqs[i]].len <= 0) return fail("sequence %d is empty: nothing to attend to", seqs[i]);
    if (scale <= 0.f) scale = 1.0f / sqrtf((float)c->L.D);
    cudaStream_t stream = (cudaStream_t)stream_;
    DeviceGuard guard(c->cfg.device);
    const int64_t no_strides[3] = {0, 0, 0};
    const int64_t* os = out ? out_strides : no_strides;
    const QueryRope ends{cos, sin, rope_stride, scratch};
    if (n_seqs <= INLINE_BATCH) return launch_shared(c, n_seqs, seqs, n_q_heads, q, q_strides, out, os, dtype, scale, stream, ends);
    // the quantised activation of a larger batch is laid out for all of its rows at once: the regular call writes it
    if (scratch) return launch_decode(c, n_seqs, seqs, n_q_heads, q, q_strides, out, os, dtype, scale, stream, 0, &ends);
    const int esz = dtype_size(dtype);
    for (int at = 0; at < n_seqs; at += INLINE_BATCH) {
        const QueryRope part{cos ? (const uint8_t*)cos + (int64_t)at * rope_stride * esz : nullptr,
                             sin ? (const uint8_t*)sin + (int64_t)at * rope_stride * esz : nullptr, rope_stride, nullptr};
        if (launch_shared(c, std::min(INLINE_BATCH, n_seqs - at), seqs + at, n_q_heads, (const uint8_t*)q + (int64_t)at * q_strides[0] * esz, q_strides,
                          (uint8_t*)out + (int64_t)at * os[0] * esz, os, dtype, scale, stream, part) != B200KV_OK)
            return B200KV_KO;
    }
    return B200KV_OK;
}
