// Launch parameters shared by the two decode kernels (CUDA-core and tensor-core formulations).
#pragma once
#include "internal.h"

namespace b200kv {

struct WorkItem {
    int32_t trow;        // page-table row of the sequence
    int32_t len;         // cached length of the sequence
    int32_t page_begin;  // first page of this split
    int32_t n_pages;     // pages in this split
    int32_t batch;       // batch entry
    int32_t split;       // split index inside the batch entry
    int32_t first;       // first visible token: a sliding window, or a sequence whose front pages were given back (0: all)
    int32_t pad1;
};

struct DecodeParams {
    const uint8_t* pool;
    const int32_t* table;
    const WorkItem* items;
    int* status;
    const void* q;
    int64_t qb, qh;  // q strides {batch, head} in elements
    // ApplyRope on the query as it is loaded (null: q is used as it is): rows of D values of type dtype, one per batch entry
    const void* q_cos;
    const void* q_sin;
    int64_t rope_b;  // cos / sin stride between batch entries, in elements
    float* part_o;   // [item][Hkv][G][D]   unnormalised partial outputs
    float* part_ml;  // [item][Hkv][G][2]   running max (natural-log units), running sum
    int64_t page_bytes;
    int32_t n_pages, max_pages_per_seq, Hkv, G, dtype;
    float scale;
    uint64_t wait_ns = 1000000000ull;  // limit of each bounded barrier wait
    int32_t stall_item = -1;  // -1, or (a test hook) the work item whose CTA of kv head 0 never issues its copies: its first wait
                         // runs out, it flags STATUS_WAIT_EXPIRED, publishes an empty partial and returns
    // The launch before this one (the attention over shared pages) runs beside it: nothing of it is read here, it has waited for
    // everything before itself, and one CTA of this grid ends only after it, so that who waits for this grid waits for both.
    int32_t beside = 0;
};

// Per-call batch description small enough to travel as a kernel parameter (no host-to-device copy, no
// staging slot): one entry per sequence of the call, {page-table row, cached length, first work item,
// number of splits}.  The work items are a pure function of it: split k of a sequence with `pages` pages
// covers pages [k * base + min(k, rem), ...) where base = pages / splits, rem = pages % splits.
constexpr int INLINE_BATCH = 256;
constexpr int MAX_SPLITS = 64;  // most partials per sequence the combine pass merges
struct InlineBatch {
    int32_t n;  // entries in use; 0 = the kernels read p.items / batch_info from device memory instead
    int32_t pad[3];
    int4 ent[INLINE_BATCH];
    int32_t first[INLINE_BATCH];  // first visible token of each entry (0: the whole sequence)
};

// Channel `ch` of the query row of (batch, head), after ApplyRope when the call carries cos / sin.  The rotated value is
// rounded to dtype after every operation, so it equals what a separate rope kernel would have stored and this load
// would have read back.
__device__ inline float load_query(const DecodeParams& p, int D, int batch, int head, int ch) {
    const int64_t row = (int64_t)batch * p.qb + (int64_t)head * p.qh;
    if (!p.q_cos) return ld_as_f32(p.q, p.dtype, row + ch);
    const int esz = p.dtype == B200KV_F32 ? 4 : 2;
    return rope_row_elem((const uint8_t*)p.q + row * esz, (const uint8_t*)p.q_cos + (int64_t)batch * p.rope_b * esz,
                         (const uint8_t*)p.q_sin + (int64_t)batch * p.rope_b * esz, p.dtype, D, ch);
}

__host__ __device__ inline WorkItem make_work_item(const int4& e, int batch, int k, int first = 0) {
    const int p0 = first / PAGE_TOKENS;  // pages before the first visible token are not walked (they may have been freed)
    const int pages = (e.y + PAGE_TOKENS - 1) / PAGE_TOKENS - p0;
    const int base = pages / e.w, rem = pages % e.w;
    WorkItem w;
    w.trow = e.x, w.len = e.y;
    w.page_begin = p0 + k * base + (k < rem ? k : rem);
    w.n_pages = base + (k < rem ? 1 : 0);
    w.batch = batch, w.split = k, w.first = first, w.pad1 = 0;
    return w;
}
// Work item `item` of an inline batch: binary search for the sequence that owns it.
__device__ inline WorkItem resolve_work_item(const InlineBatch& ib, int item) {
    int lo = 0, hi = ib.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (ib.ent[mid].z <= item) lo = mid;
        else hi = mid - 1;
    }
    return make_work_item(ib.ent[lo], lo, item - ib.ent[lo].z, ib.first[lo]);
}

// One run of batch entries that share their first n_pages pages.
struct PrefixGroup {
    int32_t trow;       // page-table row of one of them
    int32_t n_pages;    // shared pages, all of them full
    int32_t b0, n_seqs; // batch entries b0 .. b0 + n_seqs - 1
    int32_t tiles;      // CTAs (x) that cover the n_seqs * G rows between them
    int32_t splits;     // runs of pages, one partial each
    int32_t cta0;       // first CTA (x) of the group, after the work items of the sequences' own pages: cta0 + split * tiles + tile
    int32_t base;       // first partial record: base + (split * Hkv + kvh) * n_seqs * G + row
};
constexpr int PREFIX_GROUPS = INLINE_BATCH / 2;
struct PrefixBatch {
    int32_t n;
    int32_t n_own;  // work items of the sequences' own pages in the same launch: CTAs (x) 0 .. n_own - 1
    int32_t pad[2];
    PrefixGroup g[PREFIX_GROUPS];
};
struct NoPrefix {};  // a decode launch without shared pages
__device__ inline PrefixGroup prefix_group_of(const PrefixBatch& pb, int cta) {
    int lo = 0, hi = pb.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (pb.g[mid].cta0 <= cta) lo = mid;
        else hi = mid - 1;
    }
    return pb.g[lo];
}
// pages [first, first + count) of run k of n
__device__ inline void prefix_run(const PrefixGroup& g, int n, int k, int* first, int* count) {
    const int base = g.n_pages / n, rem = g.n_pages % n;
    *first = k * base + min(k, rem);
    *count = base + (k < rem ? 1 : 0);
}

// What a CTA of a decode kernel works on: a run of pages of one sequence against the query heads of a kv head's group, or of
// pages shared by a run of sequences against the rows (sequence, head of the group) of all of them.
struct DecodeWork {
    WorkItem w;
    int32_t row0, rows;  // first row of this CTA, rows in all: row r is query head kvh * G + r % G of batch entry w.batch + r / G
    int64_t base;        // partial record of row 0
};
template <typename SHARED>
__device__ inline DecodeWork decode_work(const DecodeParams& p, const InlineBatch& ib, const SHARED& sb, int kvh, int rows_per_cta) {
    DecodeWork d;
    if constexpr (sizeof(SHARED) > sizeof(NoPrefix)) {
        if ((int)blockIdx.x >= sb.n_own) {
            const PrefixGroup g = prefix_group_of(sb, blockIdx.x);
            const int local = (int)blockIdx.x - g.cta0, split = local / g.tiles;
            d.rows = g.n_seqs * p.G, d.row0 = (local % g.tiles) * rows_per_cta;
            prefix_run(g, g.splits, split, &d.w.page_begin, &d.w.n_pages);
            d.w.trow = g.trow, d.w.len = g.n_pages * PAGE_TOKENS, d.w.batch = g.b0, d.w.split = split, d.w.first = 0, d.w.pad1 = 0;
            d.base = (int64_t)g.base + ((int64_t)split * p.Hkv + kvh) * d.rows;
            return d;
        }
    }
    d.w = ib.n ? resolve_work_item(ib, blockIdx.x) : p.items[blockIdx.x];
    d.row0 = 0, d.rows = p.G;
    d.base = ((int64_t)blockIdx.x * p.Hkv + kvh) * p.G;
    return d;
}
__device__ inline void decode_begin(const DecodeParams& p) {
    if (!p.beside) grid_dependency_wait();  // the append that precedes this launch has written its pages
    grid_launch_dependents();               // the combine pass may be scheduled; it waits for this grid before reading partials
}
__device__ inline void decode_end(const DecodeParams& p) {
    if (p.beside && (blockIdx.x | blockIdx.y | blockIdx.z) == 0) grid_dependency_wait();
}
// load_query for row `row` of the work
template <typename SHARED>
__device__ inline float load_query_row(const DecodeParams& p, const DecodeWork& d, int D, int kvh, int row, int ch) {
    if constexpr (sizeof(SHARED) > sizeof(NoPrefix)) return load_query(p, D, d.w.batch + row / p.G, kvh * p.G + row % p.G, ch);
    else return load_query(p, D, d.w.batch, kvh * p.G + row, ch);
}

// decode.cu
int launch_decode_simt(int fmt, int D, const DecodeParams& p, int n_items, cudaStream_t stream, const InlineBatch* ib = nullptr,
                       const PrefixBatch* sb = nullptr, int shared_ctas = 0);
int launch_combine(const DecodeParams& p, const int32_t* batch_info, void* out, int64_t ob, int64_t oh, int n_seqs,
                   int n_q_heads, int D, cudaStream_t stream, const InlineBatch* ib = nullptr);
// decode_mma.cu
bool decode_mma_supported(int fmt, int D, int dtype);
int launch_decode_mma(int fmt, const DecodeParams& p, int n_items, cudaStream_t stream, const InlineBatch* ib = nullptr, const PrefixBatch* sb = nullptr,
                      int shared_ctas = 0);
// An InlineBatch with n = 0, for launches that read their batch from device memory.
const InlineBatch& empty_inline_batch();

}  // namespace b200kv
