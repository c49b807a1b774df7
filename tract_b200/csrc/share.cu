// Sequences that share the pages of a common beginning: b200kv_fork_shared, and the copy of a shared, partly filled page
// that an append makes before it writes into one.
//
// b200kv_fork (OpStateFreeze::freeze / unfreeze, gpu/src/ops/dyn_kv_cache.rs:136-168) gives the copy of a state pages of
// its own.  n continuations of one prompt never write the prompt's full pages again, so here a child takes the parent's
// full pages by reference -- the host counts the holders of every page, the device page table just names the page twice
// -- and only the last, partly filled page is copied, because parent and child both go on in it.
//
// What a call moves: one page-table row per child (4 bytes per 64 tokens), and the filled rows of the parent's last page
// per child, read once per child from L2 after the first.  It is bound by the launch: one child of a 4096-token f16
// prompt (8 kv heads of 128) is 256 bytes of table and at most 258 KB of rows, 0.1 us of HBM time.
#include <algorithm>

#include "internal.h"

namespace b200kv {

constexpr int SHARE_BATCH = 256;  // children (or page copies) per launch: the description travels as a kernel parameter

struct ShareEntry {
    int32_t parent_row, child_row;  // page-table rows (child_row < 0: no table row to copy)
    int32_t n_pages;                // entries of the row
    int32_t src, dst;               // page to copy (dst < 0: none)
    int32_t table_at;               // page-table index that takes dst
    int32_t n_tokens;               // filled slots of the page
};
struct ShareBatch {
    ShareEntry e[SHARE_BATCH];
};
struct ShareParams {
    uint8_t* pool;
    int32_t* table;
    int64_t page_bytes;
    uint32_t chunk_bytes, plane_bytes, data_bytes, plane_w;
    int32_t max_pages_per_seq;
};

// grid.y = entry.  The page is walked in 16-byte units; a 128-byte line of a plane holds 128 / plane_w token slots (the
// swizzle stays inside a line), so the lines behind the last filled slot are left out.  The scales of the block formats,
// 1/17 of a chunk, are copied whole: they interleave the slots of a pair.
__global__ void __launch_bounds__(256) share_kernel(ShareParams p, const __grid_constant__ ShareBatch batch) {
    grid_launch_dependents();
    grid_dependency_wait();  // the calls before have written the pages and the table, and are done reading the pages taken here
    const ShareEntry e = batch.e[blockIdx.y];
    const uint32_t first = blockIdx.x * blockDim.x + threadIdx.x, step = gridDim.x * blockDim.x;
    if (e.child_row >= 0) {
        const int32_t* from = p.table + (int64_t)e.parent_row * p.max_pages_per_seq;
        int32_t* to = p.table + (int64_t)e.child_row * p.max_pages_per_seq;
        const int32_t n = e.dst >= 0 ? e.n_pages - 1 : e.n_pages;  // the last entry is the copy's
        for (uint32_t i = first; i < (uint32_t)n; i += step) to[i] = from[i];
    }
    if (e.dst < 0) return;
    if (first == 0) p.table[e.table_at] = e.dst;
    const uint8_t* src = p.pool + (int64_t)e.src * p.page_bytes;
    uint8_t* dst = p.pool + (int64_t)e.dst * p.page_bytes;
    const uint32_t units = (uint32_t)(p.page_bytes / 16), filled = ((uint32_t)e.n_tokens * p.plane_w + 127u) & ~127u;
    for (uint32_t u = first; u < units; u += step) {
        const uint32_t at = (u * 16) % p.chunk_bytes;
        if (at < p.data_bytes && at % p.plane_bytes >= filled) continue;
        ((uint4*)dst)[u] = ((const uint4*)src)[u];
    }
}

static int launch_share(b200kv_cache* c, const ShareEntry* entries, int n, bool pages, cudaStream_t stream) {
    ShareParams p{};
    p.pool = c->pool, p.table = c->d_table, p.page_bytes = c->L.page_bytes, p.max_pages_per_seq = c->max_pages_per_seq;
    p.chunk_bytes = (uint32_t)c->L.chunk_bytes, p.data_bytes = (uint32_t)c->L.data_bytes, p.plane_w = (uint32_t)c->L.plane_w;
    p.plane_bytes = (uint32_t)(PAGE_TOKENS * c->L.plane_w);
    // four units of a page per thread; without pages to copy one block per entry walks the table row
    const unsigned blocks = pages ? (unsigned)std::min<int64_t>(1024, (c->L.page_bytes / 16 + 1023) / 1024) : 1u;
    ProfScope ps(c, K_SHARE, stream);
    for (int at = 0; at < n; at += SHARE_BATCH) {
        ShareBatch b;
        const int m = std::min(SHARE_BATCH, n - at);
        std::copy(entries + at, entries + at + m, b.e);
        B200KV_CUDA(launch_after_predecessor(share_kernel, dim3(blocks, (unsigned)m), dim3(256), 0, stream, p, b));
    }
    return B200KV_OK;
}

int launch_page_copies(b200kv_cache* c, const PageCopy* copies, int n, cudaStream_t stream) {
    std::vector<ShareEntry> e((size_t)n);
    for (int i = 0; i < n; i++) e[i] = {0, -1, 0, copies[i].src, copies[i].dst, copies[i].table_at, copies[i].n_tokens};
    return launch_share(c, e.data(), n, true, stream);
}

}  // namespace b200kv

using namespace b200kv;

extern "C" int b200kv_fork_shared(b200kv_cache* c, int32_t n, const int32_t* seqs, int32_t* new_seqs_out, void* stream_) {
    if (!c || !seqs || !new_seqs_out) return fail("null argument");
    if (n <= 0) return fail("need at least one sequence");
    if (fmt_is_kivi(c->L.fmt)) return fail("a KIVI cache keeps f32 rows of every sequence beside its pages: its sequences cannot share them, use b200kv_fork");
    int64_t tails = 0, slots = 0;
    for (int i = 0; i < n; i++) {
        const int s = seqs[i];
        if (s < 0 || s >= (int)c->seqs.size() || !c->seqs[s].live) return fail("sequence %d is not live", s);
        tails += c->seqs[s].len % PAGE_TOKENS != 0;
    }
    for (const SeqState& s : c->seqs) slots += !s.live;
    if (slots < n) return fail("%d new sequences, but %lld of %zu sequence slots are free", n, (long long)slots, c->seqs.size());
    if (tails > (int64_t)c->free_pages.size())
        return fail("page pool exhausted: the new sequences need %lld pages for their last tokens, %zu free", (long long)tails, c->free_pages.size());
    DeviceGuard guard(c->cfg.device);
    std::vector<ShareEntry> entries;
    entries.reserve((size_t)n);
    size_t slot = 0;
    for (int i = 0; i < n; i++) {
        while (c->seqs[slot].live) slot++;
        const SeqState& src = c->seqs[seqs[i]];
        SeqState& dst = c->seqs[slot];
        dst.live = true, dst.len = src.len, dst.start = src.start, dst.pages = src.pages;
        ShareEntry e{seqs[i], (int32_t)slot, (int32_t)src.pages.size(), -1, -1, 0, 0};
        const bool tail = src.len % PAGE_TOKENS != 0;
        for (size_t k = 0; k + (tail ? 1 : 0) < dst.pages.size(); k++)
            if (dst.pages[k] >= 0) page_share(c, dst.pages[k]);
        if (tail) {
            e.src = src.pages.back(), e.dst = dst.pages.back() = page_take(c);
            e.table_at = (int32_t)((int64_t)slot * c->max_pages_per_seq + e.n_pages - 1), e.n_tokens = (int32_t)(src.len % PAGE_TOKENS);
        }
        if (e.n_pages) entries.push_back(e);
        new_seqs_out[i] = (int32_t)slot;
    }
    if (!entries.empty() && launch_share(c, entries.data(), (int)entries.size(), tails > 0, (cudaStream_t)stream_) != B200KV_OK) {
        for (int i = 0; i < n; i++) b200kv_seq_free(c, new_seqs_out[i]);
        return B200KV_KO;
    }
    return B200KV_OK;
}
