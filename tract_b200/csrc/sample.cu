// b200kv_sample: the next token of every row of logits -- temperature, top-k, top-p, min-p -- for a given uniform number.
// It stands beside b200kv_argmax (ArgMax over the logits, examples/causal_llm/src/lib.rs:290-408 decodes greedily).
//
//   w_i = exp((x_i - max x) / T)
//   in the order of falling x, equal ones by rising index: the first k; of these the shortest beginning whose mass reaches
//   top_p x the mass of the k; of these the ones with w_i >= min_p       -- every filter keeps a beginning of the same order
//   token = the first kept index i, in rising order, with  sum_{kept j <= i} w_j > u x sum_kept w_j
//
// A token changes when u falls between a border of the distribution and its rounded value; 128k borders with the error of
// 32-bit sums would move one row in a hundred.  Weights are therefore computed in double and added up in fixed point with 44
// bits behind the point: integer sums, so that neither the order of the threads nor that of the atomics has any influence.
//
// One launch, one thread-block cluster per row, the row split over the shared memories of its CTAs: the logits are read from
// HBM once, and everything else happens on chip.
//   1. load, maximum (one exchange over the cluster).  A greedy row ends here.
//   2. the cut of top-k / top-p: a histogram over 1024 bins of log2 w (counts, and for top-p masses).  The CTAs exchange the
//      sums of 32 runs of 32 bins; then each finds the run in which the count or mass is reached and reads that run's bins
//      from the others: one cluster barrier for the whole search.
//   3. at most 1024 tokens down to the lower border of the bin: the first CTA gathers and sorts them, applies all filters
//      and draws.  At most 1024 in the bin (top-p): every CTA gathers and sorts those; the masses above the bin are known from
//      the histograms, so the CTA into whose share the draw falls finds the token alone.  Otherwise the bin is refined, by the
//      same histogram over the bit patterns in it, until the last kept token is known.
//   4. the draw over whole slices: the kept mass of every CTA, one exchange, and the CTA into whose share the draw falls
//      finds the token (also the way of rows without top-k and top-p, which start here).
// Bound: the logits once (4 bytes each in f32), and, for rows that need every weight, 9 double operations per logit and pass.
#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "internal.h"

namespace cg = cooperative_groups;

namespace b200kv {

constexpr int SP_MAX_WARPS = 32;
constexpr int SP_CLUSTER = 8;       // most CTAs of a row (the portable cluster size)
constexpr int SP_SLICE = 16384;     // logits a CTA takes before another one is added: 64 KB, two CTAs per SM
constexpr int SP_BINS = 1024;
constexpr int SP_LIST = 1024;       // tokens that are gathered
constexpr int SP_COUNT = 256;       // up to so many are put in order by counting, more by sorting
constexpr int SP_TABLE = 256;       // steps of 2^(1 / 256)
constexpr int W_BITS = 44;          // fractional bits of a weight
constexpr int SP_LIMB = 15;         // a weight enters a histogram as three 15-bit limbs: 2^17 of them fit a 32-bit counter
constexpr int MAX_VOCAB = 1 << 19;  // so many weights of 1 add up to 2^63
constexpr int MAX_ON_CHIP = SP_CLUSTER * 32768;  // 128 KB per CTA; the slices of longer rows go to the workspace
constexpr int MAX_SLICE = 1 << 17;  // logits whose limbs a 32-bit counter holds
static_assert(MAX_VOCAB <= SP_CLUSTER * MAX_SLICE, "slices of the longest rows");

typedef unsigned long long u64;

struct SampleParams {
    const void* logits;
    int64_t stride;
    int32_t dtype, n, slice, vec;  // slice: logits per CTA; vec: rows start on 16-byte boundaries
    const float* temperature;
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    const float* uniform;
    int32_t* out;
    float* scratch;  // null, or [rows][SP_CLUSTER][slice]: slices that do not fit on the chip
};

// The settings of a row, with what means "off" made explicit.
struct RowSettings {
    float t, p, min_p, u;
    int32_t k;
    bool greedy, use_p, use_k, use_m;
};
__device__ inline RowSettings row_settings(const SampleParams& p, int row) {
    RowSettings s;
    s.t = p.temperature ? p.temperature[row] : 1.f;
    s.k = p.top_k ? p.top_k[row] : 0;
    s.p = p.top_p ? p.top_p[row] : 1.f;
    s.min_p = p.min_p ? p.min_p[row] : 0.f;
    const float u = p.uniform[row];
    s.u = u > 0.f ? fminf(u, 1.f) : 0.f;
    s.greedy = !(s.t > 0.f);
    s.t = fminf(fmaxf(s.t, 1e-30f), 1e30f);  // beyond: the maxima alone, or a draw among all finite logits, as it is there
    s.use_k = s.k > 0 && s.k < p.n;
    s.use_p = s.p < 1.f;
    s.use_m = s.min_p > 0.f;
    s.min_p = fminf(s.min_p, 1.f);                                  // the likeliest token always stays
    s.greedy |= (s.use_k && s.k == 1) || (s.use_p && !(s.p > 0.f));  // an empty beginning: the first token alone
    return s;
}
__device__ inline float clean(float x) { return fmaxf(x + 0.f, -INFINITY); }  // NaN is never chosen; -0 and +0 are the same logit
// monotone bit pattern of a logit
__device__ inline uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ inline float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
constexpr uint32_t KEY_NEG_INF = 0x007fffffu;

// 2^(j / 256), j < 256: e^x by its series, x = j ln 2 / 256 < 0.7 (the 20th term is below 1e-21)
struct Exp2Table {
    double v[SP_TABLE];
};
constexpr Exp2Table make_exp2_table() {
    Exp2Table t{};
    for (int j = 0; j < SP_TABLE; j++) {
        const double x = j * 0.69314718055994530942 / SP_TABLE;
        double sum = 0.0;
        for (int k = 20; k > 0; k--) sum = (sum + 1.0) * x / k;  // from the smallest terms on
        t.v[j] = 1.0 + sum;
    }
    return t;
}
__device__ const Exp2Table g_exp2_table = make_exp2_table();

// The place where the running count or mass passes its goal.
struct Hit {
    uint32_t bin;               // 0xffffffff: nowhere
    uint32_t n_before, n_here;  // tokens before the bin and in it
    u64 w_before, w_here;       // their weights
    u64 all;                    // the whole count or mass
};

struct RowShared {
    uint32_t hist[4][SP_BINS];     // limbs of the masses; counts
    u64 list[SP_LIST];             // gathered tokens
    double exp2_table[SP_TABLE];   // 2^(j / SP_TABLE)
    // written by the other CTAs of the cluster.  This CTA writes none of them itself while they may: a CTA that is ahead may have
    // written what it gathered before this one has left the search (last, pick_w and list are its own once nobody else writes them)
    float x_max[SP_CLUSTER];
    u64 x_w[SP_CLUSTER];
    u64 last, pick_w;                // the last kept token, and the kept mass
    uint32_t run_n[SP_CLUSTER][32];  // sums of 32 runs of 32 bins of every CTA
    u64 run_w[SP_CLUSTER][32];
    uint32_t part[SP_CLUSTER];       // entries of every CTA in the list
    // of this CTA
    uint16_t part_n[1024];
    uint32_t bin_n[SP_CLUSTER][32];  // the bins of one run of every CTA
    u64 bin_w[SP_CLUSTER][32];
    u64 before_w[SP_CLUSTER];        // mass of every CTA before the hit
    u64 sums64[SP_MAX_WARPS + 1];
    u64 warp_w[SP_MAX_WARPS];
    float red_max[SP_MAX_WARPS];
    uint32_t n_list;                 // this CTA's entries of the list so far
    uint32_t key_lo, key_hi, found;
    Hit hit;
    double t_unit;                   // 256 log2 e / T
};

// Inclusive sums over the CTA in thread order.
__device__ inline u64 block_scan(u64 v, u64* warp_sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 up = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += up;
    }
    __syncthreads();  // the sums of the scan before are no longer read
    if (lane == 31) warp_sums[warp] = v;
    __syncthreads();
    u64 mine = lane < warp ? warp_sums[lane] : 0ull;
#pragma unroll
    for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    return mine + v;
}

// Smallest key in [lo, hi] for which the predicate holds (it holds from some key on, for hi at the latest); one warp.
template <typename F>
__device__ inline uint32_t first_key(uint32_t lo, uint32_t hi, F holds) {
    const int lane = threadIdx.x & 31;
    while (lo < hi) {
        const uint32_t step = (hi - lo) / 32 + 1;
        const uint32_t k = lo + step * lane;
        const bool ok = k >= lo && k <= hi ? holds(k) : true;
        const uint32_t votes = __ballot_sync(0xffffffffu, ok);
        if (!votes) {  // none of the 32 samples: it lies behind the last
            lo = lo + step * 31 + 1;
            continue;
        }
        const int f = __ffs(votes) - 1;
        const uint32_t at = lo + step * f;
        if (at <= hi && at >= lo) hi = at;
        if (f > 0) lo = lo + step * (f - 1) + 1;
    }
    return lo;
}

// atomicAdd to shared memory under a predicate: as an `if` each one costs a branch and its reconvergence
__device__ inline void add_if(uint32_t* p, uint32_t v, bool yes) {
    asm volatile("{\n.reg .pred q;\nsetp.ne.u32 q, %2, 0;\n@q red.shared.add.u32 [%0], %1;\n}\n" ::"r"(smem_u32(p)), "r"(v), "r"((uint32_t)yes) : "memory");
}
__device__ inline void cp_async16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(__cvta_generic_to_global(src)) : "memory");
}
__device__ inline void cp_async8(void* dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(dst)), "l"(__cvta_generic_to_global(src)) : "memory");
}
__device__ inline void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ inline void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
constexpr int RING = 4;  // quads of a thread on their way

// T threads, 1024 per SM.  ON_CHIP: the slice stays in shared memory; otherwise every pass reads it again, from L2 for the
// most part, and many rows are in flight at once.
template <int T, bool ON_CHIP>
__global__ void __launch_bounds__(T, 1024 / T) sample_kernel(SampleParams p) {
    constexpr int SP_WARPS = T / 32;
    extern __shared__ __align__(16) uint8_t row_smem[];
    RowShared& sh = *(RowShared*)row_smem;
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), row = blockIdx.y;
    // the slice on the chip, cleaned, and filled up with -inf to a multiple of 4
    float* x_s = p.scratch ? p.scratch + ((int64_t)row * C + rank) * p.slice : (float*)(row_smem + ((sizeof(RowShared) + 15) & ~(size_t)15));
    const int first = rank * p.slice, count = max(0, min(p.slice, p.n - first)), quads = (count + 3) / 4;
    const uint8_t* base = (const uint8_t*)p.logits + ((int64_t)row * p.stride + first) * dtype_size(p.dtype);
    auto other = [&](int r) -> RowShared* { return cluster.map_shared_rank(&sh, r); };
    auto widen = [&](uint32_t lo, uint32_t hi) -> float4 {  // four 16-bit logits
        if (p.dtype == B200KV_F16) {
            const float2 a = __half22float2(*(const __half2*)&lo), b = __half22float2(*(const __half2*)&hi);
            return make_float4(a.x, a.y, b.x, b.y);
        }
        return make_float4(__uint_as_float(lo << 16), __uint_as_float(lo & 0xffff0000u), __uint_as_float(hi << 16), __uint_as_float(hi & 0xffff0000u));
    };
    // logits 4 u .. 4 u + 3 of the slice as they are (a NaN stays one off the chip: it passes no comparison and has no weight)
    auto from_memory = [&](int u) -> float4 {
        if (p.vec && 4 * u + 4 <= count) {
            if (p.dtype == B200KV_F32) return __ldg((const float4*)base + u);
            const uint2 w = __ldg((const uint2*)base + u);
            return widen(w.x, w.y);
        }
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = 4 * u + e < count ? ld_as_f32(base, p.dtype, 4 * u + e) : -INFINITY;
        return make_float4(v[0], v[1], v[2], v[3]);
    };
    auto quad = [&](int u) -> float4 { return ON_CHIP ? ((const float4*)x_s)[u] : from_memory(u); };
    auto logit = [&](int i) -> float { return ON_CHIP ? x_s[i] : i < count ? ld_as_f32(base, p.dtype, i) : -INFINITY; };
    // f(quad, its number) for quads u, u + step, .. < end.  Off the chip a thread has RING quads on their way to slots of its own
    // in shared memory (registers for them would cost occupancy, unrolled code for them the instruction cache).
    uint4* ring = (uint4*)(row_smem + ((sizeof(RowShared) + 15) & ~(size_t)15)) + tid;
    auto sweep = [&](int u, int step, int end, auto f) {
        if (ON_CHIP || !p.vec) {
#pragma unroll 1
            for (; u < end; u += step) f(quad(u), u);
            return;
        }
        const bool f32 = p.dtype == B200KV_F32;
        const int full = min(end, count / 4), last = max(full - 1, 0);  // quads that are whole
        auto request = [&](int at, int slot) {  // past the end: the last one again
            if (f32) cp_async16(ring + slot * T, (const float4*)base + min(at, last));
            else cp_async8(ring + slot * T, (const uint2*)base + min(at, last));
            cp_async_commit();
        };
        if (full > 0) {
#pragma unroll
            for (int j = 0; j < RING; j++) request(u + j * step, j);
            int slot = 0;
#pragma unroll 1
            for (; u < full; u += step) {
                cp_async_wait<RING - 1>();
                const uint4 w = ring[slot * T];
                f(f32 ? make_float4(__uint_as_float(w.x), __uint_as_float(w.y), __uint_as_float(w.z), __uint_as_float(w.w)) : widen(w.x, w.y), u);
                request(u + RING * step, slot);  // the slot has been read: f used it
                slot = (slot + 1) % RING;
            }
            cp_async_wait<0>();
        }
        if (u == full && u < end) f(from_memory(u), u);  // the partial one
    };

    cluster.barrier_arrive();  // every CTA of the cluster runs before one writes into another's shared memory
    grid_launch_dependents();
    grid_dependency_wait();  // the kernel before has written the logits and the settings

    // ---- 1. the maximum, the slice onto the chip ----
    const RowSettings s = row_settings(p, row);
    // Bins of log2(1 / w), 28 octaves deep.  For top-p as deep as its cut can lie: what is deeper than log2(n / (1 - p)) has, all
    // of it together, less than 1 - p of the maximum's weight.  For top-k at least 30 below the maximum, where the likeliest few
    // hundred logits of a vocabulary lie: a cut below the bins takes the slow way (100 rows of 16000 logits, up to 200 of each:
    // 40 us when one row in the batch does, 14 when none does).
    const float octaves = s.use_k ? fminf(fmaxf(28.f, 30.f * 1.4426950408889634f / s.t), 96.f)
                        : s.use_p ? fminf(28.f, log2f((float)p.n / (1.f - s.p)) + 1.f) : 28.f;
    const float per_octave = (float)(SP_BINS - 1) / octaves;
    float zscale = 1.4426950408889634f / s.t * per_octave;
    if (tid == 0 && !s.greedy) sh.t_unit = (double)SP_TABLE * 1.4426950408889634074 / (double)s.t;  // one division for all
    float best = -INFINITY;
    for (int u0 = tid; u0 < quads; u0 += 8 * T) {  // every thread has eight quads on their way before it uses the first
        float4 v[8];
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (u0 + j * T < quads) v[j] = from_memory(u0 + j * T);
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (u0 + j * T < quads) {
                if (ON_CHIP) {
                    v[j] = make_float4(clean(v[j].x), clean(v[j].y), clean(v[j].z), clean(v[j].w));
                    ((float4*)x_s)[u0 + j * T] = v[j];
                }
                best = fmaxf(best, fmaxf(fmaxf(v[j].x, v[j].y), fmaxf(v[j].z, v[j].w)));
            }
    }
    const float own_max = best;  // of this thread's logits
#pragma unroll
    for (int o = 16; o; o >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (lane == 0) sh.red_max[warp] = best;
    if (!s.greedy) {
        if (s.use_k || s.use_p)
            for (int i = tid; i < SP_BINS; i += T) ((uint4*)&sh.hist[0][0])[i] = make_uint4(0u, 0u, 0u, 0u);
        for (int i = tid; i < SP_TABLE; i += T) sh.exp2_table[i] = g_exp2_table.v[i];
        if (tid == 0) sh.n_list = 0;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SP_WARPS; w++) best = fmaxf(best, sh.red_max[w]);
    cluster.barrier_wait();
    if (tid < C) other(tid)->x_max[rank] = best;
    cluster.sync();
    float x_top = -INFINITY;
    int top_rank = 0;
    for (int r = C - 1; r >= 0; r--)
        if (sh.x_max[r] >= x_top) x_top = sh.x_max[r], top_rank = r;
    if (s.greedy || x_top == -INFINITY) {  // the first maximum; nothing of another CTA is touched any more
        if (rank != top_rank) return;
        int at = x_top == -INFINITY ? 0 : 0x7fffffff;
        if (at)
            sweep(tid, T, quads, [&](const float4& v, int u) {
                const int i = v.x == x_top ? 0 : v.y == x_top ? 1 : v.z == x_top ? 2 : v.w == x_top ? 3 : 4;
                if (i < 4) at = min(at, 4 * u + i);
            });
        at = __reduce_min_sync(0xffffffffu, at);
        __syncthreads();
        if (lane == 0) sh.red_max[warp] = __int_as_float(at);
        __syncthreads();
        if (tid == 0) {
            for (int w = 1; w < SP_WARPS; w++) at = min(at, __float_as_int(sh.red_max[w]));
            p.out[row] = x_top == -INFINITY ? 0 : first + at;
        }
        return;
    }
    if (x_top == INFINITY) {  // infinite logits share the row: all of the same weight, taken by rising index
        uint32_t mine = 0;
        sweep(tid, T, quads, [&](const float4& v, int) { mine += (v.x == INFINITY) + (v.y == INFINITY) + (v.z == INFINITY) + (v.w == INFINITY); });
        mine = (uint32_t)block_scan(mine, sh.sums64);
        if (tid == T - 1)
            for (int r = 0; r < C; r++) other(r)->x_w[rank] = mine;
        cluster.sync();
        u64 n = 0, before = 0;
        for (int r = 0; r < C; r++) {
            if (r == rank) before = n;
            n += sh.x_w[r];
        }
        if (s.use_k) n = min(n, (u64)s.k);
        if (s.use_p) n = max((u64)ceil((double)s.p * (double)n), 1ull);
        const u64 place = min((u64)((double)s.u * (double)n), n - 1);
        if (place < before || place >= before + sh.x_w[rank] || tid) return;
        for (int i = 0;; i++)
            if (logit(i) == INFINITY && before++ == place) {
                p.out[row] = first + i;
                return;
            }
    }
    double t_unit = sh.t_unit;
    float t_used = s.t;
    if (s.t < fabsf(x_top) * 0x1p-34f) {
        // Other logits lie at least 2^-24 |max| below the maximum: they have no weight at this temperature, nor at the one that is
        // taken in its place, at which products with 1 / T keep their accuracy.
        t_used = fabsf(x_top) * 0x1p-34f;
        t_unit = (double)SP_TABLE * 1.4426950408889634074 / (double)t_used, zscale = 1.4426950408889634f / t_used * per_octave;
    }

    // ---- weights ----
    // the last bin takes everything that is deeper; monotone in x
    // (by its own rounded product wherever it is asked for: one that a sum took in unrounded would put a few logits next to a border
    // into the other bin)
    auto depth = [&](float x) -> float { return __fmul_rn(x_top - x, zscale); };
    auto rounded = [](float z) -> float { return __fadd_rn(z, 8388608.f); };  // to the nearest whole number, in the low bits
    auto z_bin = [&](float x) -> uint32_t { return __float_as_uint(rounded(fminf(depth(x), (float)(SP_BINS - 1)))) & (SP_BINS - 1); };
    // exp((x - max) / T) = 2^(t / 256), t = (x - max) 256 log2 e / T = n + r, n whole: 2^(n / 256) from the table and the exponent,
    // 2^(r / 256) by its Taylor polynomial of degree 3 in r ln 2 / 256 (|r| <= 1/2: what is left out is below 1.5e-13), rounded
    // to 44 fractional bits by adding 1.5 * 2^8.  What lies below 2^-46.5 (it would round to 0), -inf, a NaN and
    // the fill of a slice have no weight, by comparison: what they give in the sums is not used.
    const double t_top = -(double)x_top * t_unit;
    const float x_floor = __double2float_ru((double)x_top - 46.5 * 0.69314718055994530942 * (double)t_used);  // always finite
    constexpr double L = 0.69314718055994530942 / SP_TABLE;
    double taylor1 = L, taylor2 = L * L / 2.0, taylor3 = L * L * L / 6.0;
    asm volatile("" : "+d"(taylor1), "+d"(taylor2), "+d"(taylor3));  // in registers: two moves per use otherwise
    auto weight = [&](float x) -> u64 {
        constexpr double MAGIC = 6755399441055744.0;  // 1.5 * 2^52
        const double t = fma((double)x, t_unit, t_top);
        const double biased = t + MAGIC, r = t - (biased - MAGIC);
        const int n = __double2loint(biased);
        double q = fma(r, taylor3, taylor2);
        q = fma(q, r, taylor1);
        q = fma(q, r, 1.0);
        const double tab = sh.exp2_table[n & (SP_TABLE - 1)];
        const double scaled = __hiloint2double(__double2hiint(tab) + ((n << 12) & 0xfff00000), __double2loint(tab));
        const u64 w = (u64)(__double_as_longlong(fma(q, scaled, 384.0)) - __double_as_longlong(384.0));
        return x >= x_floor ? w : 0ull;
    };
    // f(x, place in the slice) for every logit of the slice; the fill is -inf
    auto each = [&](auto f) {
        sweep(tid, T, quads, [&](const float4& v, int u) { f(v.x, 4 * u), f(v.y, 4 * u + 1), f(v.z, 4 * u + 2), f(v.w, 4 * u + 3); });
    };
    // min-p: the smallest logit that passes
    const uint32_t key_max = key_of(clean(x_top));
    float x_m = -INFINITY;
    if (s.use_m) {
        if (warp == 0) {
            const uint32_t k = first_key(KEY_NEG_INF + 1, key_max, [&](uint32_t key) {
                return key == key_max || exp(((double)of_key(key) - (double)x_top) / (double)s.t) >= (double)s.min_p;
            });
            if (lane == 0) sh.found = k;
        }
        __syncthreads();
        x_m = of_key(sh.found);
    }

    // ---- a histogram over the cluster, and the bin in which the running count or mass first exceeds its goal ----
    // feed(f) calls f(quad, its number) for what is looked at.  bin_of(x, index): 0 .. SP_BINS - 1, or -1 for what does not take part.  goal(all): from the whole count or mass.
    // *_base: what lies before the first bin.  The caller sees to it that the histogram is clear and that the CTAs have left it.
    // counts / weights: what is added up (std::true_type or false_type); by_weight: the goal is a mass.
    auto limbs = [](const RowShared* o, int b) -> u64 { return (u64)o->hist[0][b] + ((u64)o->hist[1][b] << SP_LIMB) + ((u64)o->hist[2][b] << (2 * SP_LIMB)); };
    auto round_of = [&](auto counts_, auto weights_, auto feed, uint32_t n_base, u64 w_base, auto bin_of, auto goal, bool by_weight) -> Hit {
        // The last bin, which takes all that is deep, is added up in registers: atomics on one address follow one another.
        constexpr bool counts = decltype(counts_)::value, weights = decltype(weights_)::value;
        uint32_t deep_n = 0;
        u64 deep_w = 0;
        feed([&](const float4& v, int u) {
            const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int b = bin_of(x[e], first + 4 * u + e);
                const bool deep = b == SP_BINS - 1, binned = (b >= 0) & !deep;
                uint32_t* at = &sh.hist[0][b];
                if (counts) {
                    deep_n += deep & (x[e] > -INFINITY);
                    add_if(at + 3 * SP_BINS, 1u, binned);
                }
                if (weights) {
                    const u64 w = weight(x[e]);
                    deep_w += deep ? w : 0ull;
                    const uint32_t l0 = (uint32_t)w & 0x7fffu, l1 = (uint32_t)(w >> SP_LIMB) & 0x7fffu, l2 = (uint32_t)(w >> (2 * SP_LIMB));
                    add_if(at, l0, binned);
                    add_if(at + SP_BINS, l1, binned & (w >> SP_LIMB != 0));
                    add_if(at + 2 * SP_BINS, l2, binned & (l2 != 0));
                }
            }
        });
        if (counts) {
            deep_n = __reduce_add_sync(0xffffffffu, deep_n);
            if (lane == 0 && deep_n) atomicAdd(&sh.hist[3][SP_BINS - 1], deep_n);
        }
        if (weights) {
#pragma unroll
            for (int o = 16; o; o >>= 1) deep_w += __shfl_xor_sync(0xffffffffu, deep_w, o);
            if (lane == 0 && deep_w) {
                atomicAdd(&sh.hist[0][SP_BINS - 1], (uint32_t)deep_w & 0x7fffu);
                atomicAdd(&sh.hist[1][SP_BINS - 1], (uint32_t)(deep_w >> SP_LIMB) & 0x7fffu);
                atomicAdd(&sh.hist[2][SP_BINS - 1], (uint32_t)(deep_w >> (2 * SP_LIMB)));
            }
        }
        __syncthreads();
        {  // the sums of every run of 32 bins go to every CTA
            constexpr int PER = SP_BINS / T, LANES = 32 / PER;  // bins per thread, threads per run
            uint32_t n = 0;
            u64 w = 0;
#pragma unroll
            for (int j = 0; j < PER; j++) {
                if (counts) n += sh.hist[3][PER * tid + j];
                if (weights) w += limbs(&sh, PER * tid + j);
            }
#pragma unroll
            for (int o = LANES / 2; o; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o), w += __shfl_xor_sync(0xffffffffu, w, o);
            const int to = tid % LANES;
            if (to < C) other(to)->run_n[rank][tid / LANES] = n, other(to)->run_w[rank][tid / LANES] = w;
        }
        cluster.sync();
        // lane = run: the run in which the goal is passed, then lane = bin of that run.  Inclusive sums over the lanes.
        auto scan = [&](uint32_t& n, u64& w) {
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t un = __shfl_up_sync(0xffffffffu, n, o);
                const u64 uw = __shfl_up_sync(0xffffffffu, w, o);
                if (lane >= o) n += un, w += uw;
            }
        };
        // (a warp per CTA of the cluster: the search itself is the same in all of them)
        uint32_t n = 0, n_incl = 0, n_run = 0, runs = 0;
        u64 w = 0, w_incl = 0, w_run = 0, all = 0, target = 0;
        int run = 0;
        if (warp < C) {
            for (int r = 0; r < C; r++) n += sh.run_n[r][lane], w += sh.run_w[r][lane];
            n_incl = n, w_incl = w;
            scan(n_incl, w_incl);
            all = __shfl_sync(0xffffffffu, by_weight ? w_incl : (u64)n_incl, 31);
            target = goal(all);
            runs = __ballot_sync(0xffffffffu, (by_weight ? w_base + w_incl : (u64)(n_base + n_incl)) > target);
            if (runs) {
                run = __ffs(runs) - 1;
                const RowShared* o = other(warp);
                sh.bin_n[warp][lane] = counts ? o->hist[3][run * 32 + lane] : 0u;
                sh.bin_w[warp][lane] = weights ? limbs(o, run * 32 + lane) : 0ull;
                n_run = n_base + __shfl_sync(0xffffffffu, n_incl - n, run);
                w_run = w_base + __shfl_sync(0xffffffffu, w_incl - w, run);
            }
        }
        __syncthreads();
        if (warp < C) {
            if (runs) {
                n = 0, w = 0;
                for (int r = 0; r < C; r++) n += sh.bin_n[r][lane], w += sh.bin_w[r][lane];
                n_incl = n, w_incl = w;
                scan(n_incl, w_incl);
                const uint32_t bins = __ballot_sync(0xffffffffu, (by_weight ? w_run + w_incl : (u64)(n_run + n_incl)) > target);
                const int bin = __ffs(bins) - 1;
                if (warp == 0 && lane == bin) sh.hit = Hit{(uint32_t)(run * 32 + bin), n_run + n_incl - n, n, w_run + w_incl - w, w, all};
                if (weights) {  // what every CTA has before the bin
                    u64 v = (lane < run ? sh.run_w[warp][lane] : 0ull) + (lane < bin ? sh.bin_w[warp][lane] : 0ull);
#pragma unroll
                    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
                    if (lane == 0) sh.before_w[warp] = v;
                }
            } else if (warp == 0 && lane == 0) {
                sh.hit = Hit{0xffffffffu, 0, 0, 0, 0, all};  // in every CTA alike
            }
        }
        __syncthreads();
        return sh.hit;
    };
    const std::true_type yes;
    const std::false_type no;
    auto whole_slice = [&](auto f) { sweep(tid, T, quads, f); };
    // clears the histogram for another round, once every CTA has read what it needs of the last one
    auto next_round = [&]() {
        cluster.sync();
        for (int i = tid; i < SP_BINS; i += T) ((uint4*)&sh.hist[0][0])[i] = make_uint4(0u, 0u, 0u, 0u);
        __syncthreads();
    };

    // ---- 4. the draw over whole slices ----
    // kept: everything above x_cut, and of those that equal it the ones up to index last_same
    float x_cut = -INFINITY;
    uint32_t last_same = 0xffffffffu;
    u64 of_slice = 0;
    bool runs_known = false;
    auto kept = [&](float x, int i) -> bool { return (x > x_cut) | ((x == x_cut) & ((uint32_t)(first + i) <= last_same)); };
    auto kept_weight = [&](float x, int i) -> u64 { return kept(x, i) ? weight(x) : 0ull; };
    const int run = ((quads + SP_WARPS - 1) / SP_WARPS + 31) / 32 * 32;  // quads of a warp
    // the kept mass of the slice; of a run per warp in warp_w
    auto run_masses = [&]() -> u64 {
        u64 mine = 0;
        const int end = min(quads, (warp + 1) * run);
        if (x_cut == -INFINITY)
            sweep(warp * run + lane, 32, end, [&](const float4& v, int) { mine += weight(v.x) + weight(v.y) + weight(v.z) + weight(v.w); });
        else
        sweep(warp * run + lane, 32, end, [&](const float4& v, int u) {
            // (the votes of the lanes that are still in the loop) nothing kept in any of them: on
            if (!__any_sync(__activemask(), fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) >= x_cut)) return;
            // all four without branches: they run side by side
            const u64 w[4] = {weight(v.x), weight(v.y), weight(v.z), weight(v.w)};
            mine += (kept(v.x, 4 * u) ? w[0] : 0ull) + (kept(v.y, 4 * u + 1) ? w[1] : 0ull) + (kept(v.z, 4 * u + 2) ? w[2] : 0ull) + (kept(v.w, 4 * u + 3) ? w[3] : 0ull);
        });
#pragma unroll
        for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
        __syncthreads();
        if (lane == 0) sh.warp_w[warp] = mine;
        __syncthreads();
        u64 sum = 0;
#pragma unroll
        for (int w = 0; w < SP_WARPS; w++) sum += sh.warp_w[w];
        runs_known = true;
        return sum;
    };
    // mass: kept mass of the row; before, here: of the slices before this one, and of this one
    auto draw = [&](u64 mass, u64 before, u64 here) {
        const u64 target = min((u64)((double)s.u * (double)mass), mass - 1);
        if (target < before || target >= before + here) return;
        if (!runs_known) run_masses();
        int w = 0;
        for (; w < SP_WARPS - 1 && target >= before + sh.warp_w[w]; w++) before += sh.warp_w[w];
        const int lo = 4 * w * run, hi = 4 * min(quads, (w + 1) * run), per = (hi - lo + T - 1) / T;
        u64 mine = 0;
        for (int i = lo + tid * per; i < min(hi, lo + (tid + 1) * per); i++) mine += kept_weight(logit(i), i);
        before += block_scan(mine, sh.sums64) - mine;
        if (before <= target && target < before + mine)
            for (int i = lo + tid * per;; i++) {
                before += kept_weight(logit(i), i);
                if (target < before) {
                    p.out[row] = first + i;
                    break;
                }
            }
    };

    // ---- 2. the cut ----
    if (s.use_k || s.use_p) {
        u64 whole = 0;  // count of the row's numbers (top-k), or its mass
        auto p_goal = [&](u64 mass) -> u64 {  // the mass before a kept token is below p x mass: the cut is where the sum reaches it
            const u64 least = (u64)ceil((double)s.p * (double)mass);
            return least ? least - 1 : 0;
        };
        auto by_depth = [&](float x, int) -> int { return (int)z_bin(x); };
        auto of_k = [&](u64) -> u64 { return (u64)(s.k - 1); };
        // Top-k looks at the maxima of the threads first: the k-th largest of them bounds the k-th largest logit from below, and
        // little more than k logits lie above it.
        Hit top = s.use_k ? round_of(yes, no, [&](auto f) { f(make_float4(own_max, -INFINITY, -INFINITY, -INFINITY), 0); }, 0, 0, by_depth, of_k, false)
                          : round_of(no, yes, whole_slice, 0, 0, by_depth, p_goal, true);
        whole = top.all;
        // bitonic sort of list[0 .. n): every step, a thread per pair; steps of up to 32 stay inside the 64 entries of a warp
        auto sort = [&](int n) {
            int size = 64;
            while (size < n) size <<= 1;
            __syncthreads();
            for (int i = n + tid; i < size; i += T) sh.list[i] = ~0ull;
            __syncthreads();
            for (int k = 2; k <= size; k <<= 1)
                for (int j = k >> 1; j; j >>= 1) {
                    for (int pair = tid; pair < size / 2; pair += T) {
                        const int a = 2 * pair - (pair & (j - 1)), b = a + j;
                        const u64 va = sh.list[a], vb = sh.list[b];
                        if ((va > vb) == ((a & k) == 0)) sh.list[a] = vb, sh.list[b] = va;
                    }
                    if (j > 32 || (j == 1 && k >= 64)) __syncthreads();
                    else __syncwarp();
                }
        };
        auto token_of = [&](float x, int i) -> u64 { return ((u64)~key_of(clean(x)) << 32) | (u64)(uint32_t)(first + i); };  // sorts by falling logits, then by index
        auto logit_of = [](u64 token) -> float { return of_key(~(uint32_t)(token >> 32)); };
        constexpr int PLACES = SP_LIST / T;  // of a sorted list, a thread has places e0 .. e0 + PLACES - 1
        const int e0 = PLACES * tid;
        // For every entry of list[0 .. n), n <= SP_COUNT, what lies before it in the order of the entries: their number and the
        // sum of weights[].  Thread i < n gets entry i.  All threads count: every warp walks a share of the list, each lane for
        // an entry of its own.
        u64* weights = (u64*)&sh.hist[0][0];          // the histogram is not used any more by then
        u64* part_w = weights + SP_LIST;              // [T]
        static_assert((SP_LIST + 1024) * 8 <= sizeof(sh.hist), "weights, and a sum for each thread");
        auto count_before = [&](int n, uint32_t* n_before, u64* w_before) {
            int wide = 32;
            while (wide < n) wide <<= 1;
            const int shares = T / wide, i = tid & (wide - 1), share = tid / wide;
            const u64 mine = i < n ? sh.list[i] : 0ull;
            uint32_t cn = 0;
            u64 cw = 0;
            for (int j = share * n / shares; j < (share + 1) * n / shares; j++)
                if (sh.list[j] < mine) cn++, cw += weights[j];
            __syncthreads();
            part_w[tid] = cw, sh.part_n[tid] = (uint16_t)cn;
            __syncthreads();
            cn = 0, cw = 0;
            if (tid < n)
                for (int j = 0; j < shares; j++) cn += sh.part_n[j * wide + tid], cw += part_w[j * wide + tid];
            *n_before = cn, *w_before = cw;
        };
        // ---- 3. few enough tokens: put them in order ----
        // Each CTA has a part of the list, `cap` entries; false: more than that in some CTA (the same answer in every CTA).
        const int cap_bits = 10 - (31 - __clz(C)), cap = 1 << cap_bits;
        static_assert(SP_LIST == 1 << 10, "the parts of the list");
        auto gather = [&](bool to_all, auto takes) -> bool {
            each([&](float x, int i) {
                if (!takes(x)) return;
                const uint32_t slot = atomicAdd(&sh.n_list, 1u);
                if (slot >= (uint32_t)cap) return;
                const u64 token = token_of(x, i);
                if (!to_all) other(0)->list[rank * cap + slot] = token;
                else
                    for (int r = 0; r < C; r++) other(r)->list[rank * cap + slot] = token;
            });
            __syncthreads();
            if (tid < C) other(tid)->part[rank] = sh.n_list;
            cluster.sync();
            uint32_t most = 0;
            for (int r = 0; r < C; r++) most = max(most, sh.part[r]);
            return most <= (uint32_t)cap;
        };
        if (s.use_k && top.bin < SP_BINS - 1 && gather(false, [&](float x) { return z_bin(x) <= top.bin; })) {
            if (rank != 0) return;
            // close the gaps between the parts
            int n = 0, to[PLACES];
            u64 tok[PLACES], w[PLACES];
#pragma unroll
            for (int j = 0; j < PLACES; j++) tok[j] = sh.list[e0 + j], to[j] = -1;
            for (int r = 0; r < C; r++) {
#pragma unroll
                for (int j = 0; j < PLACES; j++) {
                    const int d = e0 + j - r * cap;
                    if (d >= 0 && d < (int)sh.part[r]) to[j] = n + d;
                }
                n += (int)sh.part[r];
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < PLACES; j++)
                if (to[j] >= 0) sh.list[to[j]] = tok[j];
            __syncthreads();
            if (n <= SP_COUNT) {
                const u64 tok = tid < n ? sh.list[tid] : ~0ull, w = tid < n ? weight(logit_of(tok)) : 0ull;
                if (tid < n) weights[tid] = w;
                __syncthreads();
                uint32_t at;
                u64 before;
                count_before(n, &at, &before);
                if (tid < n && (int)at == min(n, s.k) - 1) sh.pick_w = before + w;  // the mass of the first k
                __syncthreads();
                const u64 goal = s.use_p ? p_goal(sh.pick_w) : ~0ull;
                const bool keeps = tid < n && (int)at < s.k && before <= goal && (logit_of(tok) >= x_m || at == 0);
                const int n_kept = __syncthreads_count(keeps);
                if (keeps && (int)at == n_kept - 1) sh.pick_w = before + w;  // the kept mass
                if (tid < n) sh.list[tid] = (tok << 32) | (u64)tid, weights[tid] = keeps ? w : 0ull;  // by rising index now
                __syncthreads();
                const u64 mass = sh.pick_w, target = min((u64)((double)s.u * (double)mass), mass - 1);
                count_before(n, &at, &before);
                if (keeps && before <= target && before + w > target) p.out[row] = (int32_t)(uint32_t)tok;
                return;
            }
            sort(n);
            u64 sum = 0;
            bool passes[PLACES];
#pragma unroll
            for (int j = 0; j < PLACES; j++) {
                passes[j] = e0 + j < n && e0 + j < s.k;
                tok[j] = passes[j] ? sh.list[e0 + j] : ~0ull;
                w[j] = passes[j] ? weight(logit_of(tok[j])) : 0ull;
                sum += w[j];
            }
            u64 incl = block_scan(sum, sh.sums64);
            if (tid == T - 1) sh.pick_w = incl;
            __syncthreads();
            const u64 goal = s.use_p ? p_goal(sh.pick_w) : ~0ull;
            u64 before = incl - sum;
            int n_kept = 0;
#pragma unroll
            for (int j = 0; j < PLACES; j++) {
                passes[j] = passes[j] && before <= goal && (logit_of(tok[j]) >= x_m || e0 + j == 0);
                before += w[j];
                n_kept += __syncthreads_count(passes[j]);
            }
            // the kept ones by rising index, each with its place in the order of weights, where its weight stays
#pragma unroll
            for (int j = 0; j < PLACES; j++)
                if (passes[j]) weights[e0 + j] = w[j], sh.list[e0 + j] = (tok[j] << 32) | (u64)(uint32_t)(e0 + j);
            sort(n_kept);
            sum = 0;
#pragma unroll
            for (int j = 0; j < PLACES; j++) {
                tok[j] = e0 + j < n_kept ? sh.list[e0 + j] : ~0ull;
                w[j] = e0 + j < n_kept ? weights[(uint32_t)tok[j]] : 0ull;
                sum += w[j];
            }
            incl = block_scan(sum, sh.sums64);
            if (tid == T - 1) sh.pick_w = incl;
            __syncthreads();
            const u64 mass = sh.pick_w, target = min((u64)((double)s.u * (double)mass), mass - 1);
            before = incl - sum;
#pragma unroll
            for (int j = 0; j < PLACES; j++) {
                if (before <= target && before + w[j] > target) p.out[row] = (int32_t)(tok[j] >> 32);
                before += w[j];
            }
            return;
        }
        if (!s.use_k && !s.use_m && top.bin < SP_BINS - 1) {
            // top-p alone: the tokens of the bin, in every CTA
            const float in_bin = 8388608.f + (float)top.bin;  // z_bin(x) == top.bin, which is not the last bin
            if (gather(true, [&](float x) { return rounded(depth(x)) == in_bin; })) {
                for (int i = tid; i < C * cap; i += T)
                    if ((i & (cap - 1)) < (int)sh.part[i >> cap_bits]) weights[i] = weight(logit_of(sh.list[i]));
                __syncthreads();
                // the mass before each of this CTA's own tokens, in the order of the whole bin; a few threads per token
                constexpr int LANES = T >= 1024 ? 8 : 4;
                const u64 goal = p_goal(whole);
                const int n_own = (int)sh.part[rank];
                u64 kept_here = 0;
                for (int m0 = 0; m0 < n_own; m0 += T / LANES) {
                    const int m = m0 + tid / LANES;
                    const u64 token = m < n_own ? sh.list[rank * cap + m] : 0ull;
                    u64 sum = 0;
                    for (int r = 0; r < C; r++) {
                        const int end = r * cap + (int)sh.part[r];
#pragma unroll 4
                        for (int j = r * cap + tid % LANES; j < end; j += LANES) sum += sh.list[j] < token ? weights[j] : 0ull;
                    }
#pragma unroll
                    for (int o = LANES / 2; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                    sum += top.w_before;
                    const u64 w = m < n_own ? weights[rank * cap + m] : 0ull;
                    if (!w || sum > goal || tid % LANES) continue;
                    kept_here += w;
                    if (sum + w > goal)  // the last kept token: everybody learns of it
                        for (int r = 0; r < C; r++) other(r)->last = token, other(r)->pick_w = sum + w;
                }
#pragma unroll
                for (int o = 16; o; o >>= 1) kept_here += __shfl_xor_sync(0xffffffffu, kept_here, o);
                __syncthreads();
                if (lane == 0) sh.warp_w[warp] = kept_here;
                __syncthreads();
                if (tid < C) {
                    kept_here = sh.before_w[rank];
                    for (int w = 0; w < SP_WARPS; w++) kept_here += sh.warp_w[w];
                    other(tid)->x_w[rank] = kept_here;
                }
                cluster.sync();
                x_cut = logit_of(sh.last), last_same = (uint32_t)sh.last;
                u64 below = 0;
                for (int r = 0; r < rank; r++) below += sh.x_w[r];
                draw(sh.pick_w, below, sh.x_w[rank]);
                return;
            }
        }
        // Many tokens: down to the last kept one, by the same histogram over bit patterns (falling logits) or indices, 1024
        // positions at a time.  Four questions, one after the other, through one piece of code:
        //   K     the k-th logit, among the bit patterns of its bin
        //   MASS  top-p of the first k: their mass, and the bin of log2 w in which p of it is reached
        //   P     the logit at which it is reached, among the bit patterns of that bin
        //   SAME  of the logits equal to the last kept one, the index of the last that is kept
        if (s.use_k) {
            next_round();
            top = round_of(yes, no, whole_slice, 0, 0, by_depth, of_k, false);
        }
        enum { K, MASS, P, SAME };
        uint32_t n_cut = 0xffffffffu, n_same = 0xffffffffu;
        Hit hit = top;
#pragma unroll 1
        for (int step = K; step <= SAME; step++) {
            uint32_t lo = 0, hi = SP_BINS - 1, n_base = 0;
            u64 w_base = 0, goal = 0;
            u64 over = 0;  // mass of logits equal to the k-th that are not among the first k
            if (step == K) {
                if (!s.use_k || hit.bin == 0xffffffffu) continue;
                goal = (u64)(s.k - 1);
            } else if (step == MASS) {
                if (!s.use_k || !s.use_p) continue;
                if (n_same != 0xffffffffu) over = (u64)(n_same - n_cut) * weight(x_cut);
            } else if (step == P) {
                if (!s.use_p) continue;
                goal = p_goal(whole);
            } else {
                if (x_m > x_cut) x_cut = x_m, n_cut = n_same = 0xffffffffu;
                if (n_cut >= n_same) continue;
                hi = (uint32_t)p.n - 1, goal = (u64)(n_cut - 1);
            }
            if (step == K || step == P) {  // the bit patterns of the bin
                const uint32_t bin = hit.bin;
                __syncthreads();
                if (warp < 2) {
                    const uint32_t border = bin + 1 - (uint32_t)warp;  // the first pattern less deep than that
                    const uint32_t k = border == 0 ? key_max + 1 : first_key(KEY_NEG_INF + 1, key_max, [&](uint32_t k) { return z_bin(of_key(k)) < border; });
                    if (lane == 0) (warp ? sh.key_hi : sh.key_lo) = k;
                }
                __syncthreads();
                lo = key_max - (sh.key_hi - 1), hi = key_max - max(sh.key_lo, key_of(x_cut));
                n_base = hit.n_before, w_base = step == P ? hit.w_before : 0ull;
            }
            Hit f;
#pragma unroll 1
            for (;;) {
                const int bits = 32 - __clz((hi - lo) | 1u), shift = bits > 10 ? bits - 10 : 0;
                next_round();
                f = round_of(yes, yes, whole_slice, n_base, w_base, [&](float x, int i) -> int {
                    const uint32_t at = step == MASS ? z_bin(x) : step == SAME ? (uint32_t)i : key_max - key_of(clean(x));
                    const bool part = step == SAME ? x == x_cut : x > -INFINITY && x >= x_cut;
                    return part && at >= lo && at <= hi ? (int)((at - lo) >> shift) : -1;
                }, [&](u64 all) -> u64 { return step == MASS ? p_goal(all - over) : goal; }, step == MASS || step == P);
                f.bin = lo + (f.bin << shift);
                if (shift == 0) break;
                lo = f.bin, hi = min(hi, lo + ((1u << shift) - 1u));
                n_base = f.n_before, w_base = f.w_before;
            }
            if (step == K) {
                x_cut = of_key(key_max - f.bin), n_cut = (uint32_t)s.k - f.n_before, n_same = f.n_here;
            } else if (step == MASS) {
                hit = f, whole = f.all - over;
            } else if (step == P) {
                const u64 w = f.w_here / f.n_here;  // all of them have the same weight, which is not 0
                const uint32_t n = (uint32_t)min((goal + 1 - f.w_before + w - 1) / w, (u64)f.n_here);
                const float x = of_key(key_max - f.bin);
                if (x > x_cut || n < n_cut) x_cut = x, n_cut = n, n_same = f.n_here;
            } else {
                last_same = f.bin;
            }
        }
    } else {
        x_cut = x_m;
    }
    of_slice = run_masses();
    if (tid < C) other(tid)->x_w[rank] = of_slice;
    cluster.sync();
    u64 mass = 0, before = 0;
    for (int r = 0; r < C; r++) {
        if (r == rank) before = mass;
        mass += sh.x_w[r];
    }
    draw(mass, before, of_slice);
}

// How a launch is cut: up to eight CTAs per row (of at least 1024 logits each).
//   every CTA has an SM of its own           1024 threads, the slices on the chip
//   up to three to an SM                     512 threads, the slices on the chip; two are resident
//   more                                     256 threads, four per SM, that read their slice again from L2 where they need it: twice
//                                            as many rows are in flight, and the exchanges of one hide behind the work of the others
// Measured on rows of 128256 f32 logits, top-p 0.9 (us for 1024 / 512 / 256 threads): 8 rows 24.8 / 26.7 / 35.3; 15 rows 25.5 /
// 31.0; 16 rows 36.6 / 30.8; 37 rows 59.6 / 48.0 / 57.8; 48 rows - / 56.1 / 59.9; 64 rows 94 / 65 / 63; 256 rows 321 / 223 / 193.
struct SampleCut {
    int c, slice, threads;  // CTAs per row, logits per CTA (the next slice starts on a 16-byte boundary when the row does)
};
// CTAs that get an SM of their own: the SMs of a processing cluster that are left over hold no whole cluster.
static int sample_alone(int c) { return c == 8 ? 120 : c == 4 ? 128 : 148; }
static SampleCut sample_cut(int64_t rows, int32_t n) {
    SampleCut k{1, 0, 1024};
    while (k.c < SP_CLUSTER && n >= 2 * k.c * 1024 && (n > k.c * SP_SLICE || rows * k.c * 2 <= sample_alone(k.c * 2))) k.c *= 2;
    if (n > MAX_ON_CHIP) k.c = SP_CLUSTER;
    k.slice = ((n + k.c - 1) / k.c + 7) / 8 * 8;
    const bool two_fit = k.slice <= SP_SLICE;
    if (n <= MAX_ON_CHIP && rows * k.c > sample_alone(k.c)) k.threads = two_fit && rows * k.c <= 3 * 148 ? 512 : 256;
    return k;
}

}  // namespace b200kv

using namespace b200kv;

extern "C" int64_t b200kv_sample_scratch_bytes(int64_t rows, int32_t n) {
    if (rows <= 0 || n <= 0 || n > MAX_VOCAB) {
        fail("rows and n must be positive, n at most %d", MAX_VOCAB);
        return -1;
    }
    return n <= MAX_ON_CHIP ? 0 : rows * SP_CLUSTER * (int64_t)sample_cut(rows, n).slice * (int64_t)sizeof(float);
}

extern "C" int b200kv_sample(const void* logits, int64_t stride, int32_t dtype, int64_t rows, int32_t n, const float* temperature,
                             const int32_t* top_k, const float* top_p, const float* min_p, const float* uniform, int32_t* out, void* scratch,
                             void* stream_) {
    if (!logits || !uniform || !out) return fail("null tensor");
    if (rows <= 0 || n <= 0) return fail("rows and n must be positive");
    if (rows > 65535) return fail("%lld rows in one call: at most 65535", (long long)rows);
    if (n > MAX_VOCAB) return fail("a vocabulary of %d tokens: at most %d", n, MAX_VOCAB);
    if (dtype < B200KV_F32 || dtype > B200KV_BF16) return fail("unknown dtype %d", dtype);
    if (stride < n && rows > 1) return fail("rows of %d logits cannot be %lld elements apart", n, (long long)stride);
    if (n > MAX_ON_CHIP && !scratch) return fail("rows of %d logits need a workspace: b200kv_sample_scratch_bytes", n);
    if ((uintptr_t)scratch % 16) return fail("scratch must be 16-byte aligned");
    SampleParams p{};
    p.logits = logits, p.stride = stride, p.dtype = dtype, p.n = n;
    p.temperature = temperature, p.top_k = top_k, p.top_p = top_p, p.min_p = min_p, p.uniform = uniform, p.out = out;
    p.vec = (uintptr_t)logits % 16 == 0 && (rows == 1 || (stride * dtype_size(dtype)) % 16 == 0);
    const SampleCut cut = sample_cut(rows, n);
    p.slice = cut.slice;
    p.scratch = n > MAX_ON_CHIP ? (float*)scratch : nullptr;
    const size_t smem = ((sizeof(RowShared) + 15) & ~(size_t)15) + (p.scratch ? 0 : cut.threads > 256 ? (size_t)p.slice * sizeof(float) : (size_t)RING * 256 * 16);
    constexpr size_t most = ((sizeof(RowShared) + 15) & ~(size_t)15) + 4 * std::max(MAX_ON_CHIP / SP_CLUSTER, 4 * 256 * RING);
    auto kernel = cut.threads == 1024 ? sample_kernel<1024, true> : cut.threads == 512 ? sample_kernel<512, true> : sample_kernel<256, false>;
    B200KV_CUDA((cut.threads == 1024 ? allow_shared_memory<sample_kernel<1024, true>>(most)
                                     : cut.threads == 512 ? allow_shared_memory<sample_kernel<512, true>>(most) : allow_shared_memory<sample_kernel<256, false>>(most)));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)cut.c, (unsigned)rows), cfg.blockDim = dim3((unsigned)cut.threads), cfg.dynamicSmemBytes = smem, cfg.stream = (cudaStream_t)stream_;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)cut.c, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr, cfg.numAttrs = 2;
    B200KV_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
    return B200KV_OK;
}
