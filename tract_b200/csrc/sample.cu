// b200kv_sample: the next token of every row of logits -- temperature, top-k, top-p, min-p -- for a given uniform number.
// It stands beside b200kv_argmax (ArgMax over the logits, examples/causal_llm/src/lib.rs:290-408 decodes greedily).
//
//   w_i = exp((x_i - max x) / T)
//   in the order of falling x, equal ones by rising index: the first k; of these the shortest beginning whose mass reaches
//   top_p x the mass of the k; of these the ones with w_i >= min_p       -- every filter keeps a beginning of the same order
//   token = the first kept index i, in rising order, with  sum_{kept j <= i} w_j > u x sum_kept w_j
//
// A token changes when u falls between a border of the distribution and its rounded value; 128k borders with the error of
// 32-bit sums would move one row in a hundred.  Weights are therefore 64-bit: doubles over whole slices of a row, and fixed
// point with 44 bits behind the point where single tokens are added up -- integer sums, so that the order in which threads
// add has no influence.
//
// Two launches.  sample_stats_kernel reads the logits once, a slice of a row per CTA: maximum and its place, mass (only where
// a filter or the draw needs the mass of the whole row), and a histogram of every eighth logit over octaves of w.
// sample_pick_kernel has one CTA per row: the histogram tells how deep the filters can reach, the tokens above that threshold
// are gathered into shared memory, the cut is found by radix refinement of their bit patterns (1024 bins of counts and masses
// per round), the token by the same refinement over the indices.  The threshold is an estimate and only that: whether the
// gathered tokens hold the cut is checked exactly, and if they do not, or do not fit, the rounds read the row itself.
// Without filters the draw picks the slice from the slices' masses and the token inside it.
// Bound: the logits once (4 bytes each in f32) plus 11 double operations per logit where the mass is needed.
#include <algorithm>
#include <cmath>

#include "internal.h"

namespace b200kv {

constexpr int ST_THREADS = 256;   // stats kernel
constexpr int PK_THREADS = 1024;  // pick kernel
constexpr int ST_BINS = 32;       // octaves of w below the slice's maximum; the last one takes everything deeper
constexpr int ST_SAMPLE = 8;      // one logit in this many enters the histogram
constexpr int PK_CHUNK = 8192;    // logits of a gathering step
constexpr int PK_BINS = 1024;     // bins of a refinement round
constexpr int PK_CAP = 5888;      // gathered tokens: 16 bytes each, two CTAs per SM
constexpr int W_BITS = 44;        // fractional bits of a fixed-point weight
constexpr int MAX_VOCAB = 1 << 19;  // so many weights of 1 add up to 2^63

struct SliceStats {
    double mass;    // sum of exp((x - max of the slice) / T)
    float max;      // -inf: no number above -inf
    int32_t at;     // first index of the maximum
};
struct SliceBins {
    uint32_t count[ST_BINS];
    float mass[ST_BINS];  // relative to 2^floor(max * log2 e / T)
};

struct SampleParams {
    const void* logits;
    int64_t stride;
    int32_t dtype, n, n_slices, slice;  // slice: elements per slice
    const float* temperature;
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    const float* uniform;
    int32_t* out;
    SliceStats* stats;  // [rows][n_slices]
    SliceBins* bins;    // [rows][n_slices]
    int32_t vec;        // rows start on 16-byte boundaries
};

// The settings of a row, with what means "off" made explicit.
struct RowSettings {
    float t, p, min_p, u;
    int32_t k;
    bool greedy, use_p, use_k, use_m;
    __device__ bool need_mass() const { return !greedy && !use_k && (use_p || !use_m); }
};
__device__ inline RowSettings row_settings(const SampleParams& p, int row) {
    RowSettings s;
    s.t = p.temperature ? p.temperature[row] : 1.f;
    s.k = p.top_k ? p.top_k[row] : 0;
    s.p = p.top_p ? p.top_p[row] : 1.f;
    s.min_p = p.min_p ? p.min_p[row] : 0.f;
    s.u = p.uniform[row];
    s.greedy = !(s.t > 0.f);
    s.use_k = s.k > 0 && s.k < p.n;
    s.use_p = s.p < 1.f;
    s.use_m = s.min_p > 0.f;
    s.min_p = fminf(s.min_p, 1.f);  // the likeliest token always stays
    if (s.use_p && !(s.p > 0.f)) s.use_k = true, s.k = 1, s.use_p = false;  // an empty beginning: the first token alone
    if (s.use_k && s.k == 1) s.greedy = true;
    return s;
}
__device__ inline float clean(float x) { return x != x ? -INFINITY : x + 0.f; }  // NaN is never chosen; -0 and +0 are the same logit
__device__ inline float load_logit(const SampleParams& p, const uint8_t* row, int64_t i) { return clean(ld_as_f32(row, p.dtype, i)); }
// monotone bit pattern of a logit
__device__ inline uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ inline float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
constexpr uint32_t KEY_NEG_INF = 0x007fffffu;

// w of a logit against the row's maximum, in 64 bits; a maximum of +inf shares the row among the infinite logits
__device__ inline double weight_of(float x, float max, double t) {
    if (x == max) return 1.0;
    if (x == -INFINITY || max == INFINITY) return 0.0;
    return exp(((double)x - (double)max) / t);
}
__device__ inline unsigned long long fixed_weight(float x, float max, double t) {
    return (unsigned long long)__double2ll_rn(weight_of(x, max, t) * (double)(1ull << W_BITS));
}

// ---- first launch ---------------------------------------------------------------------------------------------------------
// EPT logits per thread, all of them in registers: read once, used for the maximum, then for mass and histogram.
template <int EPT>
__global__ void __launch_bounds__(ST_THREADS) sample_stats_kernel(SampleParams p) {
    __shared__ float red_max[ST_THREADS / 32];
    __shared__ int red_at[ST_THREADS / 32];
    __shared__ double red_mass[ST_THREADS / 32];
    __shared__ double exp2_table[64];  // 2^(j / 64)
    __shared__ uint32_t bin_count[ST_BINS];
    __shared__ float bin_mass[ST_BINS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int slice = blockIdx.x, row = blockIdx.y;
    const int first = slice * p.slice, count = min(p.slice, p.n - first);
    if (tid < ST_BINS) bin_count[tid] = 0, bin_mass[tid] = 0.f;
    if (tid < 64) exp2_table[tid] = exp2((double)tid / 64.0);
    grid_launch_dependents();
    grid_dependency_wait();  // the kernel before has written the logits and the settings
    const RowSettings s = row_settings(p, row);
    const uint8_t* base = (const uint8_t*)p.logits + ((int64_t)row * p.stride + first) * dtype_size(p.dtype);

    float x[EPT];
    int at0, per;  // element e of this thread is at0 + (e / per) * per * ST_THREADS + e % per
    if (p.vec && p.dtype == B200KV_F32) {
        per = 4, at0 = tid * 4;
#pragma unroll
        for (int e = 0; e < EPT; e += 4) {
            const int i = at0 + e * ST_THREADS;
            if (i + 4 <= count) {
                const float4 v = *(const float4*)(base + (int64_t)i * 4);
                x[e] = v.x, x[e + 1] = v.y, x[e + 2] = v.z, x[e + 3] = v.w;
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++) x[e + j] = i + j < count ? ((const float*)base)[i + j] : -INFINITY;
            }
        }
    } else if (p.vec) {
        per = 8, at0 = tid * 8;
#pragma unroll
        for (int e = 0; e < EPT; e += 8) {
            const int i = at0 + e * ST_THREADS;
            if (i + 8 <= count) {
                const uint4 v = *(const uint4*)(base + (int64_t)i * 2);
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if (p.dtype == B200KV_F16) {
                        const float2 f = __half22float2(*(const __half2*)&w[j]);
                        x[e + 2 * j] = f.x, x[e + 2 * j + 1] = f.y;
                    } else {
                        x[e + 2 * j] = __uint_as_float(w[j] << 16), x[e + 2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
                    }
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) x[e + j] = i + j < count ? ld_as_f32(base, p.dtype, i + j) : -INFINITY;
            }
        }
    } else {
        per = 1, at0 = tid;
#pragma unroll
        for (int e = 0; e < EPT; e++) {
            const int i = at0 + e * ST_THREADS;
            x[e] = i < count ? ld_as_f32(base, p.dtype, i) : -INFINITY;
        }
    }
    float best = -INFINITY;
    int best_e = 0;
#pragma unroll
    for (int e = 0; e < EPT; e++) {  // a thread's elements come in rising order of their index
        x[e] = clean(x[e]);
        if (x[e] > best) best = x[e], best_e = e;
    }
    int at = best > -INFINITY ? first + at0 + (best_e / per) * per * ST_THREADS + best_e % per : 0x7fffffff;
    auto merge = [&](float ov, int oi) {
        if (ov > best || (ov == best && oi < at)) best = ov, at = oi;
    };
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const float ov = __shfl_xor_sync(0xffffffffu, best, o);
        const int oi = __shfl_xor_sync(0xffffffffu, at, o);
        merge(ov, oi);
    }
    if (lane == 0) red_max[warp] = best, red_at[warp] = at;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < ST_THREADS / 32; w++) merge(red_max[w], red_at[w]);

    double mass = 0.0;
    if (!s.greedy && best > -INFINITY) {
        if (s.need_mass()) {
            // exp((x - max) / T) = 2^(t / 64), t = (x - max) * 64 log2 e / T = n + r:  2^(n / 64) from the table and the exponent,
            // 2^(r / 64) by its Taylor polynomial of degree 4 in r ln 2 / 64 (|r| <= 1/2: the next term is below 4e-14)
            const double c = 64.0 * 1.4426950408889634074 / (double)s.t, m = (double)best;
            constexpr double L = 0.69314718055994530942 / 64.0, MAGIC = 6755399441055744.0;  // 1.5 * 2^52
            double part[2] = {0.0, 0.0};
#pragma unroll
            for (int e = 0; e < EPT; e++) {
                const double t = fmax(((double)x[e] - m) * c, -64.0 * 1000.0);  // below: 2^-1000, nothing beside the maximum's 1
                const double biased = t + MAGIC, r = t - (biased - MAGIC);
                const int n = __double2loint(biased);
                double q = fma(r, L * L * L * L / 24.0, L * L * L / 6.0);
                q = fma(q, r, L * L / 2.0);
                q = fma(q, r, L);
                q = fma(q, r, 1.0);
                const double tab = exp2_table[n & 63];
                const double scaled = __hiloint2double(__double2hiint(tab) + ((n >> 6) << 20), __double2loint(tab));
                part[e & 1] = fma(q, scaled, part[e & 1]);
            }
            mass = best == INFINITY ? 0.0 : part[0] + part[1];
            if (best == INFINITY) {
#pragma unroll
                for (int e = 0; e < EPT; e++) mass += x[e] == INFINITY ? 1.0 : 0.0;
            }
        }
        if (s.use_k || s.use_p) {
            const float c = 1.4426950408889634f / s.t, top = floorf(best * c);
#pragma unroll
            for (int e = 0; e < EPT; e += ST_SAMPLE) {
                if (x[e] > -INFINITY) {
                    const float z = x[e] * c;
                    const int j = (int)fmaxf(fminf(top - floorf(z), (float)(ST_BINS - 1)), 0.f);
                    atomicAdd(&bin_count[j], 1u);
                    atomicAdd(&bin_mass[j], exp2f(z - top));
                }
            }
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) mass += __shfl_xor_sync(0xffffffffu, mass, o);
        if (lane == 0) red_mass[warp] = mass;
    }
    __syncthreads();
    const int64_t slot = (int64_t)row * p.n_slices + slice;
    if (tid == 0) {
        double sum = 0.0;
        if (!s.greedy && best > -INFINITY)
            for (int w = 0; w < ST_THREADS / 32; w++) sum += red_mass[w];
        SliceStats st;
        st.mass = sum, st.max = best, st.at = at;
        p.stats[slot] = st;
    }
    if (tid < ST_BINS && !s.greedy && (s.use_k || s.use_p)) p.bins[slot].count[tid] = bin_count[tid], p.bins[slot].mass[tid] = bin_mass[tid];
}

// ---- second launch --------------------------------------------------------------------------------------------------------
// Inclusive sums over the CTA in thread order.
template <typename T>
__device__ inline T warp_scan(T v, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T up = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += up;
    }
    return v;
}
template <typename T>
__device__ inline T block_scan(T v, T* warp_sums /* [33] */) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    v = warp_scan(v, lane);
    __syncthreads();  // the sums of the scan before are no longer read
    if (lane == 31) warp_sums[warp] = v;
    __syncthreads();
    T before = T(0);
    if (warp > 0) {  // every warp adds up the sums before it
        T mine = lane < warp ? warp_sums[lane] : T(0);
#pragma unroll
        for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
        before = mine;
    }
    return before + v;
}

struct Token {
    unsigned long long w;
    uint32_t key;
    int32_t at;
};
struct PickShared {
    unsigned long long mass[PK_BINS];
    uint32_t count[PK_BINS];
    unsigned long long sums64[33];
    double sums_d[33];
    uint32_t sums32[33];
    float max;
    int32_t at;
    double total;
    uint32_t n_list;
    float bin_count[ST_BINS], bin_mass[ST_BINS];
    uint32_t hit;                      // bin of a refinement round
    uint32_t above_n;                  // what lies before that bin
    unsigned long long above_w;
    unsigned long long list_mass;
    int32_t token;
    float theta;
};

__global__ void __launch_bounds__(PK_THREADS, 2) sample_pick_kernel(SampleParams p) {
    extern __shared__ __align__(16) uint8_t pick_smem[];
    Token* list = (Token*)pick_smem;
    PickShared& sh = *(PickShared*)(pick_smem + PK_CAP * sizeof(Token));
    const int tid = threadIdx.x, lane = tid & 31, row = blockIdx.x;
    grid_launch_dependents();
    grid_dependency_wait();
    const RowSettings s = row_settings(p, row);
    const SliceStats* stats = p.stats + (int64_t)row * p.n_slices;
    const SliceBins* bins = p.bins + (int64_t)row * p.n_slices;
    const uint8_t* base = (const uint8_t*)p.logits + (int64_t)row * p.stride * dtype_size(p.dtype);

    // ---- the row's maximum and its first index ----
    if (tid < 32) {
        float best = -INFINITY;
        int at = 0x7fffffff;
        for (int i = lane; i < p.n_slices; i += 32) {
            const float m = stats[i].max;
            if (m > best) best = m, at = stats[i].at;  // slices in rising order: the first maximum of this lane
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            const float ov = __shfl_xor_sync(0xffffffffu, best, o);
            const int oi = __shfl_xor_sync(0xffffffffu, at, o);
            if (ov > best || (ov == best && oi < at)) best = ov, at = oi;
        }
        if (lane == 0) sh.max = best, sh.at = best > -INFINITY ? at : 0;  // a row of -inf / NaN only: index 0
    }
    if (tid == 0) sh.token = -1, sh.n_list = 0, sh.list_mass = 0;
    if (tid < ST_BINS) sh.bin_count[tid] = 0.f, sh.bin_mass[tid] = 0.f;
    __syncthreads();
    const float max = sh.max;
    if (s.greedy || max == -INFINITY) {
        if (tid == 0) p.out[row] = sh.at;
        return;
    }
    const double t = (double)s.t;
    const float u = s.u > 0.f ? fminf(s.u, 1.f) : 0.f;

    // ---- the mass of the row, relative to its maximum; without filters also the slice in which the draw falls ----
    double total = 0.0;
    if (s.need_mass()) {
        auto slice_mass = [&](int i) -> double {
            if (i >= p.n_slices) return 0.0;
            return stats[i].mass * weight_of(stats[i].max, max, t);
        };
        for (int i0 = 0; i0 < p.n_slices; i0 += PK_THREADS) {
            const double incl = block_scan(slice_mass(i0 + tid), sh.sums_d);
            if (tid == PK_THREADS - 1) sh.total = incl;
            __syncthreads();
            total += sh.total;
        }
        if (!s.use_p && !s.use_m) {
            double target = (double)u * total, before = 0.0;
            for (int i0 = 0; i0 < p.n_slices; i0 += PK_THREADS) {
                const double mine = slice_mass(i0 + tid), incl = block_scan(mine, sh.sums_d) + before;
                // several may pass where rounding makes the sums meet: the first one is taken
                if (mine > 0.0 && incl > target) atomicMin((unsigned int*)&sh.token, (unsigned)(i0 + tid));  // -1 is the largest
                if (tid == PK_THREADS - 1) sh.total = incl;
                __syncthreads();
                before = sh.total;
                if (sh.token >= 0) break;
            }
            int slice = sh.token;
            __syncthreads();
            if (slice < 0) {  // the draw is past the last sum by a rounding: the last slice that has mass
                for (int i = tid; i < p.n_slices; i += PK_THREADS)
                    if (stats[i].mass > 0.0 && weight_of(stats[i].max, max, t) > 0.0) atomicMax(&sh.token, i);
                __syncthreads();
                slice = sh.token;
            }
            // what lies before the slice, added up in the same order as above
            double prior = 0.0;
            for (int i0 = 0; i0 <= slice; i0 += PK_THREADS) {
                const double incl = block_scan(i0 + tid < slice ? slice_mass(i0 + tid) : 0.0, sh.sums_d);
                if (tid == PK_THREADS - 1) sh.total = incl;
                __syncthreads();
                prior += sh.total;
            }
            target -= prior;
            if (tid == 0) sh.token = -1;
            // the token: every thread adds up a run of the slice
            const int first = slice * p.slice, count = min(p.slice, p.n - first), per = (count + PK_THREADS - 1) / PK_THREADS;
            double mine = 0.0;
            for (int e = 0; e < per; e++) {
                const int i = tid * per + e;
                if (i < count) mine += weight_of(load_logit(p, base, first + i), max, t);
            }
            const double incl = block_scan(mine, sh.sums_d);
            double run = incl - mine;
            if (mine > 0.0 && incl > target) {
                int pick = 0x7fffffff, last = 0x7fffffff;
                for (int e = 0; e < per; e++) {
                    const int i = tid * per + e;
                    if (i >= count) break;
                    const double w = weight_of(load_logit(p, base, first + i), max, t);
                    run += w;
                    if (w > 0.0) last = first + i;
                    if (w > 0.0 && run > target) {
                        pick = first + i;
                        break;
                    }
                }
                atomicMin((unsigned int*)&sh.token, (unsigned)(pick != 0x7fffffff ? pick : last));
            }
            __syncthreads();
            int token = sh.token;
            if (token < 0) {  // past the slice's last sum by a rounding: its last token that has weight
                for (int i = tid; i < count; i += PK_THREADS)
                    if (weight_of(load_logit(p, base, first + i), max, t) > 0.0) atomicMax(&sh.token, first + i);
                __syncthreads();
                token = sh.token;
            }
            if (tid == 0) p.out[row] = token;
            return;
        }
    }

    // ---- how deep the filters reach ----
    const float c = 1.4426950408889634f / s.t, top = floorf(max * c);
    uint32_t key_m = KEY_NEG_INF + 1;  // min-p: the smallest bit pattern that passes
    if (s.use_m) {
        if (tid == 0) {
            // x = max + T ln(min_p) up to rounding, then the neighbours: w is monotone in x
            const float guess = max == INFINITY ? max : (float)((double)max + t * log((double)s.min_p));
            uint32_t k = std::max(KEY_NEG_INF + 1, std::min(key_of(clean(guess)), key_of(max)));
            for (int i = 0; i < 4096 && k > KEY_NEG_INF + 1 && weight_of(of_key(k - 1), max, t) >= (double)s.min_p; i++) k--;
            for (int i = 0; i < 4096 && k < key_of(max) && !(weight_of(of_key(k), max, t) >= (double)s.min_p); i++) k++;
            sh.hit = k;
        }
        __syncthreads();
        key_m = sh.hit;
    }
    if (s.use_k || s.use_p) {
        for (int i = tid; i < p.n_slices * ST_BINS; i += PK_THREADS) {
            const int sl = i / ST_BINS;
            const uint32_t n = bins[sl].count[i % ST_BINS];
            if (!n) continue;
            const float lower = top - floorf(stats[sl].max * c);
            const int j = (int)fmaxf(fminf((float)(i % ST_BINS) + lower, (float)(ST_BINS - 1)), 0.f);
            atomicAdd(&sh.bin_count[j], (float)n);
            atomicAdd(&sh.bin_mass[j], bins[sl].mass[i % ST_BINS] * exp2f(-lower));
        }
        __syncthreads();
        if (tid == 0) {
            int j = ST_BINS - 1;  // the last octave to gather; the last bin of all: everything
            if (s.use_k) {
                float n = 0.f;
                for (int b = 0; b < ST_BINS - 1; b++) {
                    n += sh.bin_count[b] * ST_SAMPLE;
                    if (n >= 1.5f * (float)s.k + 100.f) {
                        j = b;
                        break;
                    }
                }
            } else {
                const float allowed = 0.7f * (1.f - s.p) * (float)total * exp2f(max * c - top);
                float tail = 0.f;
                for (int b = ST_BINS - 1; b > 0; b--) {
                    tail += sh.bin_mass[b] * ST_SAMPLE;
                    if (!(tail <= allowed)) break;
                    j = b - 1;
                }
            }
            const float theta = (top - (float)j) / c;
            sh.theta = j == ST_BINS - 1 || !(theta < max) ? -INFINITY : theta;
        }
        __syncthreads();
    }
    uint32_t theta = s.use_k || s.use_p ? std::max(key_of(clean(sh.theta)), KEY_NEG_INF + 1) : KEY_NEG_INF + 1;
    if (s.use_m && !s.use_k) theta = std::max(theta, key_m);  // nothing below passes min-p, and no mass below is asked for one by one

    // ---- gather ----
    const double unit = (double)(1ull << W_BITS);
    const unsigned long long reach = s.use_p && !s.use_k ? (unsigned long long)ceil((double)s.p * total * unit) : 0ull;
    bool in_list;
    uint32_t n_list;
    for (;;) {
        const float theta_x = of_key(theta);
        const int per_chunk = PK_CHUNK / p.slice;  // slices, of 2048 or 8192 logits, in a chunk
        for (int chunk = 0; chunk * PK_CHUNK < p.n; chunk++) {
            bool any = false;
            for (int sl = chunk * per_chunk; sl < min((chunk + 1) * per_chunk, p.n_slices); sl++) any |= stats[sl].max >= theta_x;
            if (!any) continue;
            float x[PK_CHUNK / PK_THREADS];  // all of them in flight
#pragma unroll
            for (int e = 0; e < PK_CHUNK / PK_THREADS; e++) {
                const int i = chunk * PK_CHUNK + e * PK_THREADS + tid;
                x[e] = i < p.n ? load_logit(p, base, i) : -INFINITY;
            }
#pragma unroll
            for (int e = 0; e < PK_CHUNK / PK_THREADS; e++) {
                const bool take = x[e] >= theta_x;
                const uint32_t vote = __ballot_sync(0xffffffffu, take);
                if (vote) {
                    uint32_t at = 0;
                    if (lane == 0) at = atomicAdd(&sh.n_list, (uint32_t)__popc(vote));
                    at = __shfl_sync(0xffffffffu, at, 0) + (uint32_t)__popc(vote & ((1u << lane) - 1u));
                    if (take && at < PK_CAP) list[at] = {0ull, key_of(x[e]), chunk * PK_CHUNK + e * PK_THREADS + tid};
                }
            }
        }
        __syncthreads();
        n_list = sh.n_list;
        in_list = n_list <= PK_CAP;
        if (in_list) {
            unsigned long long mine = 0;
            for (uint32_t i = tid; i < n_list; i += PK_THREADS) {
                const unsigned long long w = fixed_weight(of_key(list[i].key), max, t);
                list[i].w = w;
                mine += w;
            }
            atomicAdd(&sh.list_mass, mine);
        }
        __syncthreads();
        const unsigned long long list_mass = sh.list_mass;
        // does the cut lie among the gathered ones?
        const bool covered = theta <= KEY_NEG_INF + 1 || !in_list || (s.use_k ? n_list >= (uint32_t)s.k : !s.use_p || list_mass >= reach || (s.use_m && theta == key_m));
        __syncthreads();
        if (covered) break;
        theta = s.use_m && !s.use_k ? key_m : KEY_NEG_INF + 1;
        if (tid == 0) sh.n_list = 0, sh.list_mass = 0;
        __syncthreads();
    }
    // f(key, index, weight) for every gathered token: from the list, or from the row
    auto for_each = [&](auto f) {
        if (in_list) {
            for (uint32_t i = tid; i < n_list; i += PK_THREADS) f(list[i].key, list[i].at, list[i].w);
        } else {
            for (int i = tid; i < p.n; i += PK_THREADS) {
                const float x = load_logit(p, base, i);
                const uint32_t key = key_of(x);
                if (key >= theta) f(key, i, fixed_weight(x, max, t));
            }
        }
    };
    // One refinement: of the tokens that `part` admits, `place` gives the position on an axis, [lo, hi].  Finds the position at
    // which the sum (of weights, or of ones) first exceeds `target`, and what lies before it; hi + 1 if it never does.
    struct Found {
        uint32_t at, n;
        unsigned long long w;
        uint32_t n_here;
        unsigned long long w_here;
    };
    auto refine = [&](uint32_t lo, uint32_t hi, unsigned long long target, bool by_weight, auto place, auto part) -> Found {
        Found r{hi, 0, 0, 0, 0};
        const uint32_t end = hi;
        uint32_t n_before = 0;
        unsigned long long w_before = 0;
        for (;;) {
            const uint32_t range = hi - lo;
            const int bits = 32 - __clz(range | 1u), shift = bits > 10 ? bits - 10 : 0;
            sh.count[tid] = 0, sh.mass[tid] = 0;
            if (tid == 0) sh.hit = 0xffffffffu;
            __syncthreads();
            for_each([&](uint32_t key, int32_t at, unsigned long long w) {
                const uint32_t x = place(key, at);
                if (x < lo || x > hi || !part(key, at)) return;
                const uint32_t b = (x - lo) >> shift;
                atomicAdd(&sh.count[b], 1u);
                if (w) atomicAdd(&sh.mass[b], w);
            });
            __syncthreads();
            const uint32_t n = sh.count[tid];
            const unsigned long long w = sh.mass[tid];
            const unsigned long long w_incl = block_scan(w, sh.sums64) + w_before;
            const uint32_t n_incl = block_scan(n, sh.sums32) + n_before;
            const unsigned long long incl = by_weight ? w_incl : (unsigned long long)n_incl;
            const unsigned long long excl = by_weight ? w_incl - w : (unsigned long long)(n_incl - n);
            if (excl <= target && incl > target) sh.hit = (uint32_t)tid, sh.above_n = n_incl - n, sh.above_w = w_incl - w;
            __syncthreads();
            const uint32_t hit = sh.hit;
            if (hit == 0xffffffffu) {
                __syncthreads();
                return Found{end + 1, 0, 0, 0, 0};
            }
            n_before = sh.above_n, w_before = sh.above_w;
            r.at = lo + (hit << shift), r.n = n_before, r.w = w_before, r.n_here = sh.count[hit], r.w_here = sh.mass[hit];
            __syncthreads();
            if (shift == 0) return r;
            hi = std::min(hi, r.at + ((1u << shift) - 1u));
            lo = r.at;
        }
    };
    // ---- the cut: everything above key_cut, and the first n_cut tokens (by index) of those that equal it ----
    const uint32_t key_max = key_of(max);
    auto by_rank = [&](uint32_t key, int32_t) { return key_max - key; };  // positions rise as logits fall
    auto all = [](uint32_t, int32_t) { return true; };
    uint32_t key_cut = theta, n_cut = 0xffffffffu, n_same = 0xffffffffu;
    unsigned long long mass_k = 0;
    if (s.use_k) {
        const Found f = refine(0, key_max - theta, (unsigned long long)(s.k - 1), false, by_rank, all);
        if (f.at <= key_max - theta) {
            key_cut = key_max - f.at, n_cut = (uint32_t)s.k - f.n, n_same = f.n_here;
            mass_k = f.w + (unsigned long long)n_cut * (f.w_here / f.n_here);
        } else {
            // fewer tokens than k: all of them
            for_each([&](uint32_t, int32_t, unsigned long long w) { mass_k += w; });
            mass_k = block_scan(mass_k, sh.sums64);
            if (tid == PK_THREADS - 1) sh.above_w = mass_k;
            __syncthreads();
            mass_k = sh.above_w;
            __syncthreads();
        }
    }
    if (s.use_p) {
        const double whole = s.use_k ? (double)mass_k : total * unit;
        const double goal = (double)s.p * whole;  // kept while the mass before is below it: cut at the first sum >= goal
        const unsigned long long least = (unsigned long long)ceil(goal);
        const Found f = refine(0, key_max - key_cut, least ? least - 1 : 0, true, by_rank, all);
        if (f.at <= key_max - key_cut) {
            const unsigned long long w = f.w_here / f.n_here, missing = least > f.w ? least - f.w : 1;
            const unsigned long long need = w ? (missing + w - 1) / w : 1;
            const uint32_t n = (uint32_t)std::min<unsigned long long>(std::max<unsigned long long>(need, 1), f.n_here);
            const uint32_t key = key_max - f.at;
            if (key > key_cut || n < n_cut) key_cut = key, n_cut = n, n_same = f.n_here;
        }
    }
    if (s.use_m && key_m > key_cut) key_cut = key_m, n_cut = n_same = 0xffffffffu;
    // ---- the last index among the equal ones that is kept ----
    uint32_t last_same = 0xffffffffu;
    if (n_cut < n_same) {
        const Found f = refine(0, (uint32_t)p.n - 1, (unsigned long long)(n_cut - 1), false, [](uint32_t, int32_t at) { return (uint32_t)at; },
                               [&](uint32_t key, int32_t) { return key == key_cut; });
        last_same = f.at;
    }
    auto kept = [&](uint32_t key, int32_t at) { return key > key_cut || (key == key_cut && (uint32_t)at <= last_same); };
    // ---- the draw ----
    unsigned long long mass = 0;
    for_each([&](uint32_t key, int32_t at, unsigned long long w) {
        if (kept(key, at)) mass += w;
    });
    mass = block_scan(mass, sh.sums64);
    if (tid == PK_THREADS - 1) sh.above_w = mass;
    __syncthreads();
    mass = sh.above_w;
    __syncthreads();
    const unsigned long long target = std::min((unsigned long long)((double)u * (double)mass), mass - 1);
    const Found f = refine(0, (uint32_t)p.n - 1, target, true, [](uint32_t, int32_t at) { return (uint32_t)at; }, kept);
    if (tid == 0) p.out[row] = (int32_t)f.at;
}

// Slices of 8 logits per thread where a launch would otherwise leave SMs without work (a row of 128256 logits is then 63
// CTAs instead of 16), of 32 otherwise: fewer slices to merge and more loads in flight per thread.
static int slice_elements(int64_t rows, int32_t n) {
    const int64_t wide = ST_THREADS * 32;
    return rows * ((n + wide - 1) / wide) >= 4 * 148 ? (int)wide : ST_THREADS * 8;
}

}  // namespace b200kv

using namespace b200kv;

extern "C" int64_t b200kv_sample_scratch_bytes(int64_t rows, int32_t n) {
    if (rows <= 0 || n <= 0) {
        fail("rows and n must be positive");
        return -1;
    }
    const int64_t slice = ST_THREADS * 8;  // the finer cut needs more
    return rows * ((n + slice - 1) / slice) * (int64_t)(sizeof(SliceStats) + sizeof(SliceBins));
}

extern "C" int b200kv_sample(const void* logits, int64_t stride, int32_t dtype, int64_t rows, int32_t n, const float* temperature,
                             const int32_t* top_k, const float* top_p, const float* min_p, const float* uniform, int32_t* out, void* scratch,
                             void* stream_) {
    if (!logits || !uniform || !out || !scratch) return fail("null tensor");
    if (rows <= 0 || n <= 0) return fail("rows and n must be positive");
    if (rows > 65535) return fail("%lld rows in one call: at most 65535", (long long)rows);
    if (n > MAX_VOCAB) return fail("a vocabulary of %d tokens: at most %d", n, MAX_VOCAB);
    if (dtype < B200KV_F32 || dtype > B200KV_BF16) return fail("unknown dtype %d", dtype);
    if (stride < n && rows > 1) return fail("rows of %d logits cannot be %lld elements apart", n, (long long)stride);
    if ((uintptr_t)scratch % 16) return fail("scratch must be 16-byte aligned");
    cudaStream_t stream = (cudaStream_t)stream_;
    SampleParams p{};
    p.logits = logits, p.stride = stride, p.dtype = dtype, p.n = n;
    p.slice = slice_elements(rows, n), p.n_slices = (n + p.slice - 1) / p.slice;
    p.temperature = temperature, p.top_k = top_k, p.top_p = top_p, p.min_p = min_p, p.uniform = uniform, p.out = out;
    p.stats = (SliceStats*)scratch, p.bins = (SliceBins*)(p.stats + rows * p.n_slices);
    p.vec = (uintptr_t)logits % 16 == 0 && (stride * dtype_size(dtype)) % 16 == 0;
    const dim3 grid((unsigned)p.n_slices, (unsigned)rows);
    if (p.slice == ST_THREADS * 32) B200KV_CUDA(launch_after_predecessor(sample_stats_kernel<32>, grid, dim3(ST_THREADS), 0, stream, p));
    else B200KV_CUDA(launch_after_predecessor(sample_stats_kernel<8>, grid, dim3(ST_THREADS), 0, stream, p));
    constexpr size_t smem = PK_CAP * sizeof(Token) + sizeof(PickShared);
    B200KV_CUDA(cudaFuncSetAttribute(sample_pick_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    B200KV_CUDA(launch_after_predecessor(sample_pick_kernel, dim3((unsigned)rows), dim3(PK_THREADS), smem, stream, p));
    return B200KV_OK;
}
