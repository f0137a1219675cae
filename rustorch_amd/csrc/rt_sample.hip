// Sampling of one token per row of logits on the device: what rustorch_amd/sampling.py does on the host
// (example-cli/src/model/sampling.rs:118-274 of the reference), with min-p beside top-k and top-p, from given random numbers.
//
// With M the row's largest logit and T its temperature, token i weighs w_i = exp((l_i - M) / T).  Sorted by logit, equal
// logits by index, the tokens that may be drawn are a prefix of the row whatever the settings say: the first top_k; of these
// the shortest prefix whose weight reaches top_p of theirs; of these the ones with w_i >= min_p.  The draw runs over them by
// index: the first token whose running weight exceeds u times their total.
//
// Weights are 64-bit integers, round(w_i * 2^F) with 2^F * vocab <= 2^62: sums of them are exact in any order, so the cut and
// the draw do not depend on how the row is split over threads, and a token is lost to rounding only below 2^-(F+1) of the
// largest weight (F = 45 for a vocabulary of 131072).  32-bit sums would move the cuts of a large vocabulary by whole tokens.
//
// Large vocabularies take four launches.  sample_range_kernel finds each row's largest and smallest logit, sample_histogram_kernel counts
// and weighs the tokens by how far below it they are, sample_collect_kernel finds from the histogram the bins that the cuts fall
// into, lists the tokens of just those bins and sums the weights of the tokens above them, sample_finish_kernel ranks the listed
// tokens exactly and draws.  The first three split a row over as many workgroups as fill the device.  Up to 32768 tokens one workgroup
// does all of it for its row in one launch (sample_row_kernel).
#include "rt_device.h"

#include <algorithm>

namespace rt {
namespace {

struct SampleArgs {
    const float *logits;
    size_t ld;
    int n_rows, vocab, frac_bits;
    const double *u;
    const float *temperature, *top_p, *min_p;      // nullptr: 1, off, off
    const int *top_k;                              // nullptr: off
    int *out_token;
    float *out_prob;                               // nullptr: not wanted
};

// Larger for larger logits; NaN counts as -inf and -0 as +0.
__device__ __forceinline__ uint32_t logit_order(float x) {
    x = x != x ? -INFINITY : x + 0.0f;
    const uint32_t b = (uint32_t)__float_as_int(x);
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float order_logit(uint32_t o) { return __uint_as_float((o & 0x80000000u) ? o & 0x7FFFFFFFu : ~o); }
// x above -inf; beside an infinite largest logit everything finite weighs nothing, whatever the temperature
__device__ __forceinline__ double weight_of(float x, float top, double temperature) {
    return x == top ? 1.0 : (top == INFINITY ? 0.0 : exp(((double)x - (double)top) / temperature));
}
__device__ __forceinline__ unsigned long long fixed_weight(float x, float top, double temperature, int frac_bits) {
    return (unsigned long long)rint(ldexp(weight_of(x, top, temperature), frac_bits));
}

// Running sum over the lanes of a wave, this one's included: shifts inside the rows of 16 lanes, then the rows' ends passed on
// (one vector instruction a step; a shuffle through LDS takes ten times as long, and these sums wait for one another).
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned long long dpp_add_u64(unsigned long long v) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xf, false);
    return v + (((unsigned long long)hi << 32) | lo);
}
__device__ __forceinline__ unsigned long long wave_scan_u64(unsigned long long v) {
    v = dpp_add_u64<0x111, 0xf>(v);          // row_shr:1, 2, 4, 8
    v = dpp_add_u64<0x112, 0xf>(v);
    v = dpp_add_u64<0x114, 0xf>(v);
    v = dpp_add_u64<0x118, 0xf>(v);
    v = dpp_add_u64<0x142, 0xa>(v);          // row_bcast:15 into rows 1 and 3
    return dpp_add_u64<0x143, 0xc>(v);       // row_bcast:31 into rows 2 and 3
}
__device__ __forceinline__ unsigned long long lane_u64(unsigned long long v, int l) {
    return ((unsigned long long)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), l) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, l);
}
__device__ __forceinline__ unsigned long long wave_sum_u64(unsigned long long v) { return lane_u64(wave_scan_u64(v), 63); }
// the wave's largest value, smallest value, by the same steps
template <class F>
__device__ __forceinline__ int wave_fold(int v, F f) {
    v = f(v, __builtin_amdgcn_update_dpp(v, v, 0x111, 0xf, 0xf, false));
    v = f(v, __builtin_amdgcn_update_dpp(v, v, 0x112, 0xf, 0xf, false));
    v = f(v, __builtin_amdgcn_update_dpp(v, v, 0x114, 0xf, 0xf, false));
    v = f(v, __builtin_amdgcn_update_dpp(v, v, 0x118, 0xf, 0xf, false));
    v = f(v, __builtin_amdgcn_update_dpp(v, v, 0x142, 0xa, 0xf, false));
    v = f(v, __builtin_amdgcn_update_dpp(v, v, 0x143, 0xc, 0xf, false));
    return __builtin_amdgcn_readlane(v, 63);
}
__device__ __forceinline__ float wave_top(float v) {
    return __int_as_float(wave_fold(__float_as_int(v), [](int a, int b) { return __float_as_int(fmaxf(__int_as_float(a), __int_as_float(b))); }));
}
__device__ __forceinline__ float wave_low(float v) {
    return __int_as_float(wave_fold(__float_as_int(v), [](int a, int b) { return __float_as_int(fminf(__int_as_float(a), __int_as_float(b))); }));
}
__device__ __forceinline__ int wave_low(int v) {
    return wave_fold(v, [](int a, int b) { return min(a, b); });
}
// Every thread of the workgroup gets the sum; red holds one value per wave.
__device__ __forceinline__ unsigned long long block_sum_u64(unsigned long long v, unsigned long long *red) {
    v = wave_sum_u64(v);
    const int nw = (int)(blockDim.x >> 6);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    unsigned long long t = 0;
    for (int i = 0; i < nw; i++) t += red[i];
    return t;
}

// ---- bins: a row's tokens by their distance d = M - l below the largest logit, up to the distance R beyond which the weight
// rounds to zero (or the smallest logit, if that is nearer).  The bin's number is d * (kBins - 1) / R in f32: only its
// being monotone in d matters, and that the last bin ends past R.
// 4096 bins hold at most a hundred tokens each where the cuts of real rows fall; 1024 held several hundred, whose ranking (every
// one against every other) took most of the time.
constexpr int kBins = 4096, kThreads = 256, kCountThreads = 1024, kCoarse = kBins / 64, kListMost = 2048, kFewMost = kListMost / 2, kPart = 4096, kCountSort = 128;

struct RowRange { float top, low; int arg, pad; };        // of one split of a row: largest and smallest logit; where only the largest counts, its index
// What the histogram says of a row's cuts.
struct RowBorders {
    unsigned long long all;                                // weight of the row
    unsigned long long k_weight_above, k_weight_with;      // above the bin that top-k ends in, and with it
    unsigned long long k_above, k_in;                      // tokens above that bin and in it
    unsigned long long k;                                  // top-k, 0 where it keeps every token that weighs anything
    unsigned long long above_list;                         // weight above the first listed bin of top-p
    int k_bin;                                             // kBins: no top-k
    int p_first, p_last;                                   // the bins that top-p may end in (p_last = -1: no top-p)
    int keep_below;                                        // bins below this one stay whole
};
constexpr RowBorders kNoBorders{ 0, 0, 0, 0, 0, 0, 0, kBins, 0, -1, kBins };
struct SampleWork {
    RowRange *range;                                       // [row][split]
    unsigned long long *sum;                               // [row][kBins]
    uint32_t *count;                                       // [row][kBins]
    unsigned long long *coarse_sum;                        // [row][64], the same of kBins / 64 bins at a time
    uint32_t *coarse_count;
    RowBorders *borders;                                   // [row]
    int *listed;                                           // [row]: tokens listed
    unsigned long long *list;                              // [row][kListMost]: their keys
    unsigned long long *part_sum;                          // [row][part]: weight that stays whole, of kPart tokens each
    int row0;                                              // this launch's first row
    int splits, per_split, per_count, parts, parts_each;
};

struct RowBins {
    double top, rate;             // rate = log2(e) / T
    float topf, half_top, scale;
    int frac_bits;
};
__device__ __forceinline__ RowBins row_bins(float top, float low, double T, int frac_bits) {
    const double reach = (double)(frac_bits + 1) * 0.69314718055994531 * T, span = (double)top - (double)low, R = reach < span ? reach : span;
    RowBins b;
    b.top = (double)top;
    b.rate = 1.4426950408889634 / T;
    b.topf = top;
    b.half_top = 0.5f * top;      // half of d always fits f32
    b.scale = R > 0.0 ? fminf((float)(kBins - 1) / (float)(0.5 * R), 1e37f) : 0.0f;
    b.frac_bits = frac_bits;
    return b;
}
__device__ __forceinline__ float bin_at(const RowBins &b, float x) { return (b.half_top - 0.5f * x) * b.scale; }      // NaN, or kBins and more: no bin
__device__ __forceinline__ int bin_of(const RowBins &b, float x) {
    const float at = bin_at(b, x);
    return at < (float)kBins ? (int)at : kBins;                          // false for NaN
}
// exp((x - M) / T) * 2^frac_bits in 64 bits: 2^t with t split into a whole number and |f| <= 1/2, the latter by the series of the
// exponential to the twelfth power (the next term is below 2^-52): eighteen operations, a third of what exp() takes.
__device__ __forceinline__ double token_weight(const RowBins &b, float x) {
    if (x == b.topf) return ldexp(1.0, b.frac_bits);
    const double t = fmax(((double)x - b.top) * b.rate, -2000.0), n = rint(t), y = (t - n) * 0.69314718055994531;
    double e = fma(y, 1.0 / 479001600.0, 1.0 / 39916800.0);
    e = fma(e, y, 1.0 / 3628800.0);
    e = fma(e, y, 1.0 / 362880.0);
    e = fma(e, y, 1.0 / 40320.0);
    e = fma(e, y, 1.0 / 5040.0);
    e = fma(e, y, 1.0 / 720.0);
    e = fma(e, y, 1.0 / 120.0);
    e = fma(e, y, 1.0 / 24.0);
    e = fma(e, y, 1.0 / 6.0);
    e = fma(e, y, 0.5);
    e = fma(e, y, 1.0);
    e = fma(e, y, 1.0);
    return ldexp(e, (int)n + b.frac_bits);
}
__device__ __forceinline__ unsigned long long whole(double w) {          // rounded to nearest, 0 <= w <= 2^51: the sum's last bits
    return __builtin_bit_cast(unsigned long long, w + 4503599627370496.0) - 0x4330000000000000ull;
}

// What a row asks for.
struct RowAsks {
    double T, min_w;
    float p;                      // 0: off
    int k;                        // 0: off
    bool greedy;
    bool few;                     // top-k so small that all its tokens are listed: nothing has to be weighed before
};
__device__ __forceinline__ RowAsks row_asks(const SampleArgs &a, int r) {
    // one load each, none behind a branch, so that they go out together: a setting left out reads the row's random number instead
    const float *none = reinterpret_cast<const float *>(a.u + r);
    const float t0 = *(a.temperature ? a.temperature + r : none), p0 = *(a.top_p ? a.top_p + r : none), low0 = *(a.min_p ? a.min_p + r : none);
    const int k0 = *(a.top_k ? a.top_k + r : reinterpret_cast<const int *>(none));
    const float t = a.temperature ? t0 : 1.0f, p = a.top_p ? p0 : 0.f, low = a.min_p ? low0 : 0.f;
    RowAsks q;
    q.k = a.top_k ? k0 : 0;
    q.greedy = !(t > 0.f) || q.k == 1;       // temperature 0: the largest, the lowest index among equals
    if (q.k < 0 || q.k >= a.vocab) q.k = 0;
    q.few = q.k > 0 && q.k <= kFewMost;
    q.T = (double)t;
    q.p = p > 0.f && p < 1.f ? p : 0.f;
    q.min_w = low > 0.f ? fmin((double)low, 1.0) : 0.0;
    return q;
}

// the range of all lanes' ranges
__device__ __forceinline__ void fold_range(RowRange &g) {
    const float top = wave_top(g.top);
    g.arg = wave_low(g.top == top ? g.arg : INT32_MAX);
    g.top = top;
    g.low = wave_low(g.low);
}
// Orders the LDS traffic of one wave: the hardware runs it in order, the compiler may not move it across this point.
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
// A row with nothing to draw from, or nothing to draw: written here.
__device__ __forceinline__ bool undrawn_row(const SampleArgs &a, int r, const RowAsks &q, const RowRange &g) {
    if (g.top != -INFINITY && !q.greedy) return false;
    if (threadIdx.x == 0) {
        a.out_token[r] = g.top == -INFINITY ? -1 : g.arg;
        if (a.out_prob) a.out_prob[r] = g.top == -INFINITY ? 0.f : 1.f;
    }
    return true;
}

// N values, STEP apart, of a row of which `left` are left from x on (the same for all threads); NaN behind its end.  The requests
// go out together.
template <int N, int STEP>
__device__ __forceinline__ void load_steps(const float *x, int left, float (&v)[N]) {
    const unsigned tid = threadIdx.x;
    if (left >= N * STEP) {
#pragma unroll
        for (int j = 0; j < N; j++) v[j] = (x + j * STEP)[tid];
    } else {
#pragma unroll
        for (int j = 0; j < N; j++) v[j] = (int)tid + j * STEP < left ? (x + j * STEP)[tid] : NAN;
    }
}

// The lowest index at which the n values from x on are equal to `top`, counted from `from`; INT32_MAX for none.  STEP threads.
template <int STEP>
__device__ __forceinline__ int first_of(const float *x, int n, int from, float top) {
    int arg = INT32_MAX;
#pragma unroll 1
    for (int i = 0; i < n; i += 8 * STEP) {
        float v[8];
        load_steps<8, STEP>(x + i, n - i, v);
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (v[j] == top) arg = min(arg, from + i + j * STEP + (int)threadIdx.x);
    }
    return arg;
}

// The range of one split of a row; also clears the split's share of the row's histogram.
__global__ __launch_bounds__(kThreads) void sample_range_kernel(SampleArgs a, SampleWork w) {
    __shared__ float tops[4], lows[4];
    __shared__ int args[4];
    const int tid = threadIdx.x, split = blockIdx.x, row = blockIdx.y, r = w.row0 + row;
    const float *x = a.logits + (size_t)r * a.ld;
    const int i0 = split * w.per_split, n = max(0, min(a.vocab, i0 + w.per_split) - i0);
    float top = -INFINITY, low = INFINITY;
    for (int i = 0; i < n; i += 8 * kThreads) {
        float v[8];
        load_steps<8, kThreads>(x + i0 + i, n - i, v);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            top = fmaxf(top, v[j]);                             // NaN: neither
            low = fminf(low, v[j]);
        }
    }
    top = wave_top(top);
    low = wave_low(low);
    if ((tid & 63) == 0) { tops[tid >> 6] = top; lows[tid >> 6] = low; }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kThreads / 64; i++) {
        top = fmaxf(top, tops[i]);
        low = fminf(low, lows[i]);
    }
    int arg = row_asks(a, r).greedy ? first_of<kThreads>(x + i0, n, i0, top) : INT32_MAX;
    arg = wave_low(arg);
    if ((tid & 63) == 0) args[tid >> 6] = arg;
    __syncthreads();
    if (tid == 0) {
        for (int i = 1; i < kThreads / 64; i++) arg = min(arg, args[i]);
        w.range[(size_t)row * w.splits + split] = RowRange{ top, low, arg, 0 };
    }
    if (split == 0) {
        if (tid == 0) w.listed[row] = 0;
        if (tid < kCoarse) {
            w.coarse_sum[(size_t)row * kCoarse + tid] = 0;
            w.coarse_count[(size_t)row * kCoarse + tid] = 0;
        }
    }
    const int share = (kBins + w.splits - 1) / w.splits, b1 = min(kBins, (split + 1) * share);
    for (int b = split * share + tid; b < b1; b += 256) {
        w.sum[(size_t)row * kBins + b] = 0;
        w.count[(size_t)row * kBins + b] = 0;
    }
}

// The whole row's range; whole waves call this.
__device__ __forceinline__ RowRange row_range(const SampleWork &w, int row) {
    RowRange g{ -INFINITY, INFINITY, INT32_MAX, 0 };
    for (int s = (int)(threadIdx.x & 63); s < w.splits; s += 64) {
        const RowRange o = w.range[(size_t)row * w.splits + s];
        if (o.top > g.top) { g.top = o.top; g.arg = o.arg; }
        g.low = fminf(g.low, o.low);
    }
    fold_range(g);
    return g;
}

__global__ __launch_bounds__(kCountThreads) void sample_histogram_kernel(SampleArgs a, SampleWork w) {
    __shared__ unsigned long long sum[kBins];
    __shared__ uint32_t count[kBins];
    const int tid = threadIdx.x, split = blockIdx.x, row = blockIdx.y, r = w.row0 + row;
    const float *x = a.logits + (size_t)r * a.ld;
    const int i0 = split * w.per_count, n = max(0, min(a.vocab, i0 + w.per_count) - i0);
    float v[8];
    load_steps<8, kCountThreads>(x + i0, n, v);                           // on their way while the rest is looked up
    const RowAsks q = row_asks(a, r);
    if (q.greedy || !(q.k > 0 || q.p > 0.f)) return;                      // no cut to find
    const RowRange g = row_range(w, row);
    if (g.top == -INFINITY || g.top == INFINITY) return;                  // without weights
    const bool weighs = q.p > 0.f && !q.few;                              // top-k alone counts
    const RowBins b = row_bins(g.top, g.low, q.T, a.frac_bits);
    for (int i = tid; i < kBins; i += kCountThreads) {
        sum[i] = 0;
        count[i] = 0;
    }
    __syncthreads();
    for (int i = 0; i < n; i += 8 * kCountThreads) {
        float next[8];
        load_steps<8, kCountThreads>(x + i0 + i + 8 * kCountThreads, n - i - 8 * kCountThreads, next);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int bin = bin_of(b, v[j]);
            if (bin < kBins) {
                if (weighs) __hip_atomic_fetch_add(&sum[bin], whole(token_weight(b, v[j])), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                __hip_atomic_fetch_add(&count[bin], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            }
            v[j] = next[j];
        }
    }
    __syncthreads();
    for (int i = tid; i < kBins; i += kCountThreads) {      // a wave has the 64 bins of one coarse bin
        const uint32_t n = count[i];
        const unsigned long long s = weighs ? sum[i] : 0;
        const uint32_t n64 = (uint32_t)wave_sum_u64(n);
        if (n64 == 0) continue;
        const unsigned long long s64 = weighs ? wave_sum_u64(s) : 0;
        if (n) {
            __hip_atomic_fetch_add(&w.count[(size_t)row * kBins + i], n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (weighs) __hip_atomic_fetch_add(&w.sum[(size_t)row * kBins + i], s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        if ((tid & 63) == 0) {
            __hip_atomic_fetch_add(&w.coarse_count[(size_t)row * kCoarse + i / 64], n64, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (weighs) __hip_atomic_fetch_add(&w.coarse_sum[(size_t)row * kCoarse + i / 64], s64, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
}

// A token's place in the order: ascending keys are descending logits, ascending indexes among equals.
__device__ __forceinline__ unsigned long long rank_key(float x, int i) { return ((unsigned long long)(uint32_t)~logit_order(x) << 32) | (uint32_t)i; }

// Exclusive running sum over the workgroup's threads; red holds one value per wave, total the sum of all.
__device__ __forceinline__ unsigned long long block_scan_u64(unsigned long long v, unsigned long long *red, unsigned long long &total) {
    const int lane = (int)(threadIdx.x & 63), wave = (int)(threadIdx.x >> 6);
    const unsigned long long s = wave_scan_u64(v);
    __syncthreads();
    if (lane == 63) red[wave] = s;
    __syncthreads();
    unsigned long long before = 0;
    total = 0;
    for (int i = 0; i < (int)(blockDim.x >> 6); i++) {
        if (i == wave) before = total;
        total += red[i];
    }
    return before + s - v;
}

// Which of a wave's 64 pieces it is in which a running sum reaches a goal, by `reaches(before, with)`; 63 if it says so of none.
template <class F>
__device__ __forceinline__ int find_piece(unsigned long long before, unsigned long long with, F reaches) {
    const unsigned long long is = __ballot(reaches(before, with));
    return __builtin_amdgcn_readfirstlane(is ? __ffsll(is) - 1 : 63);
}

// The cuts' bins, from the row's histogram: of the coarse bins the one, then of its 64 bins the one.  One wave calls this; two reads
// that wait for one another behind the coarse bins, one where only one cut is asked for.
__device__ RowBorders find_borders(const unsigned long long *sum, const uint32_t *count, const unsigned long long *coarse_sum, const uint32_t *coarse_count,
                                   const RowAsks &q) {
    const int lane = (int)(threadIdx.x & 63);
    const bool weighed = q.p > 0.f && !q.few;
    const unsigned long long sums = weighed ? coarse_sum[lane] : 0, counts = coarse_count[lane];
    const unsigned long long sum_to = wave_scan_u64(sums), count_to = wave_scan_u64(counts), all = lane_u64(sum_to, 63), tokens = lane_u64(count_to, 63);
    RowBorders o{ all, all, all, 0, 0, q.k > 0 && (unsigned long long)q.k < tokens ? (unsigned long long)q.k : (q.few ? tokens : 0), 0, kBins, 0, -1, kBins };
    if (o.k) {
        const auto holds_k = [k = o.k](unsigned long long from, unsigned long long to) { return from < k && k <= to; };
        const int c = find_piece(count_to - counts, count_to, holds_k);
        const unsigned long long n = count[c * 64 + lane], s = weighed ? sum[c * 64 + lane] : 0;
        const unsigned long long n_to = lane_u64(count_to - counts, c) + wave_scan_u64(n), s_to = lane_u64(sum_to - sums, c) + wave_scan_u64(s);
        const int l = find_piece(n_to - n, n_to, holds_k);
        o.k_bin = c * 64 + l;
        o.k_above = lane_u64(n_to - n, l);
        o.k_in = lane_u64(n, l);
        o.k_weight_above = lane_u64(s_to - s, l);
        o.k_weight_with = lane_u64(s_to, l);
    }
    o.keep_below = o.k_bin;
    if (q.few) {                                            // the list holds every token down to the last of the top k
        o.k_in += o.k_above;
        o.k_above = 0;
        o.p_last = o.k_bin;
        o.keep_below = 0;
    } else if (q.p > 0.f) {
        // the weight of the top k lies between that of the bins above its last one and that with it; nothing above: from bin 0 on
        const double lo = (double)q.p * (double)o.k_weight_above, hi = (double)q.p * (double)o.k_weight_with;
        const auto reaches_lo = [lo](unsigned long long from, unsigned long long to) { return (double)from < lo && lo <= (double)to; };
        const auto reaches_hi = [hi](unsigned long long from, unsigned long long to) { return (double)from < hi && hi <= (double)to; };
        const int cl = find_piece(sum_to - sums, sum_to, reaches_lo), ch = find_piece(sum_to - sums, sum_to, reaches_hi);
        const unsigned long long a = sum[cl * 64 + lane], b = sum[ch * 64 + lane];
        const unsigned long long a_to = lane_u64(sum_to - sums, cl) + wave_scan_u64(a), b_to = lane_u64(sum_to - sums, ch) + wave_scan_u64(b);
        if (lo > 0.0) {
            const int l = find_piece(a_to - a, a_to, reaches_lo);
            o.p_first = cl * 64 + l;
            o.above_list = lane_u64(a_to - a, l);
        }
        o.p_last = ch * 64 + find_piece(b_to - b, b_to, reaches_hi);
        o.keep_below = o.p_first;
    }
    return o;
}

// The same borders as a token's place among the bins meets them.
struct Wanted {
    float keep, p0, p1, k0, k1;
    __device__ explicit Wanted(const RowBorders &c)
        : keep((float)c.keep_below), p0((float)c.p_first), p1((float)(c.p_last + 1)), k0((float)c.k_bin), k1(c.k_bin < kBins ? (float)(c.k_bin + 1) : 0.f) {}
    __device__ bool kept(float at) const { return at < keep; }
    __device__ bool listed(float at) const { return (at >= p0 && at < p1) || (at >= k0 && at < k1); }
};

// Lists the tokens of the cuts' bins and sums the weights of the tokens above them, kPart tokens at a time; a workgroup has
// parts_each such parts of a row.  Finding the borders takes a workgroup longer than a part does: 77 rows of 131071 with top-k 40 and
// top-p 0.95 take 59.5 us in all with one part each, 49.8 us with two (1024 workgroups), 51.5 with four, 61.5 with nine.
__global__ __launch_bounds__(kThreads) void sample_collect_kernel(SampleArgs a, SampleWork w) {
    __shared__ unsigned long long found[kListMost], red[kThreads / 64];
    __shared__ RowBorders borders;
    __shared__ int n_found, place;
    const int tid = threadIdx.x, row = blockIdx.y, r = w.row0 + row, first = (int)blockIdx.x * w.parts_each, last = min(w.parts, first + w.parts_each);
    const float *x = a.logits + (size_t)r * a.ld + (size_t)first * kPart;
    const int n_tokens = min(a.vocab, last * kPart) - first * kPart;
    float v[8], next[8];
    load_steps<8, kThreads>(x, n_tokens, v);                // on their way while the borders are looked for
    const RowAsks q = row_asks(a, r);
    if (q.greedy) return;
    const RowRange g = row_range(w, row);
    if (g.top == -INFINITY || g.top == INFINITY) return;
    const RowBins b = row_bins(g.top, g.low, q.T, a.frac_bits);
    if (tid < 64) {
        const RowBorders o = q.k > 0 || q.p > 0.f ? find_borders(w.sum + (size_t)row * kBins, w.count + (size_t)row * kBins, w.coarse_sum + (size_t)row * kCoarse,
                                                                 w.coarse_count + (size_t)row * kCoarse, q)
                                                  : kNoBorders;
        if (tid == 0) {
            borders = o;
            n_found = 0;
        }
    }
    __syncthreads();
    if (first == 0 && tid == 0) w.borders[row] = borders;
    const Wanted want(borders);
    const double min_w = ldexp(q.min_w, a.frac_bits);
    unsigned long long mine = 0;
#pragma unroll 1
    for (int h = 0; h < n_tokens; h += 8 * kThreads) {
        load_steps<8, kThreads>(x + h + 8 * kThreads, n_tokens - h - 8 * kThreads, next);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float at = bin_at(b, v[j]);
            if (want.kept(at)) {
                const double f = token_weight(b, v[j]);
                if (f >= min_w) mine += whole(f);
            } else if (want.listed(at)) {
                const int place = __hip_atomic_fetch_add(&n_found, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                if (place < kListMost) found[place] = rank_key(v[j], first * kPart + h + tid + j * kThreads);
            }
            v[j] = next[j];
        }
        if ((h / (8 * kThreads)) % (kPart / (8 * kThreads)) == kPart / (8 * kThreads) - 1 || h + 8 * kThreads >= n_tokens) {      // the end of a part
            mine = want.keep > 0.f ? block_sum_u64(mine, red) : 0;
            if (tid == 0) w.part_sum[(size_t)row * w.parts + first + h / kPart] = mine;
            mine = 0;
        }
    }
    __syncthreads();
    if (tid == 0) place = n_found ? __hip_atomic_fetch_add(&w.listed[row], n_found, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
    __syncthreads();
    const int at = place, n = min(n_found, kListMost);      // more than the list holds: the count says so
    for (int i = tid; i < n; i += kThreads)
        if (at + i < kListMost) w.list[(size_t)row * kListMost + at + i] = found[i];
}

// The row on its own, without bins: the cuts by bisection over the 32 bits of the logits' order, one pass over the row per bit.
// For rows with infinite logits and for rows with more equal or nearly equal logits in the cuts' bins than the list of
// finish_row holds: right, and slow (one row of 32000 equal logits with top-p 180 us; 128256 that were once bf16, so flat that thousands
// share a bin, 6 ms where 40 us are usual).  run: kThreads entries, tie as many.
template <int kThreads>
__device__ void sample_by_bisection(const SampleArgs &a, int r, const RowAsks &q, float top, unsigned long long *run, int *tie, unsigned long long *red) {
    const int tid = threadIdx.x, V = a.vocab, k = q.k > 0 ? q.k : V;
    const float *x = a.logits + (size_t)r * a.ld;
    const uint32_t top_order = logit_order(top);
    const float p_keep = q.p;
    const double T = q.T, min_w = q.min_w;

    // ---- the cut: tokens above `cut` stay, of those at `cut` the first `ties` by index
    auto count_from = [&](uint32_t o) {              // tokens at o or above
        unsigned long long n = 0;
        for (int i = tid; i < V; i += kThreads) n += logit_order(x[i]) >= o ? 1 : 0;
        return block_sum_u64(n, red);
    };
    auto weight_from = [&](uint32_t o) {
        unsigned long long n = 0;
        for (int i = tid; i < V; i += kThreads)
            if (logit_order(x[i]) >= o) n += fixed_weight(x[i], top, T, a.frac_bits);
        return block_sum_u64(n, red);
    };
    uint32_t cut = logit_order(-INFINITY) + 1;
    unsigned long long ties = (unsigned long long)V;
    {
        uint32_t c = 0;                              // the largest order that at least k tokens reach
        for (int bit = 31; bit >= 0; bit--) {
            const uint32_t want = c | (1u << bit);
            if (want <= top_order && count_from(want) >= (unsigned long long)k) c = want;
        }
        if (c >= cut) {
            cut = c;
            ties = (unsigned long long)k - (c == 0xFFFFFFFFu ? 0 : count_from(c + 1));
        }
    }
    auto kept_weight = [&](uint32_t o) {             // of the tokens at o or above, o >= cut, those that the cut keeps
        if (o > cut) return weight_from(o);
        return weight_from(cut + 1) + ties * fixed_weight(order_logit(cut), top, T, a.frac_bits);
    };
    if (p_keep > 0.f && p_keep < 1.f) {
        // ties may be V (no top-k): the weight of a cut that no token sits at is not counted
        const unsigned long long at_cut = count_from(cut) - count_from(cut + 1);
        if (ties > at_cut) ties = at_cut;
        const double goal = (double)p_keep * (double)kept_weight(cut);
        uint32_t c = 0;                              // the largest order from which the kept weight reaches the goal
        for (int bit = 31; bit >= 0; bit--) {
            const uint32_t want = c | (1u << bit);
            if (want <= top_order && (want <= cut || (double)kept_weight(want) >= goal)) c = want;
        }
        if (c < cut) c = cut;
        const unsigned long long above = c >= top_order ? 0 : weight_from(c + 1), each = fixed_weight(order_logit(c), top, T, a.frac_bits);
        // equal tokens go in one by one until the goal is reached
        unsigned long long lo = 1, hi = c > cut ? count_from(c) - count_from(c + 1) : ties;
        while (lo < hi) {
            const unsigned long long mid = (lo + hi) / 2;
            if ((double)(above + mid * each) >= goal) hi = mid;
            else lo = mid + 1;
        }
        cut = c;
        ties = lo;
    }

    // ---- the draw, by index: each thread owns consecutive tokens
    const int per = (V + kThreads - 1) / kThreads, i0 = min(V, tid * per), i1 = min(V, i0 + per);
    int mine = 0;
    for (int i = i0; i < i1; i++) mine += logit_order(x[i]) == cut ? 1 : 0;
    tie[tid] = mine;
    __syncthreads();
    unsigned long long seen = 0;
    for (int j = 0; j < tid; j++) seen += (unsigned long long)tie[j];
    const unsigned long long seen0 = seen;
    auto weight_at = [&](int i) -> unsigned long long {        // in ascending order of i: counts the ties
        const uint32_t o = logit_order(x[i]);
        if (o < cut || (o == cut && seen++ >= ties)) return 0;
        if (weight_of(x[i], top, T) < min_w) return 0;
        return fixed_weight(x[i], top, T, a.frac_bits);
    };
    unsigned long long sum = 0;
    for (int i = i0; i < i1; i++) sum += weight_at(i);
    run[tid] = sum;
    __syncthreads();
    unsigned long long total = 0, before = 0;
    for (int j = 0; j < kThreads; j++) {
        if (j == tid) before = total;
        total += run[j];
    }
    const double u = fmin(fmax(a.u[r], 0.0), 1.0);
    // first token with (running weight) > u * total; for u that rounds up to the total, the last one that weighs anything
    unsigned long long goal = (unsigned long long)floor(u * (double)total);
    if (goal >= total) goal = total - 1;
    if (before <= goal && goal < before + sum) {
        seen = seen0;
        unsigned long long at = before;
        for (int i = i0; i < i1; i++) {
            const unsigned long long w = weight_at(i);
            if (w && goal < at + w) {
                a.out_token[r] = i;
                if (a.out_prob) a.out_prob[r] = (float)(ldexp(weight_of(x[i], top, T), a.frac_bits) / (double)total);
                break;
            }
            at += w;
        }
    }
}

// The end of a row: ranks the listed tokens, finds the last one that stays, draws.  buf: kPart entries, the list's keys in the
// first n_list; parts: the weight that stays whole of each kPart tokens, n_parts <= kThreads of them.  The whole workgroup calls this.
// Loops stay loops here and below: this code runs once per row, and straight-line code of tens of kilobytes is paid for in
// instruction fetches (one row of 1000 tokens, no filter: 13.4 us with 82 KB of code, 8.2 us with 34 KB).
template <int kThreads>
__device__ __forceinline__ void finish_row(const SampleArgs &a, int r, const RowAsks &q, const RowBins &b, const RowBorders &c, int n_list, unsigned long long *buf,
                                           unsigned long long *parts, int n_parts, unsigned long long *red) {
    constexpr int kOwn = kPart / kThreads;
    __shared__ unsigned long long found_cut, before_chosen;
    __shared__ int chosen;
    static_assert(2 * kListMost <= kPart && kListMost >= 2 * kCountSort && kThreads >= kCountSort, "what buf is used for");
    unsigned long long *upto = buf + kListMost;             // running weight of the sorted list, each token's own included
    const int tid = threadIdx.x, V = a.vocab;
    const float *x = a.logits + (size_t)r * a.ld;
    const double min_w = ldexp(q.min_w, a.frac_bits);

    // ---- the last key that stays
    unsigned long long cut = ~0ull;
    if (n_list > 0) {
        if (n_list <= kCountSort) {          // sorted by counting the keys before each
            const unsigned long long mine = tid < n_list ? buf[tid] : 0;
            int rank = 0;
#pragma unroll 4
            for (int j = 0; j < n_list; j++) rank += buf[j] < mine ? 1 : 0;
            __syncthreads();
            if (tid < n_list) buf[rank] = mine;
            __syncthreads();
        } else {                             // bitonic sort: log2(span) * (log2(span) + 1) / 2 steps of span / 2 exchanges
            int span = 2 * kCountSort;
            while (span < n_list) span <<= 1;
            for (int i = n_list + tid; i < span; i += kThreads) buf[i] = ~0ull;
            __syncthreads();
            for (int size = 2; size <= span; size <<= 1)
                for (int stride = size >> 1; stride > 0; stride >>= 1) {
                    for (int t = tid; t < span / 2; t += kThreads) {
                        const int i = 2 * t - (t & (stride - 1)), o = i + stride;
                        const unsigned long long x0 = buf[i], x1 = buf[o];
                        if ((x0 > x1) == ((i & size) == 0)) {
                            buf[i] = x1;
                            buf[o] = x0;
                        }
                    }
                    // a wave's exchanges of stride 64 and less lie in 128 keys of its own
                    if (stride > 64 || (stride == 1 && size > 64)) __syncthreads();
                    else wave_lds_fence();
                }
            __syncthreads();
        }
        unsigned long long run = 0;
#pragma unroll 1
        for (int i0 = 0; i0 < n_list; i0 += kThreads) {
            const int i = i0 + tid;
            const unsigned long long weight = i < n_list ? whole(token_weight(b, order_logit(~(uint32_t)(buf[i] >> 32)))) : 0;
            unsigned long long sum;
            const unsigned long long before = run + block_scan_u64(weight, red, sum);
            if (i < n_list) upto[i] = before + weight;
            run += sum;
        }
        __syncthreads();
        // the listed bins are top-p's, one after the other, and top-k's, which is the last of them or comes behind them
        double goal = (double)q.p * (double)c.all;
        int stay = n_list;
        if (c.k) {
            const int k_from = n_list - (int)c.k_in;        // the list's part in the bin of top-k
            stay = k_from + (int)(c.k - c.k_above);
            cut = buf[stay - 1];
            goal = (double)q.p * (double)(c.k_weight_above + upto[stay - 1] - (k_from > 0 ? upto[k_from - 1] : 0));
        }
        if (q.p > 0.f) {
            // the first token at which the weight reaches the goal; it is one of the listed, and not behind top-k's last
#pragma unroll 1
            for (int i = tid; i < stay; i += kThreads) {
                const unsigned long long before = c.above_list + (i > 0 ? upto[i - 1] : 0);
                if ((double)before < goal && (double)(c.above_list + upto[i]) >= goal) found_cut = buf[i];
            }
            __syncthreads();
            cut = found_cut;
        }
        // what stays of the listed tokens joins the parts' sums
#pragma unroll 1
        for (int i = tid; i < n_list; i += kThreads) {
            const unsigned long long key = buf[i];
            const double f = token_weight(b, order_logit(~(uint32_t)(key >> 32)));
            if (key <= cut && f >= min_w) __hip_atomic_fetch_add(&parts[(uint32_t)key / kPart], whole(f), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        }
    }
    __syncthreads();                                        // the list's memory is free from here on

    // ---- the draw, by index, over the tokens whose key is at most the cut: which part, then which token of it
    unsigned long long total;
    const unsigned long long part = tid < n_parts ? parts[tid] : 0, before_part = block_scan_u64(part, red, total);
    const double u = fmin(fmax(a.u[r], 0.0), 1.0);          // NaN: 0
    unsigned long long goal = (unsigned long long)floor(u * (double)total);      // the first token with (running weight) > goal
    if (goal >= total) goal = total - 1;
    if (part && before_part <= goal && goal < before_part + part) {
        chosen = tid;
        before_chosen = before_part;
    }
    __syncthreads();
    const int i0 = chosen * kPart;
#pragma unroll 4
    for (int j = 0; j < kOwn; j++) {
        const int i = i0 + j * kThreads + tid;
        const float v = i < V ? x[i] : NAN;
        const int bin = bin_of(b, v);
        unsigned long long weight = 0;
        if (bin < kBins && rank_key(v, i) <= cut) {
            const double f = token_weight(b, v);
            if (f >= min_w) weight = whole(f);
        }
        buf[j * kThreads + tid] = weight;
    }
    __syncthreads();
    // a thread per kOwn consecutive tokens
    unsigned long long mine = 0, sum;
    for (int j = 0; j < kOwn; j++) mine += buf[tid * kOwn + j];
    unsigned long long at = before_chosen + block_scan_u64(mine, red, sum);
    if (mine && at <= goal && goal < at + mine)
#pragma unroll 1
        for (int j = 0; j < kOwn; j++) {
            const unsigned long long weight = buf[tid * kOwn + j];
            if (weight && goal < at + weight) {
                const int i = i0 + tid * kOwn + j;
                a.out_token[r] = i;
                if (a.out_prob) a.out_prob[r] = (float)(token_weight(b, x[i]) / (double)total);
                break;
            }
            at += weight;
        }
}

__global__ __launch_bounds__(kThreads) void sample_finish_kernel(SampleArgs a, SampleWork w) {
    __shared__ unsigned long long buf[kPart], parts[kThreads], red[kThreads / 64];
    const int tid = threadIdx.x, row = blockIdx.x, r = w.row0 + row;
    const unsigned long long part = tid < w.parts ? w.part_sum[(size_t)row * w.parts + tid] : 0;      // at most kThreads parts
    const RowAsks q = row_asks(a, r);
    const RowRange g = row_range(w, row);
    const int n_list = w.listed[row];
    if (undrawn_row(a, r, q, g)) return;
    if (g.top == INFINITY || n_list > kListMost) {
        sample_by_bisection<kThreads>(a, r, q, g.top, buf, reinterpret_cast<int *>(buf + kThreads), red);
        return;
    }
    const RowBorders c = w.borders[row];
    parts[tid] = part;
    for (int i = tid; i < n_list; i += kThreads) buf[i] = w.list[(size_t)row * kListMost + i];
    __syncthreads();
    finish_row<kThreads>(a, r, q, row_bins(g.top, g.low, q.T, a.frac_bits), c, n_list, buf, parts, w.parts, red);
}

// ---- the whole of it by one workgroup per row, in one launch: the row is read three times, the last two from the L2.
constexpr int kRowThreads = 1024, kStep = 8;
__global__ __launch_bounds__(kRowThreads) void sample_row_kernel(SampleArgs a) {
    __shared__ unsigned long long sum[kBins], coarse_sum[kCoarse], parts[kThreads + kStep / 4], red[kRowThreads / 64];
    __shared__ uint32_t count[kBins], coarse_count[kCoarse];
    __shared__ RowBorders borders;
    __shared__ float tops[kRowThreads / 64], lows[kRowThreads / 64];
    __shared__ int args[kRowThreads / 64], n_found;
    static_assert(kBins >= kPart && kPart == 4 * kRowThreads, "the list takes the histogram's place; four steps are a part");
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = blockIdx.x, n_parts = (a.vocab + kPart - 1) / kPart;
    const float *x = a.logits + (size_t)r * a.ld;
    const RowAsks q = row_asks(a, r);
    for (int i = tid; i < kBins; i += kRowThreads) {
        sum[i] = 0;
        count[i] = 0;
    }
    if (tid < kThreads) parts[tid] = 0;
    if (tid == 0) n_found = 0;
    RowRange g{ -INFINITY, INFINITY, INT32_MAX, 0 };
    float v[kStep], next[kStep];             // the next step's values are on their way while a step's are used
    load_steps<kStep, kRowThreads>(x, a.vocab, v);
#pragma unroll 1
    for (int i0 = 0; i0 < a.vocab; i0 += kStep * kRowThreads) {
        load_steps<kStep, kRowThreads>(x + i0 + kStep * kRowThreads, a.vocab - i0 - kStep * kRowThreads, next);
#pragma unroll
        for (int j = 0; j < kStep; j++) {
            g.top = fmaxf(g.top, v[j]);                          // NaN: neither
            g.low = fminf(g.low, v[j]);
            v[j] = next[j];
        }
    }
    load_steps<kStep, kRowThreads>(x, a.vocab, v);
    g.top = wave_top(g.top);
    g.low = wave_low(g.low);
    if (lane == 0) { tops[wave] = g.top; lows[wave] = g.low; }
    __syncthreads();
    g.top = wave_top(lane < kRowThreads / 64 ? tops[lane] : -INFINITY);
    g.low = wave_low(lane < kRowThreads / 64 ? lows[lane] : INFINITY);
    if (q.greedy) {
        g.arg = wave_low(first_of<kRowThreads>(x, a.vocab, 0, g.top));
        if (lane == 0) args[wave] = g.arg;
        __syncthreads();
        g.arg = wave_low(lane < kRowThreads / 64 ? args[lane] : INT32_MAX);
    }
    if (undrawn_row(a, r, q, g)) return;
    int n_list = g.top == INFINITY ? kListMost + 1 : 0;
    if (n_list == 0) {
        const RowBins b = row_bins(g.top, g.low, q.T, a.frac_bits);
        const bool cuts = q.k > 0 || q.p > 0.f, weighs = q.p > 0.f && !q.few;
        if (cuts) {
#pragma unroll 1
            for (int i0 = 0; i0 < a.vocab; i0 += kStep * kRowThreads) {
                load_steps<kStep, kRowThreads>(x + i0 + kStep * kRowThreads, a.vocab - i0 - kStep * kRowThreads, next);
#pragma unroll
                for (int j = 0; j < kStep; j++) {
                    const int bin = bin_of(b, v[j]);
                    if (bin < kBins) {
                        if (weighs) __hip_atomic_fetch_add(&sum[bin], whole(token_weight(b, v[j])), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                        __hip_atomic_fetch_add(&count[bin], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                    }
                    v[j] = next[j];
                }
            }
            load_steps<kStep, kRowThreads>(x, a.vocab, v);
            __syncthreads();
#pragma unroll 1
            for (int i = tid; i < kBins; i += kRowThreads) {              // a wave has the 64 bins of one coarse bin
                const unsigned long long n = wave_sum_u64(count[i]), s = weighs ? wave_sum_u64(sum[i]) : 0;
                if (lane == 0) {
                    coarse_count[i / 64] = (uint32_t)n;
                    coarse_sum[i / 64] = s;
                }
            }
            __syncthreads();
            if (wave == 0) {
                const RowBorders o = find_borders(sum, count, coarse_sum, coarse_count, q);
                if (lane == 0) borders = o;
            }
        } else if (tid == 0) {
            borders = kNoBorders;
        }
        __syncthreads();                                    // the histogram's memory takes the list from here on
        const RowBorders c = borders;
        const Wanted want(c);
        const double min_w = ldexp(q.min_w, a.frac_bits);
#pragma unroll 1
        for (int i0 = 0; i0 < a.vocab; i0 += kStep * kRowThreads) {
            load_steps<kStep, kRowThreads>(x + i0 + kStep * kRowThreads, a.vocab - i0 - kStep * kRowThreads, next);
            unsigned long long mine = 0;
#pragma unroll
            for (int j = 0; j < kStep; j++) {
                const float at = bin_at(b, v[j]);
                if (want.kept(at)) {
                    const double f = token_weight(b, v[j]);
                    if (f >= min_w) mine += whole(f);
                } else if (want.listed(at)) {
                    const int place = __hip_atomic_fetch_add(&n_found, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                    if (place < kListMost) sum[place] = rank_key(v[j], i0 + tid + j * kRowThreads);
                }
                v[j] = next[j];
                if (c.keep_below > 0 && j % 4 == 3) {       // the end of a part
                    mine = wave_sum_u64(mine);
                    if (lane == 0 && mine) __hip_atomic_fetch_add(&parts[i0 / kPart + j / 4], mine, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                    mine = 0;
                }
            }
        }
        __syncthreads();
        n_list = n_found;
        if (n_list <= kListMost) {
            finish_row<kRowThreads>(a, r, q, b, c, n_list, sum, parts, n_parts, red);
            return;
        }
    }
    sample_by_bisection<kRowThreads>(a, r, q, g.top, sum, reinterpret_cast<int *>(count), red);
}

}  // namespace
}  // namespace rt

using rt::fail;
using rt::Guard;
using rt::ensure_scratch;

extern "C" {

int rt_hip_sample_dev(rt_hip_ctx *ctx, const float *logits, size_t ld, int n_rows, int vocab, const float *temperature, const int *top_k, const float *top_p,
                      const float *min_p, const double *u, int *out_token, float *out_prob) {
    if (!ctx) return fail(nullptr, RT_HIP_ERR_INVALID_ARG, "ctx is NULL");
    RT_REQUIRE(ctx, logits && u && out_token, RT_HIP_ERR_INVALID_ARG, "sample: NULL argument");
    RT_REQUIRE(ctx, n_rows >= 0 && n_rows <= 65535, RT_HIP_ERR_SHAPE, "sample: n_rows=%d outside 0..65535", n_rows);
    RT_REQUIRE(ctx, vocab >= 1 && vocab <= (1 << 20), RT_HIP_ERR_SHAPE, "sample: vocab=%d outside 1..2^20", vocab);
    RT_REQUIRE(ctx, ld >= (size_t)vocab && ld <= rt::kRowsApartMost, RT_HIP_ERR_SHAPE, "sample: rows are %zu floats apart, vocab=%d", ld, vocab);
    if (n_rows == 0) return RT_HIP_OK;
    Guard g(ctx);
    int bits = 0;
    while ((1 << bits) < vocab) bits++;
    rt::SampleArgs a{ logits, ld, n_rows, vocab, bits < 11 ? 51 : 62 - bits, u, temperature, top_p, min_p, top_k, out_token, out_prob };
    // One workgroup per row, or rows split over the device in four launches (us; top-k 40 and top-p 0.95 / top-p 0.9 / no filter):
    //   rows x vocab    1 x 32000   64 x 32000  256 x 32000  64 x 65536  77 x 131071  1 x 131071
    //   one launch      23/42/23    24/44/24    28/47/27     34/73/39    59/135/73    50/127/65
    //   four            26/31/21    40/55/27    55/78/42     39/53/30    50/78/43     30/36/20
    // The rule looks at the vocabulary alone.  Up to 32768 tokens one launch is the faster from 64 rows on and needs no workspace; it costs a
    // single row up to 11 us with top-p alone.  Above, four are the faster but for a small top-k, which loses up to 5 us at 64 rows.
    if (vocab <= 32768) {
        rt::sample_row_kernel<<<dim3((unsigned)n_rows), rt::kRowThreads, 0, ctx->stream>>>(a);
        RT_TRY_HIP(ctx, hipGetLastError());
        return RT_HIP_OK;
    }
    // A row is split so that about a thousand workgroups look for the ranges (2048 tokens at least in each) and as many as there are
    // compute units count (4096 tokens at least): every one of the latter adds up to 4096 bins to the row's histogram.  77 rows
    // of 131071 with 256, 512 and 1024 workgroups: top-p 0.9 78, 88 and 105 us, top-k 40 and top-p 0.95 50, 56 and 69.  Rows go in groups whose histograms stay below 64 MB.
    const int group = std::min(n_rows, 1024);
    rt::SampleWork w;
    w.splits = std::max(1, std::min(1024 / group, (vocab + 2047) / 2048));
    const int count_splits = std::max(1, std::min(256 / group, (vocab + 4095) / 4096));
    w.per_split = (vocab + w.splits - 1) / w.splits;
    w.per_count = (vocab + count_splits - 1) / count_splits;
    w.parts = (vocab + rt::kPart - 1) / rt::kPart;
    w.parts_each = std::max(1, std::min(w.parts, w.parts * group / 1024));
    const size_t coarse = (size_t)group * rt::kCoarse, bins = (size_t)group * rt::kBins, list = (size_t)group * rt::kListMost, parts = (size_t)group * w.parts;
    int rc = ensure_scratch(ctx, (bins + list + parts + coarse) * 8 + group * sizeof(rt::RowBorders) + (size_t)group * w.splits * sizeof(rt::RowRange) +
                                 (bins + coarse + group) * 4);
    if (rc) return rc;
    w.sum = static_cast<unsigned long long *>(ctx->scratch);
    w.list = w.sum + bins;
    w.part_sum = w.list + list;
    w.coarse_sum = w.part_sum + parts;
    w.borders = reinterpret_cast<rt::RowBorders *>(w.coarse_sum + coarse);
    w.range = reinterpret_cast<rt::RowRange *>(w.borders + group);
    w.count = reinterpret_cast<uint32_t *>(w.range + (size_t)group * w.splits);
    w.coarse_count = w.count + bins;
    w.listed = reinterpret_cast<int *>(w.coarse_count + coarse);
    for (w.row0 = 0; w.row0 < n_rows; w.row0 += group) {
        const int rows = std::min(group, n_rows - w.row0);
        const dim3 grid((unsigned)w.splits, (unsigned)rows);
        rt::sample_range_kernel<<<grid, rt::kThreads, 0, ctx->stream>>>(a, w);
        rt::sample_histogram_kernel<<<dim3((unsigned)count_splits, (unsigned)rows), rt::kCountThreads, 0, ctx->stream>>>(a, w);
        rt::sample_collect_kernel<<<dim3((unsigned)((w.parts + w.parts_each - 1) / w.parts_each), (unsigned)rows), rt::kThreads, 0, ctx->stream>>>(a, w);
        rt::sample_finish_kernel<<<dim3((unsigned)rows), rt::kThreads, 0, ctx->stream>>>(a, w);
    }
    RT_TRY_HIP(ctx, hipGetLastError());
    return RT_HIP_OK;
}

}  // extern "C"
