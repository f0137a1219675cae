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
#include "rt_device.h"

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

__device__ __forceinline__ unsigned long long wave_sum_u64(unsigned long long v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint32_t lo = (uint32_t)__shfl_xor((int)(uint32_t)v, o), hi = (uint32_t)__shfl_xor((int)(uint32_t)(v >> 32), o);
        v += ((unsigned long long)hi << 32) | lo;
    }
    return v;
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

constexpr int kSampleThreads = 1024;

// One workgroup per row.  The cuts are found by bisection over the 32 bits of the logits' order, one pass over the row per bit.
__global__ __launch_bounds__(kSampleThreads) void sample_kernel(SampleArgs a) {
    __shared__ unsigned long long red[kSampleThreads / 64];
    __shared__ unsigned long long run[kSampleThreads];
    __shared__ int tie[kSampleThreads];
    __shared__ float redf[kSampleThreads / 64];
    const int tid = threadIdx.x, r = blockIdx.x, V = a.vocab;
    const float *x = a.logits + (size_t)r * a.ld;

    float top = -INFINITY;
    for (int i = tid; i < V; i += kSampleThreads) top = fmaxf(top, x[i] != x[i] ? -INFINITY : x[i]);
    top = block_max(top, redf);
    const uint32_t top_order = logit_order(top);
    if (top == -INFINITY) {                          // nothing to draw from
        if (tid == 0) {
            a.out_token[r] = -1;
            if (a.out_prob) a.out_prob[r] = 0.f;
        }
        return;
    }
    const float tf = a.temperature ? a.temperature[r] : 1.0f, p_keep = a.top_p ? a.top_p[r] : 0.f, low = a.min_p ? a.min_p[r] : 0.f;
    int k = a.top_k ? a.top_k[r] : 0;
    if (!(tf > 0.f)) k = 1;                          // temperature 0: the largest, the lowest index among equals
    if (k <= 0 || k > V) k = V;
    const double T = k == 1 ? 1.0 : (double)tf, min_w = low > 0.f ? fmin((double)low, 1.0) : 0.0;

    // ---- the cut: tokens above `cut` stay, of those at `cut` the first `ties` by index
    auto count_from = [&](uint32_t o) {              // tokens at o or above
        unsigned long long n = 0;
        for (int i = tid; i < V; i += kSampleThreads) n += logit_order(x[i]) >= o ? 1 : 0;
        return block_sum_u64(n, red);
    };
    auto weight_from = [&](uint32_t o) {
        unsigned long long n = 0;
        for (int i = tid; i < V; i += kSampleThreads)
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
    const int per = (V + kSampleThreads - 1) / kSampleThreads, i0 = min(V, tid * per), i1 = min(V, i0 + per);
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
    for (int j = 0; j < kSampleThreads; j++) {
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

}  // namespace
}  // namespace rt

using rt::fail;
using rt::Guard;

extern "C" {

int rt_hip_sample_dev(rt_hip_ctx *ctx, const float *logits, size_t ld, int n_rows, int vocab, const float *temperature, const int *top_k, const float *top_p,
                      const float *min_p, const double *u, int *out_token, float *out_prob) {
    if (!ctx) return fail(nullptr, RT_HIP_ERR_INVALID_ARG, "ctx is NULL");
    RT_REQUIRE(ctx, logits && u && out_token, RT_HIP_ERR_INVALID_ARG, "sample: NULL argument");
    RT_REQUIRE(ctx, n_rows >= 0 && n_rows <= 65535, RT_HIP_ERR_SHAPE, "sample: n_rows=%d outside 0..65535", n_rows);
    RT_REQUIRE(ctx, vocab >= 1 && vocab <= (1 << 20), RT_HIP_ERR_SHAPE, "sample: vocab=%d outside 1..2^20", vocab);
    RT_REQUIRE(ctx, ld >= (size_t)vocab, RT_HIP_ERR_SHAPE, "sample: rows are %zu floats apart, vocab=%d", ld, vocab);
    if (n_rows == 0) return RT_HIP_OK;
    Guard g(ctx);
    int bits = 0;
    while ((1 << bits) < vocab) bits++;
    rt::SampleArgs a{ logits, ld, n_rows, vocab, bits < 10 ? 52 : 62 - bits, u, temperature, top_p, min_p, top_k, out_token, out_prob };
    rt::sample_kernel<<<dim3((unsigned)n_rows), rt::kSampleThreads, 0, ctx->stream>>>(a);
    RT_TRY_HIP(ctx, hipGetLastError());
    return RT_HIP_OK;
}

}  // extern "C"
