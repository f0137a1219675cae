// What the kernels over a cache in pages share: the view of a pool and its batch (rt_paged.hip says what they hold), and the
// place of a row among the sequences.
#pragma once

#include "rt_device.h"

namespace rt {

// What a launch knows of the pool and of the batch.
struct PagedView {
    uint16_t *k, *v;
    const int *table, *kv_len, *cu_new;      // cu_new == nullptr: row s is the one new token of sequence s
    int n_pages, page_shift, n_kv, n_seq, max_blocks;
};

// ------------------------------------------------------------------ which sequence and position a row belongs to
// Whole waves call this (the sequences are looked at 64 at a time).  The row's sequence is the number of ends
// cu_new[s + 1] <= t; false for a row that no sequence owns.
__device__ __forceinline__ bool row_place(const PagedView &p, int t, int &seq, long long &pos) {
    if (!p.cu_new) {
        seq = t;
        pos = (long long)p.kv_len[t] - 1;
        return true;
    }
    const int lane = (int)(threadIdx.x & 63);
    int before = 0;
    for (int s0 = 0; s0 < p.n_seq; s0 += 64) {
        const int s = s0 + lane;
        const unsigned long long ended = __ballot(s < p.n_seq && p.cu_new[s + 1] <= t);
        before += __popcll(ended);
        if (ended != ~0ull) break;
    }
    if (before >= p.n_seq) return false;
    const int a = p.cu_new[before], b = p.cu_new[before + 1];
    if (t < a || t >= b) return false;
    seq = before;
    pos = (long long)p.kv_len[before] - b + t;
    return true;
}

// ------------------------------------------------------------------ a query's element as the sum of two halves
// The scores' products run on fp16 matrix cores once for each half, so q has to be in them to f32's accuracy: the upper half is the
// scaled value cut towards zero, the lower what the cut left, rounded (2^-22 of the value is lost).  Both have q's sign and neither is
// zero unless q is: a key element of infinity then meets the same sign twice, and the score is that infinity.  Rounding the
// upper half to nearest would leave remainders of the other sign, and values that fit a half a remainder of zero; both make
// infinity minus infinity or 0 * infinity of a score that is -inf, and NaN of a whole row that is finite.  The least half that
// stands for a zero is 2^-37 of the row's largest element (which the scaling brings to 2^13 .. 2^14).
typedef _Float16 half8v __attribute__((ext_vector_type(8)));

// Eight elements that are not zero after the scaling, |q| * scale >= 2^-24: two at a time, three instructions a pair for the lower
// halves' signs and zeros.
__device__ __forceinline__ void split_queries(const float (&q)[8], float scale, half8v &hi, half8v &lo) {
    uint4 h, l;
    uint32_t *hp = &h.x, *lp = &l.x;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        typedef _Float16 half2v __attribute__((ext_vector_type(2)));
        typedef unsigned short ushort2v __attribute__((ext_vector_type(2)));
        const float v0 = q[2 * e] * scale, v1 = q[2 * e + 1] * scale;
        const half2v up = __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_pkrtz(v0, v1));
        const half2v low = { (_Float16)(v0 - (float)up[0]), (_Float16)(v1 - (float)up[1]) };
        const ushort2v size = __builtin_elementwise_max(__builtin_bit_cast(ushort2v, __builtin_bit_cast(uint32_t, low) & 0x7FFF7FFFu), (ushort2v){ 1, 1 });
        hp[e] = __builtin_bit_cast(uint32_t, up);
        lp[e] = __builtin_bit_cast(uint32_t, size) | (hp[e] & 0x80008000u);
    }
    hi = __builtin_bit_cast(half8v, h);
    lo = __builtin_bit_cast(half8v, l);
}
// Any element.
__device__ __forceinline__ void split_query(float q, float scale, _Float16 &hi, _Float16 &lo) {
    const float v = q * scale;
    hi = (_Float16)__builtin_amdgcn_cvt_pkrtz(v, 0.f)[0];
    lo = (_Float16)(v - (float)hi);
    const _Float16 least = (_Float16)copysignf(0x1p-24f, q);
    if (q != 0.f && hi == (_Float16)0.f) hi = least;
    if (q != 0.f && lo == (_Float16)0.f) lo = least;
}

// rows s = 0 .. n_seq - 1 of q, each over the positions of its sequence.  work: paged_decode_bytes() of the same arguments.
size_t paged_decode_bytes(const PagedView &p, int head_dim, int n_heads, int max_kv_len);
hipError_t launch_paged_decode(hipStream_t s, const PagedView &p, int head_dim, int max_kv_len, const float *q, size_t q_ld, int n_heads, float *out,
                               size_t out_ld, void *work);
hipError_t launch_paged_prefill(hipStream_t s, const PagedView &p, int head_dim, int n_tok, const float *q, size_t q_ld, int n_heads, float *out, size_t out_ld);

}  // namespace rt
