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

// rows s = 0 .. n_seq - 1 of q, each over the positions of its sequence.  work: paged_decode_bytes() of the same arguments.
size_t paged_decode_bytes(const PagedView &p, int head_dim, int n_heads, int max_kv_len);
hipError_t launch_paged_decode(hipStream_t s, const PagedView &p, int head_dim, int max_kv_len, const float *q, size_t q_ld, int n_heads, float *out,
                               size_t out_ld, void *work);
hipError_t launch_paged_prefill(hipStream_t s, const PagedView &p, int head_dim, int n_tok, const float *q, size_t q_ld, int n_heads, float *out, size_t out_ld);

}  // namespace rt
