// Keys and values of many sequences in pages of one pool: the append of new tokens with the position rotation applied on the
// way, and the attention of new queries over the pages.
//   pool      [n_pages][n_kv_heads][page_size][head_dim] fp16, one for the keys and one for the values: the positions of one
//             head inside a page are one contiguous piece, so a workgroup that reads one head's keys reads whole pieces
//   table     [n_seq][max_blocks]: position p of sequence s is slot p % page_size of page table[s][p / page_size]
//   kv_len    [n_seq]: positions of each sequence, the new tokens included
//   cu_new    [n_seq + 1]: sequence s owns rows cu_new[s] .. cu_new[s + 1] - 1 of the new tokens (its last positions)
// All four live on the device and are read by the kernels: nothing here waits for the host.  What they say is checked where it
// is used: a page id outside the pool is never followed (append: the row is not stored; attention: its positions are not seen),
// a length beyond the table's width counts as the width, and a row that no sequence owns is left as it was.
// (The cache is the one KVCache::update of example-cli/src/model/transformer.rs:221-270 was meant to be, the attention the
// masked scores / softmax / weighted sum of example-cli/src/model/architectures/attention.rs:233-338 over it.)
#include "rt_paged.h"

#include <new>

struct rt_hip_paged_kv {
    uint16_t *k = nullptr, *v = nullptr;
    int n_pages = 0, page_size = 0, n_kv_heads = 0, head_dim = 0;
    bool owns = false;
};

namespace rt {
namespace {

// --------------------------------------------------------------------------------------------------------- append
// Element pair (a, b) of a head turns by pos * theta^(-2 i / head_dim): interleaved pairs (2i, 2i + 1) or halves
// (i, i + head_dim / 2).  The angle is taken in turns in 64 bits and reduced to [-1/2, 1/2] before it is rounded: at position
// 100 000 an f32 angle is off by up to 4e-3.  sin and cos of a token's angles are worked out once per workgroup and kept in LDS
// for all its heads.
// Bound by memory: 12 bytes of keys and values and 8 of queries per element read and written once.  14 334 ragged tokens of 32 + 8 heads of 128
// (646 MB): 119 us, 5.4 TB/s (a copy of 4 GiB moves 4.6); one token: 5.2 us, the launch and two dependent reads.
constexpr int kRopeNone = 0, kRopeInterleaved = 1, kRopeHalf = 2;

struct AppendArgs {
    PagedView p;
    const float *q, *k, *v;
    float *q_out;
    size_t q_ld, k_ld, v_ld, qo_ld;
    int n_tok, n_heads;                      // n_heads = 0: no queries
    double log2_theta;
};

template <int HD, int ROPE>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendArgs a) {
    constexpr int HALF = HD / 2;
    __shared__ __align__(16) float cs[HALF], sn[HALF];
    const int t = blockIdx.x, tid = threadIdx.x;
    int seq;
    long long pos;
    if (!row_place(a.p, t, seq, pos) || pos < 0) return;
    if (ROPE != kRopeNone) {
        if (tid < HALF) {
            const double turns = (double)pos * (exp2(-(double)(2 * tid) / (double)HD * a.log2_theta) * 0.15915494309189533577);
            float s, c;
            sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
            cs[tid] = c;
            sn[tid] = s;
        }
        __syncthreads();
    }
    const long long block = pos >> a.p.page_shift;
    int page = -1;
    if (block < a.p.max_blocks) page = a.p.table[(size_t)seq * a.p.max_blocks + block];
    const bool stored = page >= 0 && page < a.p.n_pages;
    const int slot = (int)(pos & ((1ll << a.p.page_shift) - 1));
    const size_t head_elems = (size_t)HD << a.p.page_shift;
    const size_t at = stored ? ((size_t)page * a.p.n_kv << a.p.page_shift) * HD + (size_t)slot * HD : 0;
    // a unit is four pairs' worth of one head: 4 + 4 elements HALF apart (halves) or 8 consecutive ones
    constexpr int UNITS = HD / 8;
    const int heads = a.n_heads + 2 * a.p.n_kv;
    for (int u = tid; u < heads * UNITS; u += 256) {
        const int h = u / UNITS, i = u % UNITS;
        const bool is_q = h < a.n_heads, is_k = !is_q && h < a.n_heads + a.p.n_kv;
        const int hk = is_q ? h : (is_k ? h - a.n_heads : h - a.n_heads - a.p.n_kv);
        if (!is_q && !stored) continue;
        const float *src = (is_q ? a.q + (size_t)t * a.q_ld : (is_k ? a.k + (size_t)t * a.k_ld : a.v + (size_t)t * a.v_ld)) + (size_t)hk * HD;
        const int e0 = ROPE == kRopeHalf ? 4 * i : 8 * i, e1 = ROPE == kRopeHalf ? HALF + 4 * i : 8 * i + 4;
        float4 x = *reinterpret_cast<const float4 *>(src + e0), y = *reinterpret_cast<const float4 *>(src + e1);
        if (ROPE != kRopeNone && (is_q || is_k)) {
            const float4 c = *reinterpret_cast<const float4 *>(cs + 4 * i), s = *reinterpret_cast<const float4 *>(sn + 4 * i);
            float4 p, q;
            if (ROPE == kRopeHalf) {
                p = make_float4(x.x * c.x - y.x * s.x, x.y * c.y - y.y * s.y, x.z * c.z - y.z * s.z, x.w * c.w - y.w * s.w);
                q = make_float4(x.x * s.x + y.x * c.x, x.y * s.y + y.y * c.y, x.z * s.z + y.z * c.z, x.w * s.w + y.w * c.w);
            } else {
                p = make_float4(x.x * c.x - x.y * s.x, x.x * s.x + x.y * c.x, x.z * c.y - x.w * s.y, x.z * s.y + x.w * c.y);
                q = make_float4(y.x * c.z - y.y * s.z, y.x * s.z + y.y * c.z, y.z * c.w - y.w * s.w, y.z * s.w + y.w * c.w);
            }
            x = p;
            y = q;
        }
        if (is_q) {
            float *dst = a.q_out + (size_t)t * a.qo_ld + (size_t)hk * HD;
            *reinterpret_cast<float4 *>(dst + e0) = x;
            *reinterpret_cast<float4 *>(dst + e1) = y;
        } else {
            uint16_t *dst = (is_k ? a.p.k : a.p.v) + at + (size_t)hk * head_elems;
            *reinterpret_cast<uint2 *>(dst + e0) = make_uint2((uint32_t)f2h_rne(x.x) | ((uint32_t)f2h_rne(x.y) << 16), (uint32_t)f2h_rne(x.z) | ((uint32_t)f2h_rne(x.w) << 16));
            *reinterpret_cast<uint2 *>(dst + e1) = make_uint2((uint32_t)f2h_rne(y.x) | ((uint32_t)f2h_rne(y.y) << 16), (uint32_t)f2h_rne(y.z) | ((uint32_t)f2h_rne(y.w) << 16));
        }
    }
}

}  // namespace
}  // namespace rt

using rt::fail;
using rt::Guard;

// ------------------------------------------------------------------------------------------------------ entry points
namespace {

bool power_of_two(int v) { return v > 0 && (v & (v - 1)) == 0; }
int log2_of(int v) { int s = 0; while ((1 << s) < v) s++; return s; }

int pool_check(rt_hip_ctx *ctx, size_t n_pages, int page_size, int n_kv_heads, int head_dim) {
    RT_REQUIRE(ctx, n_pages >= 1 && n_pages <= (size_t)INT32_MAX, RT_HIP_ERR_SHAPE, "paged_kv: n_pages=%zu outside 1..2^31-1", n_pages);
    RT_REQUIRE(ctx, power_of_two(page_size) && page_size >= 16 && page_size <= 1024, RT_HIP_ERR_SHAPE,
               "paged_kv: page_size=%d (a power of two from 16 to 1024 is supported)", page_size);
    RT_REQUIRE(ctx, n_kv_heads >= 1 && n_kv_heads <= 1024, RT_HIP_ERR_SHAPE, "paged_kv: n_kv_heads=%d outside 1..1024", n_kv_heads);
    RT_REQUIRE(ctx, head_dim == 64 || head_dim == 128, RT_HIP_ERR_SHAPE, "paged_kv: head_dim=%d (64 or 128 supported)", head_dim);
    return RT_HIP_OK;
}

// What append and attention share: the batch's arrays and sizes.
int batch_check(rt_hip_ctx *ctx, const char *who, const rt_hip_paged_kv *kv, const int *table, int max_blocks, const int *kv_len, int n_seq) {
    if (!kv || !table || !kv_len) return fail(ctx, RT_HIP_ERR_INVALID_ARG, "%s: NULL argument", who);
    RT_REQUIRE(ctx, n_seq >= 1 && n_seq <= 65535, RT_HIP_ERR_SHAPE, "%s: n_seq=%d outside 1..65535", who, n_seq);
    RT_REQUIRE(ctx, max_blocks >= 1 && (long long)max_blocks * kv->page_size <= (1ll << 30), RT_HIP_ERR_SHAPE,
               "%s: max_blocks=%d of %d positions (1 to 2^30 positions per sequence)", who, max_blocks, kv->page_size);
    return RT_HIP_OK;
}

int rows_check(rt_hip_ctx *ctx, const char *who, const char *name, const void *p, size_t ld, size_t least) {
    RT_REQUIRE(ctx, ((uintptr_t)p & 15) == 0, RT_HIP_ERR_INVALID_ARG, "%s: %s must be 16-byte aligned", who, name);
    RT_REQUIRE(ctx, ld >= least && ld <= rt::kRowsApartMost && ld % 4 == 0, RT_HIP_ERR_SHAPE, "%s: rows of %s are %zu floats apart (at least %zu, a multiple of 4)", who, name, ld,
               least);
    return RT_HIP_OK;
}

rt::PagedView view_of(const rt_hip_paged_kv *kv, const int *table, int max_blocks, const int *kv_len, const int *cu_new, int n_seq) {
    return rt::PagedView{ kv->k, kv->v, table, kv_len, cu_new, kv->n_pages, log2_of(kv->page_size), kv->n_kv_heads, n_seq, max_blocks };
}

int heads_check(rt_hip_ctx *ctx, const char *who, const rt_hip_paged_kv *kv, int n_heads) {
    RT_REQUIRE(ctx, n_heads >= 1 && n_heads <= 65535 && n_heads % kv->n_kv_heads == 0, RT_HIP_ERR_SHAPE, "%s: n_heads=%d with %d key / value heads", who, n_heads,
               kv->n_kv_heads);
    return RT_HIP_OK;
}

}  // namespace

extern "C" {

int rt_hip_paged_kv_wrap_dev(rt_hip_ctx *ctx, uint16_t *k_pages, uint16_t *v_pages, size_t n_pages, int page_size, int n_kv_heads, int head_dim,
                             rt_hip_paged_kv **out) {
    if (!ctx || !out) return fail(ctx, RT_HIP_ERR_INVALID_ARG, "rt_hip_paged_kv_wrap_dev: NULL argument");
    *out = nullptr;
    RT_REQUIRE(ctx, k_pages && v_pages, RT_HIP_ERR_INVALID_ARG, "rt_hip_paged_kv_wrap_dev: the pages are NULL");
    RT_REQUIRE(ctx, (((uintptr_t)k_pages | (uintptr_t)v_pages) & 15) == 0, RT_HIP_ERR_INVALID_ARG, "paged_kv: pages must be 16-byte aligned");
    int rc = pool_check(ctx, n_pages, page_size, n_kv_heads, head_dim);
    if (rc) return rc;
    rt_hip_paged_kv *kv = new (std::nothrow) rt_hip_paged_kv();
    if (!kv) return fail(ctx, RT_HIP_ERR_OOM, "host allocation failed");
    kv->k = k_pages; kv->v = v_pages; kv->n_pages = (int)n_pages; kv->page_size = page_size; kv->n_kv_heads = n_kv_heads; kv->head_dim = head_dim;
    *out = kv;
    return RT_HIP_OK;
}

int rt_hip_paged_kv_create(rt_hip_ctx *ctx, size_t n_pages, int page_size, int n_kv_heads, int head_dim, rt_hip_paged_kv **out) {
    if (!ctx || !out) return fail(ctx, RT_HIP_ERR_INVALID_ARG, "rt_hip_paged_kv_create: NULL argument");
    *out = nullptr;
    int rc = pool_check(ctx, n_pages, page_size, n_kv_heads, head_dim);
    if (rc) return rc;
    Guard g(ctx);
    rt_hip_paged_kv *kv = new (std::nothrow) rt_hip_paged_kv();
    if (!kv) return fail(ctx, RT_HIP_ERR_OOM, "host allocation failed");
    const size_t bytes = n_pages * (size_t)page_size * (size_t)n_kv_heads * (size_t)head_dim * sizeof(uint16_t);
    hipError_t e = hipMalloc((void **)&kv->k, bytes);
    if (e == hipSuccess) {
        e = hipMalloc((void **)&kv->v, bytes);
        if (e != hipSuccess) (void)hipFree(kv->k);
    }
    if (e != hipSuccess) {
        delete kv;
        return rt::hip_fail(ctx, e, "hipMalloc(pages)");
    }
    kv->n_pages = (int)n_pages; kv->page_size = page_size; kv->n_kv_heads = n_kv_heads; kv->head_dim = head_dim; kv->owns = true;
    *out = kv;
    return RT_HIP_OK;
}

int rt_hip_paged_kv_free(rt_hip_ctx *ctx, rt_hip_paged_kv *kv) {
    if (!kv) return RT_HIP_OK;
    if (!ctx) return fail(nullptr, RT_HIP_ERR_INVALID_ARG, "ctx is NULL");
    Guard g(ctx);
    if (kv->owns) {
        (void)hipStreamSynchronize(ctx->stream);
        (void)hipFree(kv->k);
        (void)hipFree(kv->v);
    }
    delete kv;
    return RT_HIP_OK;
}

int rt_hip_paged_kv_pages(rt_hip_ctx *ctx, const rt_hip_paged_kv *kv, uint16_t **k_pages, uint16_t **v_pages) {
    if (!ctx || !kv || !k_pages || !v_pages) return fail(ctx, RT_HIP_ERR_INVALID_ARG, "rt_hip_paged_kv_pages: NULL argument");
    *k_pages = kv->k;
    *v_pages = kv->v;
    return RT_HIP_OK;
}

int rt_hip_paged_append_dev(rt_hip_ctx *ctx, const rt_hip_paged_kv *kv, const int *block_table, int max_blocks, const int *kv_len, const int *cu_new, int n_seq,
                            int n_tok, const float *k, size_t k_ld, const float *v, size_t v_ld, const float *q, size_t q_ld, float *q_out, size_t q_out_ld,
                            int n_heads, int rope, float theta) {
    const char *who = "paged_append";
    if (!ctx) return fail(nullptr, RT_HIP_ERR_INVALID_ARG, "ctx is NULL");
    int rc = batch_check(ctx, who, kv, block_table, max_blocks, kv_len, n_seq);
    if (rc) return rc;
    RT_REQUIRE(ctx, k && v, RT_HIP_ERR_INVALID_ARG, "%s: NULL argument", who);
    RT_REQUIRE(ctx, n_tok >= 0 && (cu_new || n_tok == n_seq), RT_HIP_ERR_SHAPE, "%s: n_tok=%d (without cu_new one token per sequence: %d)", who, n_tok, n_seq);
    RT_REQUIRE(ctx, n_tok <= 1 << 22, RT_HIP_ERR_SHAPE, "%s: n_tok=%d is beyond one grid", who, n_tok);
    RT_REQUIRE(ctx, rope >= rt::kRopeNone && rope <= rt::kRopeHalf, RT_HIP_ERR_INVALID_ARG, "%s: rope=%d", who, rope);
    RT_REQUIRE(ctx, rope == rt::kRopeNone || (theta > 0.f && theta <= 1e30f), RT_HIP_ERR_INVALID_ARG, "%s: theta=%g", who, (double)theta);
    RT_REQUIRE(ctx, (q != nullptr) == (q_out != nullptr), RT_HIP_ERR_INVALID_ARG, "%s: q and q_out go together", who);
    const size_t rowkv = (size_t)kv->n_kv_heads * kv->head_dim;
    if ((rc = rows_check(ctx, who, "k", k, k_ld, rowkv)) || (rc = rows_check(ctx, who, "v", v, v_ld, rowkv))) return rc;
    if (q) {
        RT_REQUIRE(ctx, n_heads >= 1 && n_heads <= 65535, RT_HIP_ERR_SHAPE, "%s: n_heads=%d", who, n_heads);
        const size_t row = (size_t)n_heads * kv->head_dim;
        if ((rc = rows_check(ctx, who, "q", q, q_ld, row)) || (rc = rows_check(ctx, who, "q_out", q_out, q_out_ld, row))) return rc;
        RT_REQUIRE(ctx, q != q_out || q_ld == q_out_ld, RT_HIP_ERR_INVALID_ARG, "%s: in place, the rows of q and q_out must be equally far apart", who);
    }
    if (n_tok == 0) return RT_HIP_OK;
    Guard g(ctx);
    rt::AppendArgs a{ view_of(kv, block_table, max_blocks, kv_len, cu_new, n_seq), q, k, v, q_out, q_ld, k_ld, v_ld, q_out_ld, n_tok, q ? n_heads : 0,
                      rope == rt::kRopeNone ? 0.0 : log2((double)theta) };
    const dim3 grid((unsigned)n_tok);
    if (kv->head_dim == 128) {
        if (rope == rt::kRopeNone) rt::paged_append_kernel<128, rt::kRopeNone><<<grid, 256, 0, ctx->stream>>>(a);
        else if (rope == rt::kRopeHalf) rt::paged_append_kernel<128, rt::kRopeHalf><<<grid, 256, 0, ctx->stream>>>(a);
        else rt::paged_append_kernel<128, rt::kRopeInterleaved><<<grid, 256, 0, ctx->stream>>>(a);
    } else {
        if (rope == rt::kRopeNone) rt::paged_append_kernel<64, rt::kRopeNone><<<grid, 256, 0, ctx->stream>>>(a);
        else if (rope == rt::kRopeHalf) rt::paged_append_kernel<64, rt::kRopeHalf><<<grid, 256, 0, ctx->stream>>>(a);
        else rt::paged_append_kernel<64, rt::kRopeInterleaved><<<grid, 256, 0, ctx->stream>>>(a);
    }
    RT_TRY_HIP(ctx, hipGetLastError());
    return RT_HIP_OK;
}

int rt_hip_paged_attn_decode_dev(rt_hip_ctx *ctx, const rt_hip_paged_kv *kv, const int *block_table, int max_blocks, const int *kv_len, int n_seq, int max_kv_len,
                                 const float *q, size_t q_ld, int n_heads, float *out, size_t out_ld) {
    const char *who = "paged_attn_decode";
    if (!ctx) return fail(nullptr, RT_HIP_ERR_INVALID_ARG, "ctx is NULL");
    int rc = batch_check(ctx, who, kv, block_table, max_blocks, kv_len, n_seq);
    if (rc) return rc;
    RT_REQUIRE(ctx, q && out, RT_HIP_ERR_INVALID_ARG, "%s: NULL argument", who);
    RT_REQUIRE(ctx, max_kv_len >= 0, RT_HIP_ERR_INVALID_ARG, "%s: max_kv_len=%d", who, max_kv_len);
    if ((rc = heads_check(ctx, who, kv, n_heads))) return rc;
    RT_REQUIRE(ctx, (long long)n_seq * n_heads <= 1 << 22, RT_HIP_ERR_SHAPE, "%s: %d sequences of %d heads are beyond one grid", who, n_seq, n_heads);
    const size_t row = (size_t)n_heads * kv->head_dim;
    if ((rc = rows_check(ctx, who, "q", q, q_ld, row)) || (rc = rows_check(ctx, who, "out", out, out_ld, row))) return rc;
    Guard g(ctx);
    const rt::PagedView p = view_of(kv, block_table, max_blocks, kv_len, nullptr, n_seq);
    rc = rt::ensure_scratch(ctx, rt::paged_decode_bytes(p, kv->head_dim, n_heads, max_kv_len));
    if (rc) return rc;
    RT_TRY_HIP(ctx, rt::launch_paged_decode(ctx->stream, p, kv->head_dim, max_kv_len, q, q_ld, n_heads, out, out_ld, ctx->scratch));
    return RT_HIP_OK;
}

int rt_hip_paged_attn_prefill_dev(rt_hip_ctx *ctx, const rt_hip_paged_kv *kv, const int *block_table, int max_blocks, const int *kv_len, const int *cu_new,
                                  int n_seq, int n_tok, const float *q, size_t q_ld, int n_heads, float *out, size_t out_ld) {
    const char *who = "paged_attn_prefill";
    if (!ctx) return fail(nullptr, RT_HIP_ERR_INVALID_ARG, "ctx is NULL");
    int rc = batch_check(ctx, who, kv, block_table, max_blocks, kv_len, n_seq);
    if (rc) return rc;
    RT_REQUIRE(ctx, q && out && cu_new, RT_HIP_ERR_INVALID_ARG, "%s: NULL argument", who);
    RT_REQUIRE(ctx, n_tok >= 0, RT_HIP_ERR_SHAPE, "%s: n_tok=%d", who, n_tok);
    if ((rc = heads_check(ctx, who, kv, n_heads))) return rc;
    RT_REQUIRE(ctx, (long long)n_tok * (n_heads / kv->n_kv_heads) / 64 + n_seq <= 65535, RT_HIP_ERR_SHAPE, "%s: %d tokens of %d heads per key / value head are beyond one grid",
               who, n_tok, n_heads / kv->n_kv_heads);
    const size_t row = (size_t)n_heads * kv->head_dim;
    if ((rc = rows_check(ctx, who, "q", q, q_ld, row)) || (rc = rows_check(ctx, who, "out", out, out_ld, row))) return rc;
    if (n_tok == 0) return RT_HIP_OK;
    Guard g(ctx);
    const rt::PagedView p = view_of(kv, block_table, max_blocks, kv_len, cu_new, n_seq);
    RT_TRY_HIP(ctx, rt::launch_paged_prefill(ctx->stream, p, kv->head_dim, n_tok, q, q_ld, n_heads, out, out_ld));
    return RT_HIP_OK;
}

}  // extern "C"
