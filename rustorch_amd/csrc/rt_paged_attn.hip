// Attention of new queries over keys and values in pages (rt_paged.hip says how they lie):
//   scores_j = (q . k_j) / sqrt(head_dim);  p = softmax(scores) with max subtraction;  out = sum_j p_j v_j
// (example-cli/src/model/architectures/attention.rs:233-338), f32 in and out, fp16 keys and values.
#include "rt_paged.h"

#include <algorithm>

namespace rt {
namespace {

typedef float float4v __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------------------------------------- one query per sequence
// Bound by reading keys and values once (2 * 2 * head_dim bytes per position and kv head), so everything else has to fit beside
// the loads, for one query head per kv head as well as for sixteen.  Both products run on the matrix cores in shapes whose
// operands are what a lane loads, with no exchange between lanes:
//   S[key][head] = K . Q^T      v_mfma_f32_16x16x32_f16: lane (g = l / 16, c = l % 16) loads 16 bytes of key c; Q is split into
//                               two halves (split_query), f32 accuracy for two instructions; the lane ends with the scores of
//                               head c and keys 4 g + r, r < 4
//   O^T[dim][head] = V^T . P    v_mfma_f32_16x16x4_f32, k = g: the lane's register p_r is the second operand as it stands if the
//                               first is the value row 4 g + r, of which the lane loads chunk c: element e of the chunk is
//                               dim VE c + e, so there is one accumulator per e
// A lane's maximum and sum therefore belong to the head whose probabilities and outputs it holds.  The f32 products take a
// third of the matrix cores' time at the rate the loads arrive at.
// A workgroup of four waves takes one chunk of one sequence's positions for up to 16 query heads of one kv head; its waves take
// tiles of 16 G positions in turn and meet at the end, through LDS.  The next tile's keys and values are requested before the
// current one is used.
// Chunks are equally long whatever the sequences are, so that a batch of one long and many short ones keeps every compute unit
// busy to the end: the chunk length comes from the sum of the lengths, and each workgroup finds its sequence by running sums of
// the chunk counts (64 sequences at a time, one load and a few lane exchanges).  A sequence of one chunk is finished at once;
// the chunks of a longer one are joined by paged_join_kernel.
// Measured (keys and values of three batches in turn, so that none stay in the last-level cache): 537 MB of one sequence of 131071
// positions 95.3 us (5.6 TB/s), 837 MB of 48 sequences 163 us (5.1 TB/s), 278 MB of 33 sequences 64 us (4.4 TB/s), join included;
// the join alone takes 4 to 5 us.  A copy of 4 GiB moves 4.6 TB/s.
constexpr int kDecodeWaves = 4, kChunkUnit = 128, kHeadsPerBlock = 16, kChunkMinUnits = 2;

__device__ __forceinline__ int length_of(const PagedView &p, int seq) {      // the table's width is at most 2^30 positions
    return seq < p.n_seq ? max(0, min(p.kv_len[seq], p.max_blocks << p.page_shift)) : 0;
}

struct DecodeArgs {
    PagedView p;
    const float *q;
    float *out;
    size_t q_ld, out_ld;
    int n_heads, group, head_blocks;
    int budget;              // chunks that all sequences together may have beyond one each; 0: every sequence is one chunk
    float *part;             // [chunk][n_heads][HD] of the sequences with several chunks, and behind it {max, sum} per entry
    float2 *part_ml;
    int2 *plan;              // [n_seq]: first chunk and number of chunks of each sequence, for the join
};

__device__ __forceinline__ int units_of(int len) { return (len + kChunkUnit - 1) / kChunkUnit; }
// Units per chunk: whole waves call this, every wave of the grid gets the same answer.  sum(units) / budget, rounded up past
// the sum's own rounding, so that sum over sequences of ceil(units / chunk) <= budget + n_seq.
__device__ __forceinline__ int chunk_units(const PagedView &p, int budget) {
    float total = 0.f;
    for (int s0 = 0; s0 < p.n_seq; s0 += 64) total += (float)units_of(length_of(p, s0 + (int)(threadIdx.x & 63)));
    total = wave_sum(total);
    return max(kChunkMinUnits, (int)fminf(total * 1.0002f / (float)budget, 1e9f) + 1);
}
__device__ __forceinline__ int chunks_of(int units, int per_chunk) { return max(1, (units + per_chunk - 1) / per_chunk); }

template <int HD, int G, int OCC>
__global__ __launch_bounds__(64 * kDecodeWaves, OCC) void paged_decode_kernel(DecodeArgs a) {
    constexpr int KK = HD / 32, VE = HD / 16, kTileKeys = 16 * G;
    typedef _Float16 halfv __attribute__((ext_vector_type(VE)));
    constexpr int PS = 4 * VE + 4;           // floats a lane leaves in LDS: its outputs, maximum, sum (16-byte rows)
    __shared__ __align__(16) float part[kDecodeWaves * 64 * PS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
    const int heads = a.p.n_kv * a.head_blocks, unit = (int)(blockIdx.x / (unsigned)heads), hx = (int)(blockIdx.x % (unsigned)heads);
    const int kvh = hx / a.head_blocks, hb = hx % a.head_blocks;
    const PagedView &p = a.p;
    const int head_in_group = hb * kHeadsPerBlock + c, head = kvh * a.group + head_in_group;
    const bool has_head = head_in_group < a.group;

    // ---- which chunk of which sequence
    int seq = -1, nth = 0, chunks = 1, len = 0, per_chunk = 0;
    if (a.budget == 0) {
        seq = unit;
        len = length_of(p, seq);
    } else {
        per_chunk = chunk_units(p, a.budget);
        for (int s0 = 0, before = 0; s0 < p.n_seq; s0 += 64) {
            const int its = length_of(p, s0 + lane), mine = s0 + lane < p.n_seq ? chunks_of(units_of(its), per_chunk) : 0;
            int upto = mine;                     // running sum over the lanes
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int below = __shfl_up(upto, o);
                if (lane >= o) upto += below;
            }
            const unsigned long long past = __ballot(before + upto > unit);
            if (past) {
                const int l = __builtin_amdgcn_readfirstlane(__ffsll(past) - 1);
                seq = s0 + l;
                chunks = __builtin_amdgcn_readlane(mine, l);
                len = __builtin_amdgcn_readlane(its, l);
                nth = unit - before - (__builtin_amdgcn_readlane(upto, l) - chunks);
                break;
            }
            before += __builtin_amdgcn_readlane(upto, 63);
        }
    }
    if (seq < 0) return;                     // the grid is cut for the most chunks there may be
    if (a.budget > 0 && nth == 0 && hx == 0 && threadIdx.x == 0) a.plan[seq] = make_int2(unit, chunks);
    const int first = chunks == 1 ? 0 : nth * per_chunk * kChunkUnit;
    const int n = chunks == 1 ? len : min(per_chunk * kChunkUnit, len - first);      // positions of this chunk (0: an empty sequence)
    const int tiles = (n + kTileKeys - 1) / kTileKeys;

    // ---- the chunk's pages, 64 table entries at a time: one per lane, bad ids as -1 (asked for before the queries are
    // split: the first tile waits for it; 33 sequences of 1 to 4097 positions 63.1 for 63.5 us)
    const int page0 = (int)(first >> p.page_shift);
    int window = 0, entry = -1;                               // entry of lane l: table[page0 + 64 * window + l]
    auto load_window = [&](int w) {
        const int i = page0 + 64 * w + lane;
        int id = i < p.max_blocks ? p.table[(size_t)seq * p.max_blocks + i] : -1;
        entry = id >= 0 && id < p.n_pages ? id : -1;
        window = w;
    };
    if (n > 0) load_window(0);

    // ---- the queries: lane (g, c) holds dims 32 kk + 8 g .. + 7 of head c, split in two halves
    half8v qhi[KK], qlo[KK];
    float sscale;
    {
        float qf[KK][8], amax = 0.f, amin = INFINITY;
        const float *qp = a.q + (size_t)seq * a.q_ld + (size_t)(has_head ? head : kvh * a.group) * HD + 8 * g;
#pragma unroll
        for (int kk = 0; kk < KK; kk++) {
            const float4 x = *reinterpret_cast<const float4 *>(qp + 32 * kk), y = *reinterpret_cast<const float4 *>(qp + 32 * kk + 4);
            qf[kk][0] = x.x; qf[kk][1] = x.y; qf[kk][2] = x.z; qf[kk][3] = x.w;
            qf[kk][4] = y.x; qf[kk][5] = y.y; qf[kk][6] = y.z; qf[kk][7] = y.w;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                amax = fmaxf(amax, fabsf(qf[kk][e]));
                amin = fminf(amin, fabsf(qf[kk][e]));
            }
        }
        amax = fmaxf(amax, __shfl_xor(amax, 16));
        amax = fmaxf(amax, __shfl_xor(amax, 32));
        int ex = 0;
        if (amax > 0.f) frexpf(amax, &ex);               // amax = f * 2^ex, f in [0.5, 1)
        ex = max(ex, -100);
        const float qscale = ldexpf(1.0f, 14 - ex);
        // scores in units of log2: exp2 is the hardware's own exponential
        sscale = ldexpf(1.0f, ex - 14) * (1.44269504088896341f / sqrtf((float)HD));
        if (__ballot(!(amin * qscale >= 0x1p-24f)) == 0) {
#pragma unroll
            for (int kk = 0; kk < KK; kk++) split_queries(qf[kk], qscale, qhi[kk], qlo[kk]);
        } else {
#pragma unroll
            for (int kk = 0; kk < KK; kk++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    _Float16 hi, lo;
                    split_query(qf[kk][e], qscale, hi, lo);
                    qhi[kk][e] = hi;
                    qlo[kk][e] = lo;
                }
        }
    }

    // ---- a tile: G groups of 16 consecutive positions, each inside one page
    const size_t k_lane = (size_t)c * HD + 8 * g, v_lane = (size_t)(4 * g) * HD + VE * c;
    const int in_page = (1 << p.page_shift) - 1, first_in_page = (int)(first & in_page);
    half8v kreg[G][KK];
    halfv vreg[G][4];
    int ok = 0;                                          // bit i: group i lies on a page of the pool
    auto request = [&](int t, half8v (&kr)[G][KK], halfv (&vr)[G][4], int &good) {
        good = 0;
#pragma unroll
        for (int i = 0; i < G; i++) {
            const int at = first_in_page + t * kTileKeys + 16 * i, pg = at >> p.page_shift;     // positions behind the start of page0
            if ((pg >> 6) != window) load_window(pg >> 6);
            const int id = __builtin_amdgcn_readlane(entry, pg & 63);
            good |= id >= 0 ? 1 << i : 0;
            const size_t base = ((((size_t)max(id, 0) * p.n_kv + kvh) << p.page_shift) + (size_t)(at & in_page)) * HD;
#pragma unroll
            for (int kk = 0; kk < KK; kk++) kr[i][kk] = *reinterpret_cast<const half8v *>(p.k + base + k_lane + 32 * kk);
#pragma unroll
            for (int r = 0; r < 4; r++) vr[i][r] = *reinterpret_cast<const halfv *>(p.v + base + v_lane + (size_t)r * HD);
        }
    };
    float4v acc[VE];
#pragma unroll
    for (int e = 0; e < VE; e++)
#pragma unroll
        for (int r = 0; r < 4; r++) acc[e][r] = 0.f;
    float m_run = -INFINITY, l_run = 0.f;

    if (wave < tiles) request(wave, kreg, vreg, ok);
    for (int t = wave; t < tiles; t += kDecodeWaves) {
        half8v kn[G][KK];
        halfv vn[G][4];
        int okn = 0;
        request(min(t + kDecodeWaves, tiles - 1), kn, vn, okn);      // past the end a tile is requested again: no branch around the loads

        float4v s[G];
#pragma unroll
        for (int i = 0; i < G; i++) {
            s[i] = float4v{ 0.f, 0.f, 0.f, 0.f };
#pragma unroll
            for (int kk = 0; kk < KK; kk++) {
                s[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kreg[i][kk], qhi[kk], s[i], 0, 0, 0);
                s[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kreg[i][kk], qlo[kk], s[i], 0, 0, 0);
            }
        }
        const int left = n - t * kTileKeys;              // positions of the tile that are the chunk's
        if (left >= kTileKeys && ok == (1 << G) - 1) {
#pragma unroll
            for (int i = 0; i < G; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) s[i][r] *= sscale;
        } else {                                         // what is not seen scores -inf, and its values (stale, perhaps NaN) count as zeros
#pragma unroll
            for (int i = 0; i < G; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const bool seen = 16 * i + 4 * g + r < left && ((ok >> i) & 1);
                    s[i][r] = seen ? s[i][r] * sscale : -INFINITY;
#pragma unroll
                    for (int e = 0; e < VE; e++) vreg[i][r][e] = seen ? vreg[i][r][e] : (_Float16)0.f;
                }
        }
        float mt = m_run;
#pragma unroll
        for (int i = 0; i < G; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) mt = fmaxf(mt, s[i][r]);
        mt = fmaxf(mt, __shfl_xor(mt, 16));
        mt = fmaxf(mt, __shfl_xor(mt, 32));
        const float m_ref = mt == -INFINITY ? 0.f : mt;  // nothing seen yet
        const float alpha = __builtin_amdgcn_exp2f(m_run - m_ref);
        m_run = mt;
        l_run *= alpha;
#pragma unroll
        for (int e = 0; e < VE; e++)
#pragma unroll
            for (int r = 0; r < 4; r++) acc[e][r] *= alpha;
#pragma unroll
        for (int i = 0; i < G; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float w = __builtin_amdgcn_exp2f(s[i][r] - m_ref);
                l_run += w;
#pragma unroll
                for (int e = 0; e < VE; e++) acc[e] = __builtin_amdgcn_mfma_f32_16x16x4f32((float)vreg[i][r][e], w, acc[e], 0, 0, 0);
            }
#pragma unroll
        for (int i = 0; i < G; i++) {
#pragma unroll
            for (int kk = 0; kk < KK; kk++) kreg[i][kk] = kn[i][kk];
#pragma unroll
            for (int r = 0; r < 4; r++) vreg[i][r] = vn[i][r];
        }
        ok = okn;
    }
    l_run += __shfl_xor(l_run, 16);
    l_run += __shfl_xor(l_run, 32);

    // ---- the four waves' results meet in LDS; wave w finishes dims VE (4 g + w) .. of every head
    float *mine = part + (wave * 64 + lane) * PS;
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
        for (int e = 0; e < VE; e += 4) *reinterpret_cast<float4 *>(mine + VE * r + e) = make_float4(acc[e][r], acc[e + 1][r], acc[e + 2][r], acc[e + 3][r]);
    *reinterpret_cast<float2 *>(mine + 4 * VE) = make_float2(m_run, l_run);
    __syncthreads();
    float fw[kDecodeWaves], m_all = -INFINITY, l_all = 0.f;
#pragma unroll
    for (int w = 0; w < kDecodeWaves; w++) {
        fw[w] = part[(w * 64 + lane) * PS + 4 * VE];
        m_all = fmaxf(m_all, fw[w]);
    }
    const float m_ref = m_all == -INFINITY ? 0.f : m_all;
#pragma unroll
    for (int w = 0; w < kDecodeWaves; w++) {
        fw[w] = __builtin_amdgcn_exp2f(fw[w] - m_ref);           // a wave without positions reports -inf: factor 0
        l_all += part[(w * 64 + lane) * PS + 4 * VE + 1] * fw[w];
    }
    if (!has_head) return;
    float o[VE];
#pragma unroll
    for (int e = 0; e < VE; e++) o[e] = 0.f;
#pragma unroll
    for (int w = 0; w < kDecodeWaves; w++)
#pragma unroll
        for (int e = 0; e < VE; e += 4) {
            const float4 x = *reinterpret_cast<const float4 *>(part + (w * 64 + lane) * PS + VE * wave + e);
            o[e] += x.x * fw[w]; o[e + 1] += x.y * fw[w]; o[e + 2] += x.z * fw[w]; o[e + 3] += x.w * fw[w];
        }
    float *dst;
    float inv = 1.f;
    if (chunks == 1) {
        dst = a.out + (size_t)seq * a.out_ld + (size_t)head * HD;
        inv = l_all == 0.f ? 0.f : 1.0f / l_all;
    } else {
        const size_t slot = (size_t)unit * a.n_heads + head;
        dst = a.part + slot * HD;
        if (wave == 0 && g == 0) a.part_ml[slot] = make_float2(m_all, l_all);
    }
#pragma unroll
    for (int e = 0; e < VE; e += 4)
        *reinterpret_cast<float4 *>(dst + VE * (4 * g + wave) + e) = make_float4(o[e] * inv, o[e + 1] * inv, o[e + 2] * inv, o[e + 3] * inv);
}

// The chunks of one (sequence, head): out = sum_j acc_j 2^(m_j - M) / sum_j l_j 2^(m_j - M).  HD / 4 threads read one chunk's
// outputs; every such group runs over its chunks with a maximum of its own, and the groups meet in LDS: two dependent reads of
// memory (the plan, the partial results) from start to end.
constexpr int kJoinThreads = 256;
template <int HD>
__global__ __launch_bounds__(kJoinThreads) void paged_join_kernel(DecodeArgs a) {
    constexpr int TPR = HD / 4, ROWS = kJoinThreads / TPR;
    __shared__ __align__(16) float4 sums[kJoinThreads];
    __shared__ float2 rows[ROWS];
    const int head = blockIdx.x, seq = blockIdx.y, tid = threadIdx.x, row = tid / TPR, d = tid % TPR;
    const int2 plan = a.plan[seq];
    if (plan.y == 1) return;                 // written by the kernel before
    const float2 *ml = a.part_ml + (size_t)plan.x * a.n_heads + head;
    const float *acc = a.part + ((size_t)plan.x * a.n_heads + head) * HD + 4 * d;
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int j = row; j < plan.y; j += ROWS) {
        const float2 x = ml[(size_t)j * a.n_heads];
        const float4 v = *reinterpret_cast<const float4 *>(acc + (size_t)j * a.n_heads * HD);
        const float m_new = fmaxf(m, x.x), m_ref = m_new == -INFINITY ? 0.f : m_new;
        const float keep = __builtin_amdgcn_exp2f(m - m_ref), w = __builtin_amdgcn_exp2f(x.x - m_ref);
        m = m_new;
        l = l * keep + x.y * w;
        o.x = o.x * keep + v.x * w; o.y = o.y * keep + v.y * w; o.z = o.z * keep + v.z * w; o.w = o.w * keep + v.w * w;
    }
    sums[tid] = o;
    if (d == 0) rows[row] = make_float2(m, l);
    __syncthreads();
    if (tid >= TPR) return;
    float m_all = -INFINITY;
#pragma unroll
    for (int i = 0; i < ROWS; i++) m_all = fmaxf(m_all, rows[i].x);
    const float m_ref = m_all == -INFINITY ? 0.f : m_all;
    l = 0.f;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
        const float w = __builtin_amdgcn_exp2f(rows[i].x - m_ref);
        const float4 v = sums[i * TPR + tid];
        l += rows[i].y * w;
        o.x += v.x * w; o.y += v.y * w; o.z += v.z * w; o.w += v.w * w;
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    *reinterpret_cast<float4 *>(a.out + (size_t)seq * a.out_ld + (size_t)head * HD + 4 * tid) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
}

// Chunks beyond one per sequence that a launch may cut (0: none, and no join).
//   * No position count above 256: every sequence is one chunk.  One chat of 200 positions, 32 heads: 8.6 us; cut in two and
//     joined, 11.0 us.
//   * Several sequences: about 1536 workgroups, two rounds of the three that a compute unit holds.  33 sequences of 1 to 4097
//     positions, 8 kv heads: 71 us with 512 workgroups, 66 with 1024, 63 with 1536 and 2048; 48 sequences of 1000 to 16000, 4 kv
//     heads: 188, 176, 163, 167.
//   * One sequence: its chunks are equally long, one workgroup per compute unit ends level, and fewer streams read memory faster.
//     131071 positions, 8 kv heads: 95.5 us with 256 workgroups, 101 with 512, 103 with 768, 109 with 1536.
int decode_budget(const PagedView &p, int n_heads, int max_kv_len) {
    const int group = n_heads / p.n_kv, head_blocks = (group + kHeadsPerBlock - 1) / kHeadsPerBlock;
    const long long width = (long long)p.max_blocks << p.page_shift, longest = max_kv_len > 0 ? std::min((long long)max_kv_len, width) : width;
    if (longest <= kChunkMinUnits * kChunkUnit) return 0;
    const long long useful = (longest + kChunkMinUnits * kChunkUnit - 1) / (kChunkMinUnits * kChunkUnit) * p.n_seq;
    return (int)std::max(1ll, std::min(useful, (p.n_seq == 1 ? 256ll : 1536ll) / (p.n_kv * head_blocks)));
}

}  // namespace

size_t paged_decode_bytes(const PagedView &p, int head_dim, int n_heads, int max_kv_len) {
    const size_t budget = (size_t)decode_budget(p, n_heads, max_kv_len);
    return budget == 0 ? 0 : (budget + p.n_seq) * n_heads * ((size_t)head_dim + 2) * sizeof(float) + (size_t)p.n_seq * sizeof(int2);
}

hipError_t launch_paged_decode(hipStream_t s, const PagedView &p, int head_dim, int max_kv_len, const float *q, size_t q_ld, int n_heads, float *out,
                               size_t out_ld, void *work) {
    DecodeArgs a{ p, q, out, q_ld, out_ld, n_heads, n_heads / p.n_kv, 0, decode_budget(p, n_heads, max_kv_len), nullptr, nullptr, nullptr };
    a.head_blocks = (a.group + kHeadsPerBlock - 1) / kHeadsPerBlock;
    const size_t chunks = (size_t)a.budget + p.n_seq;
    if (a.budget > 0) {
        a.part = static_cast<float *>(work);
        a.part_ml = reinterpret_cast<float2 *>(a.part + chunks * n_heads * head_dim);
        a.plan = reinterpret_cast<int2 *>(a.part_ml + chunks * n_heads);
    }
    const dim3 grid((unsigned)(chunks * p.n_kv * a.head_blocks)), join((unsigned)n_heads, (unsigned)p.n_seq);
    // 16 positions a tile and three workgroups per compute unit, against 32 and two: 163 for 164 us (48 sequences), 63 for 67 (33
    // sequences); heads of 64, whose tiles are half as large: 32 positions
    if (head_dim == 128) {
        paged_decode_kernel<128, 1, 3><<<grid, 64 * kDecodeWaves, 0, s>>>(a);
        if (a.budget > 0) paged_join_kernel<128><<<join, kJoinThreads, 0, s>>>(a);
    } else {
        paged_decode_kernel<64, 2, 4><<<grid, 64 * kDecodeWaves, 0, s>>>(a);
        if (a.budget > 0) paged_join_kernel<64><<<join, kJoinThreads, 0, s>>>(a);
    }
    return hipGetLastError();
}

namespace {

// --------------------------------------------------------------------------------------------- several queries per sequence
// Bound by the matrix cores.  The rows of one kv head of one sequence -- its new tokens times the query heads that share the kv
// head -- are packed one after the other; a wave has 32 of them, a workgroup 32 W, and the workgroup's keys and values go through
// LDS once for all of them.  Flash style, tiles of 32 positions:
//   S^T[key][row]  = K . (Qhi + Qlo)^T    v_mfma_f32_32x32x16_f16, the f32 side in two halves (split_query): f32 accuracy for twice
//                                         the products.  A lane's 16 scores belong to one row.
//   O^T[dim][row]  = V^T . (Phi + Plo)^T  a lane's 16 probabilities are, as they stand, the second operand; the first wants four
//                                         consecutive keys of one dim per register pair, which ds_read_b64_tr_b16 reads from the
//                                         row-major tile.
// Chunks of 16 bytes are swizzled inside their rows so that both kinds of reads meet all banks.  The next tile waits in registers
// while the current one is used, the one behind it is requested then: one barrier per tile.
// The grid runs kv heads first: neighbouring workgroups land on different XCDs, so an XCD sees few kv heads and keeps their keys and
// values in its L2; later rows, which have more keys, go first.
// A value that is not finite makes NaN of a row's sums where it should not: at a position that the row does not see, as 0 * inf, and
// at one that it sees, where a half of the probability is zero.  Rows whose outputs are NaN at the end though their weights are not
// are done again by themselves (attend_row), where a value meets its weight once and only if it is seen: nothing in the loop
// over the tiles looks for such values.  A weight that f32 cannot hold (below 2^-149 of the largest) is zero there too, and NaN with them.
// Measured: one prompt of 8191 tokens, 32 heads over 8 kv heads of 128: 1.04 ms = 529 TFLOP/s of the formula, 1059 of fp16 products (a
// library product of 8192^3 reaches 1139); a prompt of 512, 32 kv heads: 21.9 us.
constexpr int kPrefillKeys = 32;

struct PrefillArgs {
    PagedView p;
    const float *q;
    float *out;
    size_t q_ld, out_ld;
    int n_tok, n_heads, group;
};

// ds_read_b64_tr_b16: in each 16 lanes, lane i gets the i-th column of the 4 x 16 matrix whose row r is the 8 bytes each of lanes 4 r .. 4 r + 3
typedef short short4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) short4v lds_short4v;
typedef _Float16 half4v __attribute__((ext_vector_type(4)));
__device__ __forceinline__ half4v read_transposed(const uint16_t *p) { return __builtin_bit_cast(half4v, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4v *)p)); }

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float float16v __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// One row of one query head by one wave: nothing that is not seen is touched, and a value meets its weight once.  64 positions at a time,
// a lane scoring one of them, then their values, 16 requests on their way: bound by latency, about 6 us per 64 positions (8 rows of 32 heads
// behind 100 000 positions whose values are all NaN: 326 ms; 20 ms for one infinite value, which few rows meet with a half of zero).
template <int HD>
__device__ void attend_row(const PagedView &p, const float *q, float *out, int seq, int kvh, int n) {
    constexpr int E = HD / 64;               // elements of the output that a lane holds
    const int lane = (int)(threadIdx.x & 63);
    const float scale = 1.0f / sqrtf((float)HD);
    float acc[E], m = -INFINITY, l = 0.f;
    for (int e = 0; e < E; e++) acc[e] = 0.f;
    for (int j0 = 0; j0 < n; j0 += 64) {
        const int j = j0 + lane, page = j < n ? p.table[(size_t)seq * p.max_blocks + (j >> p.page_shift)] : -1;
        const bool seen = page >= 0 && page < p.n_pages;
        const size_t at = ((((size_t)(seen ? page : 0) * p.n_kv + kvh) << p.page_shift) + (size_t)(j & ((1 << p.page_shift) - 1))) * HD;
        float s = 0.f;
#pragma unroll
        for (int d = 0; d < HD; d += 8) {
            const half8v k = *reinterpret_cast<const half8v *>(p.k + at + d);
            const float4 x = *reinterpret_cast<const float4 *>(q + d), y = *reinterpret_cast<const float4 *>(q + d + 4);
            s += ((x.x * (float)k[0] + x.y * (float)k[1]) + (x.z * (float)k[2] + x.w * (float)k[3])) +
                 ((y.x * (float)k[4] + y.y * (float)k[5]) + (y.z * (float)k[6] + y.w * (float)k[7]));
        }
        s = seen ? s * scale : -INFINITY;
        const float m_new = fmaxf(m, wave_max(s));
        const float keep = m_new == -INFINITY ? 1.f : expf(m - m_new), w = s == -INFINITY ? 0.f : expf(s - m_new);      // a score of NaN: NaN
        l = l * keep + wave_sum(w);
        for (int e = 0; e < E; e++) acc[e] *= keep;
#pragma unroll 16
        for (int i = 0; i < 64; i++) {                            // behind the end: nothing seen, weight 0
            const size_t row = ((size_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(at >> 32), i) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)at, i);
            const float weight = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), i));
            const bool is = __builtin_amdgcn_readlane(seen ? 1 : 0, i) != 0;
            for (int e = 0; e < E; e++) {
                const float v = h2f(p.v[row + E * lane + e]);
                acc[e] += weight * (is ? v : 0.f);
            }
        }
        m = m_new;
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    for (int e = 0; e < E; e++) out[E * lane + e] = acc[e] * inv;
}

// W waves of 32 rows, and S such groups of waves that take the tiles in turn, each with running states and LDS tiles of its own; they
// meet at the end, through LDS.
template <int HD, int W, int S>
constexpr size_t prefill_lds_bytes() {
    return std::max((size_t)S * 2 * 2 * kPrefillKeys * HD * sizeof(uint16_t), (size_t)(S - 1) * 64 * W * (HD / 2 + 2) * sizeof(float));
}
template <int HD, int W, int S>
__global__ __launch_bounds__(64 * W * S, 2) void paged_prefill_kernel(PrefillArgs a) {
    constexpr int KK = HD / 16, DB = HD / 32, CPR = HD / 8, TQ = 32 * W, KT = kPrefillKeys;
    constexpr int ROWS_AT_ONCE = 64 * W / CPR, NL = KT / ROWS_AT_ONCE;     // rows of a tile that the workgroup's threads load at once, and how often
    static_assert(NL >= 1 && (16 % ROWS_AT_ONCE == 0 || ROWS_AT_ONCE % 16 == 0), "a load covers whole groups of 16 positions or lies inside one");
    RT_DYN_LDS(uint4, lds16);                // 16-byte aligned beside the static variable
    uint16_t *const lds = reinterpret_cast<uint16_t *>(lds16);
    const PagedView &p = a.p;
    const int all_waves = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), split = all_waves / W, wave = all_waves % W;
    const int tid = (int)threadIdx.x - 64 * W * split, lane = tid & 63, j = lane & 31, hh = lane >> 5;
    uint16_t *const ks = lds + (size_t)split * 4 * KT * HD, *const vs = ks + 2 * KT * HD;       // two tiles of keys, two of values
    const int kvh = blockIdx.x, tile = (int)blockIdx.y;

    // ---- which rows.  Up to 64 sequences: the one with the most positions first, and of each its last rows first, which see the most
    // (a long one that began last would end alone: six chunks behind prefixes of 0 to 3000 take 107 instead of 132 us).  More: sequence s
    // has the tiles from floor(cu_new[s] * group / TQ) + s on, the last first.
    int seq = 0, nth;
    if (p.n_seq <= 64) {
        int rows = 0, keys = 0;
        if (lane < p.n_seq) {
            const int b = p.cu_new[lane], e = p.cu_new[lane + 1];
            if (b >= 0 && e <= a.n_tok && e > b) {
                rows = (int)(((long long)(e - b) * a.group + TQ - 1) / TQ);
                keys = length_of(p, lane);
            }
        }
        int begin = 0;
        for (int o = 0; o < p.n_seq; o++) {
            const int its = __builtin_amdgcn_readlane(keys, o), many = __builtin_amdgcn_readlane(rows, o);
            if (its > keys || (its == keys && o < lane)) begin += many;
        }
        const unsigned long long here = __ballot(rows > 0 && begin <= tile && tile < begin + rows);
        if (!here) return;
        seq = __builtin_amdgcn_readfirstlane(__ffsll(here) - 1);
        nth = __builtin_amdgcn_readlane(begin + rows, seq) - 1 - tile;
    } else {
        const int back = (int)gridDim.y - 1 - tile;
        for (int s0 = 1; s0 < p.n_seq; s0 += 64) {
            const int s = s0 + lane;
            const unsigned long long begun = __ballot(s < p.n_seq && (long long)p.cu_new[s] * a.group / TQ + s <= back);
            seq += __popcll(begun);
            if (begun != ~0ull) break;
        }
        nth = (int)(back - ((long long)p.cu_new[seq] * a.group / TQ + seq));
    }
    const int t0 = p.cu_new[seq], t1 = p.cu_new[seq + 1];
    if (t0 < 0 || t1 > a.n_tok || t1 <= t0 || nth < 0) return;
    const long long first_row = (long long)nth * TQ;
    const int n_rows = (int)min((long long)TQ, (long long)(t1 - t0) * a.group - first_row);
    if (n_rows <= 0) return;
    const int width = p.max_blocks << p.page_shift, new_tok = t1 - t0;
    auto place = [&](int row, int &tok, int &head) -> int {       // of a row of the tile; returns the positions it sees
        const long long r = first_row + row;
        tok = (int)(r / a.group);
        head = (int)(r - (long long)tok * a.group);
        return (int)max(0ll, min((long long)width, (long long)p.kv_len[seq] - new_tok + tok + 1));
    };
    int tok, head_in_group, least, most;
    least = place(0, tok, head_in_group);                         // positions that the first row sees: every row sees them
    most = place(n_rows - 1, tok, head_in_group);
    const int seen = place(min(32 * wave + j, n_rows - 1), tok, head_in_group);
    const int wave_most = [&] { int t, h; return 32 * wave < n_rows ? place(min(32 * wave + 31, n_rows - 1), t, h) : 0; }();
    const float *qrow = a.q + (size_t)(t0 + tok) * a.q_ld + (size_t)(kvh * a.group + head_in_group) * HD;
    float *orow = a.out + (size_t)(t0 + tok) * a.out_ld + (size_t)(kvh * a.group + head_in_group) * HD;
    const bool has_row = 32 * wave + j < n_rows;

    // ---- the query fragments: lane (j, hh) holds elements 16 kk + 8 hh .. + 7 of its row
    half8v qhi[KK], qlo[KK];
    float sscale;
    {
        float amax = 0.f, amin = INFINITY;
        auto eight = [&](int kk, float (&f)[8]) {
            const float4 x = *reinterpret_cast<const float4 *>(qrow + 16 * kk + 8 * hh), y = *reinterpret_cast<const float4 *>(qrow + 16 * kk + 8 * hh + 4);
            f[0] = x.x; f[1] = x.y; f[2] = x.z; f[3] = x.w;
            f[4] = y.x; f[5] = y.y; f[6] = y.z; f[7] = y.w;
        };
        for (int kk = 0; kk < KK; kk++) {
            float f[8];
            eight(kk, f);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                amax = fmaxf(amax, fabsf(f[e]));
                amin = fminf(amin, fabsf(f[e]));
            }
        }
        amax = fmaxf(amax, __shfl_xor(amax, 32));
        int ex = 0;
        if (amax > 0.f) frexpf(amax, &ex);               // amax = f * 2^ex, f in [0.5, 1)
        ex = max(ex, -100);
        const float qscale = ldexpf(1.0f, 14 - ex);
        sscale = ldexpf(1.0f, ex - 14) * (1.44269504088896341f / sqrtf((float)HD));       // scores in units of log2
        if (__ballot(!(amin * qscale >= 0x1p-24f)) == 0) {
#pragma unroll
            for (int kk = 0; kk < KK; kk++) {
                float f[8];
                eight(kk, f);
                split_queries(f, qscale, qhi[kk], qlo[kk]);
            }
        } else {
#pragma unroll
            for (int kk = 0; kk < KK; kk++) {
                float f[8];
                eight(kk, f);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    _Float16 hi, lo;
                    split_query(f[e], qscale, hi, lo);
                    qhi[kk][e] = hi;
                    qlo[kk][e] = lo;
                }
            }
        }
    }

    // ---- tiles: a thread brings chunk c of rows r0 + i * ROWS_AT_ONCE
    const int tiles = (most + KT - 1) / KT, r0 = tid / CPR, c = tid % CPR;
    u32x4 kreg[NL], vreg[NL];
    int good = 0;                            // bit g: positions 16 g .. of the requested tile lie on a page of the pool
    auto request = [&](int t) {
        good = 0;
        size_t base[KT / 16];
#pragma unroll
        for (int g = 0; g < KT / 16; g++) {
            const int key = t * KT + 16 * g, pg = key >> p.page_shift;
            const int id = pg < p.max_blocks ? p.table[(size_t)seq * p.max_blocks + pg] : -1;
            const bool ok = id >= 0 && id < p.n_pages;
            good |= ok ? 1 << g : 0;
            base[g] = ((((size_t)(ok ? id : 0) * p.n_kv + kvh) << p.page_shift) + (size_t)(key & ((1 << p.page_shift) - 1))) * HD;
        }
#pragma unroll
        for (int i = 0; i < NL; i++) {
            const int r = r0 + i * ROWS_AT_ONCE;
            const size_t at = (r >= 16 ? base[1] : base[0]) + (size_t)(r & 15) * HD + 8 * c;
            kreg[i] = *reinterpret_cast<const u32x4 *>(p.k + at);
            vreg[i] = *reinterpret_cast<const u32x4 *>(p.v + at);
        }
    };
    auto put = [&](int t, int buf, int ok) {             // the requested tile t goes to LDS; values that no row sees (stale, perhaps NaN) as zeros
        if ((t + 1) * KT > least || ok != (1 << (KT / 16)) - 1) {
#pragma unroll
            for (int i = 0; i < NL; i++) {
                const int r = r0 + i * ROWS_AT_ONCE;
                const bool is = t * KT + r < most && ((ok >> (r >> 4)) & 1);
#pragma unroll
                for (int e = 0; e < 4; e++) vreg[i][e] = is ? vreg[i][e] : 0u;
            }
        }
#pragma unroll
        for (int i = 0; i < NL; i++) {
            const int r = r0 + i * ROWS_AT_ONCE;
            const int vc = HD == 128 ? c ^ (4 * (r & 3)) : c ^ (4 * ((r >> 1) & 1));
            *reinterpret_cast<u32x4 *>(ks + buf * KT * HD + r * HD + 8 * (c ^ (r & (CPR - 1)))) = kreg[i];
            *reinterpret_cast<u32x4 *>(vs + buf * KT * HD + r * HD + 8 * vc) = vreg[i];
        }
    };

    float16v acc[DB];
#pragma unroll
    for (int db = 0; db < DB; db++)
#pragma unroll
        for (int r = 0; r < 16; r++) acc[db][r] = 0.f;
    float m_run = -INFINITY, l_run = 0.f;
    int ok_now = 0, ok_next = 0;
    const int steps = (tiles + S - 1) / S;                // the group's tile of step n is S n + split; past the last it is requested again, unused
    if (tiles > 0) {
        request(min(split, tiles - 1));
        ok_now = good;
        put(min(split, tiles - 1), 0, ok_now);
        request(min(S + split, tiles - 1));
        ok_next = good;
    }
    __syncthreads();
    // the value rows of the transposed reads: source lane s of a group of 16 reads 4 dims of row s / 4
    const int s16 = lane & 15, vrow0 = 4 * hh + (s16 >> 2), vcol0 = 16 * ((lane >> 4) & 1) + 4 * (s16 & 3);
    for (int n = 0; n < steps; n++) {
        const int buf = n & 1, t = S * n + split;
        if (t < tiles && t * KT < wave_most) {
            float16v s;
#pragma unroll
            for (int r = 0; r < 16; r++) s[r] = 0.f;
#pragma unroll
            for (int kk = 0; kk < KK; kk++) {
                const half8v k = *reinterpret_cast<const half8v *>(ks + buf * KT * HD + j * HD + 8 * ((2 * kk + hh) ^ (j & (CPR - 1))));
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, qhi[kk], s, 0, 0, 0);
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, qlo[kk], s, 0, 0, 0);
            }
            // register r is position 8 (r / 4) + 4 hh + r % 4 of the tile against the lane's row
            if ((t + 1) * KT > least || ok_now != (1 << (KT / 16)) - 1) {
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int at = 8 * (r >> 2) + 4 * hh + (r & 3);
                    s[r] = t * KT + at < seen && ((ok_now >> (at >> 4)) & 1) ? s[r] : -INFINITY;
                }
            }
            float mt = s[0];
#pragma unroll
            for (int r = 1; r < 16; r++) mt = fmaxf(mt, s[r]);
            mt = fmaxf(mt, __shfl_xor(mt, 32));
            mt = fmaxf(m_run, mt);                               // running maximum of the products, before the scaling
            const float m_ref = mt == -INFINITY ? 0.f : mt;      // nothing seen yet
            if (__ballot(mt > m_run)) {
                const float alpha = __builtin_amdgcn_exp2f((m_run - m_ref) * sscale);
                l_run *= alpha;
#pragma unroll
                for (int db = 0; db < DB; db++)
#pragma unroll
                    for (int r = 0; r < 16; r++) acc[db][r] *= alpha;
                m_run = mt;
            }
            // probabilities times 2^14, so that the lower halves stay normal numbers; both halves are cut, not rounded, which leaves
            // 2^-21 of a probability
            half8v phi[2], plo[2];
            float shift = fmaf(-m_ref, sscale, 14.0f);
            // shift is rounded, to 2^-18 below 128.  Beyond that tiles with another maximum would weigh noticeably differently, and from 2^24 on
            // the largest weight would be more than an fp16 holds, or nothing: there the differences, at most 0, are taken first.
            if (__ballot(!(fabsf(shift) < 128.0f))) {
#pragma unroll
                for (int r = 0; r < 16; r++) s[r] -= m_ref;
                shift = 14.0f;
            }
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                const float w0 = __builtin_amdgcn_exp2f(fmaf(s[r], sscale, shift)), w1 = __builtin_amdgcn_exp2f(fmaf(s[r + 1], sscale, shift));
                l_run += w0 + w1;
                const half2v hi = __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_pkrtz(w0, w1));
                const half2v lo = __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_pkrtz(w0 - (float)hi[0], w1 - (float)hi[1]));
                phi[r >> 3][r & 7] = hi[0]; phi[r >> 3][(r & 7) + 1] = hi[1];
                plo[r >> 3][r & 7] = lo[0]; plo[r >> 3][(r & 7) + 1] = lo[1];
            }
            // slot e of product mm stands for row 16 mm + 8 (e / 4) + 4 hh + e % 4 of the tile; the products of one block of dims wait for
            // one another, so the blocks take turns
#pragma unroll
            for (int mm = 0; mm < 2; mm++) {
                half8v av[DB];
#pragma unroll
                for (int db = 0; db < DB; db++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const int row = 16 * mm + 8 * h + vrow0, col = 32 * db + vcol0, ch = col >> 3;
                        const int vc = HD == 128 ? ch ^ (4 * (row & 3)) : ch ^ (4 * ((row >> 1) & 1));
                        const half4v x = read_transposed(vs + buf * KT * HD + row * HD + 8 * vc + (col & 7));
#pragma unroll
                        for (int e = 0; e < 4; e++) av[db][4 * h + e] = x[e];
                    }
#pragma unroll
                for (int db = 0; db < DB; db++) acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(av[db], phi[mm], acc[db], 0, 0, 0);
#pragma unroll
                for (int db = 0; db < DB; db++) acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(av[db], plo[mm], acc[db], 0, 0, 0);
            }
        }
        if (n + 1 < steps) {
            put(min(t + S, tiles - 1), buf ^ 1, ok_next);
            ok_now = ok_next;
            request(min(t + 2 * S, tiles - 1));
            ok_next = good;
        }
        __syncthreads();
    }
    l_run += __shfl_xor(l_run, 32);
    if (S > 1) {                                          // the tiles are done with: their memory takes what the groups leave, [value][thread]
        float *left = reinterpret_cast<float *>(lds);
        constexpr int NV = 16 * DB + 2, NT = 64 * W;
        if (split > 0) {
            float *mine = left + (size_t)(split - 1) * NV * NT + tid;
#pragma unroll
            for (int db = 0; db < DB; db++)
#pragma unroll
                for (int r = 0; r < 16; r++) mine[(16 * db + r) * NT] = acc[db][r];
            mine[16 * DB * NT] = m_run;
            mine[(16 * DB + 1) * NT] = l_run;
        }
        __syncthreads();
        if (split > 0) return;
        for (int o = 0; o < S - 1; o++) {
            const float *its = left + (size_t)o * NV * NT + tid;
            const float m_its = its[16 * DB * NT], m = fmaxf(m_run, m_its), m_ref = m == -INFINITY ? 0.f : m;
            const float keep = __builtin_amdgcn_exp2f((m_run - m_ref) * sscale), add = __builtin_amdgcn_exp2f((m_its - m_ref) * sscale);
            m_run = m;
            l_run = l_run * keep + its[(16 * DB + 1) * NT] * add;
#pragma unroll
            for (int db = 0; db < DB; db++)
#pragma unroll
                for (int r = 0; r < 16; r++) acc[db][r] = acc[db][r] * keep + its[(16 * db + r) * NT] * add;
        }
    }
    // rows to be done by themselves: some dim is NaN though the weights are not
    float sums[4] = { 0.f, 0.f, 0.f, 0.f };
#pragma unroll
    for (int db = 0; db < DB; db++)
#pragma unroll
        for (int r = 0; r < 16; r++) sums[r & 3] += acc[db][r];
    const float sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    const unsigned long long nan = __ballot(has_row && sum != sum && l_run == l_run);
    uint32_t again = (uint32_t)nan | (uint32_t)(nan >> 32);
    const float inv = l_run == 0.f ? 0.f : 1.0f / l_run;
    // register r of block db is dim 32 db + 8 (r / 4) + 4 hh + r % 4
    if (has_row && !((again >> j) & 1)) {
#pragma unroll
        for (int db = 0; db < DB; db++)
#pragma unroll
            for (int g = 0; g < 4; g++)
                *reinterpret_cast<float4 *>(orow + 32 * db + 8 * g + 4 * hh) =
                    make_float4(acc[db][4 * g] * inv, acc[db][4 * g + 1] * inv, acc[db][4 * g + 2] * inv, acc[db][4 * g + 3] * inv);
    }
    for (; again; again &= again - 1) {
        int t, h;
        const int n = place(32 * wave + __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)again) - 1), t, h);
        attend_row<HD>(p, a.q + (size_t)(t0 + t) * a.q_ld + (size_t)(kvh * a.group + h) * HD, a.out + (size_t)(t0 + t) * a.out_ld + (size_t)(kvh * a.group + h) * HD, seq, kvh, n);
    }
}

}  // namespace

namespace {
template <int HD, int W, int S>
hipError_t run_prefill(hipStream_t s, const PrefillArgs &a) {
    const dim3 grid((unsigned)a.p.n_kv, (unsigned)((long long)a.n_tok * a.group / (32 * W) + a.p.n_seq));
    const size_t lds = prefill_lds_bytes<HD, W, S>();
    paged_prefill_kernel<HD, W, S><<<grid, 64 * W * S, lds, s>>>(a);
    return hipGetLastError();
}
}  // namespace

hipError_t launch_paged_prefill(hipStream_t s, const PagedView &p, int head_dim, int n_tok, const float *q, size_t q_ld, int n_heads, float *out, size_t out_ld) {
    const PrefillArgs a{ p, q, out, q_ld, out_ld, n_tok, n_heads, n_heads / p.n_kv };
    // 128 rows a workgroup and two of those per compute unit read the keys least often; with fewer than two and a half such workgroups
    // per compute unit, 64 rows and two groups of waves that share the positions end sooner (32 heads of 128, one prompt; us):
    //   tokens          64   256   512  1024  2048  3000  4096  6000
    //   128 rows       9.1  19.5  30.7  51.4   100   172   303   583
    //   64 rows, two   9.8  15.1  22.4  38.2    96   185   323   666
    // Heads of 64 take half the registers and LDS, and the smaller form throughout (16 heads, 6000 tokens: 192 us, 194 with 128 rows).
    if (head_dim == 64) return run_prefill<64, 2, 2>(s, a);
    if ((long long)n_tok * a.group / 128 * p.n_kv >= 640) return run_prefill<128, 4, 1>(s, a);
    return run_prefill<128, 2, 2>(s, a);
}

}  // namespace rt
