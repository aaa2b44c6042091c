// Attention of one query token per sequence where groups of sequences hold the same first pages of the cache: the shared keys and values of a
// group are taken once for all of its members.
//
//   o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),   s_j = scale q k_j,  m = max_j s_j
//
// A range of keys leaves (m, l, a) = (max s, sum e^(s - m), sum e^(s - m) v); ranges join by m* = max m, l* = sum l e^(m - m*), a* likewise.
// The positions below a group's shared length are one walk for the rows (member, query head) of a kv head, cut into ranges; the positions from
// there on are each member's own.
#include "common.cuh"

#include <math.h>

using namespace qt;

namespace {

constexpr int MAX_DIM = 256;
constexpr int MAX_RANGES = 64;                  // partial results of a row

struct SharedParams {
    const void* q;                              // [n_seqs, nq, d]
    const void* k_cache;                        // [n_pages, nkv, page, d]
    const void* v_cache;
    void* out;                                  // [n_seqs, nq, d]
    const int* block_table; int max_blocks;     // [n_seqs, max_blocks]
    const int* seq_len;                         // [n_seqs]
    const int* members;                         // [n_seqs]: sequences by group
    const int* share;                           // [n_groups][3]: first place in members, members, shared tokens
    int n_seqs, n_groups, nq, nkv, d, page, n_pages;
    float scale;
    int shared_ranges, own_ranges;
    float* part_acc;                            // [n_seqs, nq, ranges, d]
    float* part_ml;                             // [n_seqs, nq, ranges, 2]
};

// The group of place `at` of the member list: (its number, its shared tokens).
__device__ __forceinline__ int group_of(const SharedParams& p, int at) {
    for (int g = 0; g < p.n_groups; ++g)
        if (at >= p.share[3 * g] && at < p.share[3 * g] + p.share[3 * g + 1]) return g;
    return -1;
}

// A warp takes a row (member, query head) and one of its key ranges.
template <typename T>
__global__ void __launch_bounds__(128) shared_simple_kernel(const SharedParams p) {
    pdl_launch_dependents();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long item = (long long)blockIdx.x * 4 + warp;
    const int ranges = p.shared_ranges + p.own_ranges;
    if (item >= (long long)p.n_seqs * p.nq * ranges) return;
    const int range = (int)(item % ranges);
    const int head = (int)(item / ranges % p.nq), at = (int)(item / ranges / p.nq);
    const int group = group_of(p, at), seq = p.members[at];
    if (seq < 0 || seq >= p.n_seqs) return;
    const int len = min(p.seq_len[seq], p.max_blocks * p.page);
    const int shared = group < 0 ? 0 : min(p.share[3 * group + 2], len);
    const int kvh = head / (p.nq / p.nkv);
    const bool of_group = range < p.shared_ranges;
    const int* table = p.block_table + (size_t)(of_group && group >= 0 ? p.members[p.share[3 * group]] : seq) * p.max_blocks;
    const int from = of_group ? 0 : shared, count = of_group ? shared : len - shared;
    const int n = of_group ? p.shared_ranges : p.own_ranges, i = of_group ? range : range - p.shared_ranges;
    const int per = (count + n - 1) / n;
    const int begin = from + min(count, i * per), end = from + min(count, (i + 1) * per);
    const T* q = (const T*)p.q + ((size_t)seq * p.nq + head) * p.d;
    float qv[MAX_DIM / 32], acc[MAX_DIM / 32];
#pragma unroll
    for (int c = 0; c < MAX_DIM / 32; ++c) { qv[c] = c * 32 + lane < p.d ? to_float(q[c * 32 + lane]) * p.scale : 0.f; acc[c] = 0.f; }
    float m = -INFINITY, l = 0.f;
    for (int j = begin; j < end; ++j) {
        const int page = table[j / p.page];
        const size_t off = (((size_t)page * p.nkv + kvh) * p.page + j % p.page) * p.d;
        float s = 0.f;
#pragma unroll
        for (int c = 0; c < MAX_DIM / 32; ++c)
            if (c * 32 + lane < p.d) s += qv[c] * to_float(((const T*)p.k_cache)[off + c * 32 + lane]);
        s = warp_sum(s);
        const float m_new = fmaxf(m, s), alpha = m == -INFINITY ? 0.f : expf(m - m_new), w = s == -INFINITY ? 0.f : expf(s - m_new);
        l = l * alpha + w;
#pragma unroll
        for (int c = 0; c < MAX_DIM / 32; ++c)
            if (c * 32 + lane < p.d) acc[c] = acc[c] * alpha + w * to_float(((const T*)p.v_cache)[off + c * 32 + lane]);
        m = m_new;
    }
    const size_t slot = ((size_t)seq * p.nq + head) * ranges + range;
    for (int c = 0; c < MAX_DIM / 32; ++c)
        if (c * 32 + lane < p.d) p.part_acc[slot * p.d + c * 32 + lane] = acc[c];
    if (lane == 0) { p.part_ml[2 * slot] = m; p.part_ml[2 * slot + 1] = l; }
}

// A block joins the ranges of a row; a row without a key is zero.
template <typename T>
__global__ void __launch_bounds__(128) shared_join_kernel(const SharedParams p) {
    pdl_launch_dependents();
    pdl_wait();
    const size_t row = blockIdx.x;
    const int ranges = p.shared_ranges + p.own_ranges;
    const float* ml = p.part_ml + row * ranges * 2;
    float m = -INFINITY;
    for (int s = 0; s < ranges; ++s) m = fmaxf(m, ml[2 * s]);
    for (int c = threadIdx.x; c < p.d; c += blockDim.x) {
        float a = 0.f, l = 0.f;
        for (int s = 0; s < ranges; ++s) {
            if (ml[2 * s] == -INFINITY) continue;
            const float f = expf(ml[2 * s] - m);
            l += ml[2 * s + 1] * f;
            a += p.part_acc[(row * ranges + s) * p.d + c] * f;
        }
        ((T*)p.out)[row * p.d + c] = from_float<T>(l > 0.f ? a / l : 0.f);
    }
}

}  // namespace

extern "C" int qt_attention_decode_shared(const void* q, const void* k_cache, const void* v_cache, void* out, int dtype, const int* block_table,
                                          int max_blocks, const int* seq_len, const int* members, const int* share, int n_seqs, int n_groups,
                                          int nq, int nkv, int d, int page_tokens, int n_pages, float scale, int shared_ranges, int own_ranges,
                                          float* part_acc, float* part_ml, void* stream) {
    QT_REQUIRE(n_seqs >= 0 && n_groups > 0 && nq > 0 && nkv > 0 && nq % nkv == 0, "attention_shared: bad head counts nq=%d nkv=%d (B=%d, %d groups)", nq, nkv, n_seqs, n_groups);
    QT_REQUIRE(d > 0 && d <= MAX_DIM && page_tokens > 0 && max_blocks > 0 && n_pages > 0, "attention_shared: bad sizes d=%d page=%d", d, page_tokens);
    QT_REQUIRE(shared_ranges > 0 && own_ranges > 0 && shared_ranges + own_ranges <= MAX_RANGES, "attention_shared: %d and %d ranges", shared_ranges, own_ranges);
    if (n_seqs == 0) return QT_OK;
    const SharedParams p{q, k_cache, v_cache, out, block_table, max_blocks, seq_len, members, share, n_seqs, n_groups, nq, nkv, d, page_tokens, n_pages,
                         scale, shared_ranges, own_ranges, part_acc, part_ml};
    cudaStream_t s = (cudaStream_t)stream;
    const long long items = (long long)n_seqs * nq * (shared_ranges + own_ranges);
    QT_REQUIRE(items / 4 < 0x7fffffffll, "attention_shared: too many rows for one launch");
    return QT_DISPATCH_DTYPE(dtype, "attention_shared", {
        launch_kernel(shared_simple_kernel<T>, dim3((unsigned)((items + 3) / 4)), dim3(128), 0, s, p);
        launch_kernel(shared_join_kernel<T>, dim3((unsigned)(n_seqs * nq)), dim3(128), 0, s, p);
        QT_CHECK_LAUNCH("attention_shared");
        return QT_OK;
    });
}

QT_DEFINE_LAST_ERROR(attention_shared)
