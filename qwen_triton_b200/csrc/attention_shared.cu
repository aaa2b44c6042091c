// Attention of one query token per sequence where groups of sequences hold the same first pages of the cache: the shared keys and values of a
// group are taken once for all of its members.
//
//   o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),   s_j = scale q k_j,  m = max_j s_j
//
// A range of keys leaves (m, l, a) = (max s, sum e^(s - m), sum e^(s - m) v); ranges join by m* = max m, l* = sum l e^(m - m*), a* likewise.
// The positions below a group's shared length are one walk for the rows (member, query head) of a kv head, cut into ranges; the positions from
// there on are each member's own.
#include "tc_common.cuh"

#include <math.h>

using namespace qt;
using namespace qt_tc;

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
    int own_warps;                              // warps a block of the own keys' kernel
    int* status;                                // stays 0 unless a wait in a kernel ran out
};

// Group g of the call, held within what the member list and the page lists have.
struct Group { int first, count, shared; };
__device__ __forceinline__ Group group_at(const SharedParams& p, int g) {
    Group r;
    r.first = max(0, min(p.share[3 * g], p.n_seqs));
    r.count = max(0, min(p.share[3 * g + 1], p.n_seqs - r.first));
    r.shared = max(0, min(p.share[3 * g + 2], p.max_blocks * p.page));
    return r;
}

// The shared tokens of the group that place `at` of the member list belongs to, and the group's first member.
__device__ __forceinline__ Group group_of(const SharedParams& p, int at) {
    for (int i = 0; i < p.n_groups; ++i) {
        const Group group = group_at(p, i);
        if (at >= group.first && at < group.first + group.count) return group;
    }
    return Group{at, 1, 0};
}
__device__ __forceinline__ int member_at(const SharedParams& p, int at) { return min(max(p.members[at], 0), p.n_seqs - 1); }
__device__ __forceinline__ int page_at(const SharedParams& p, const int* table, int index) { return min(max(table[index], 0), p.n_pages - 1); }

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
    const Group group = group_of(p, at);
    const int seq = member_at(p, at);
    const int len = max(0, min(p.seq_len[seq], p.max_blocks * p.page));
    const int shared = min(group.shared, len);
    const int kvh = head / (p.nq / p.nkv);
    const bool of_group = range < p.shared_ranges;
    const int* table = p.block_table + (size_t)(of_group ? member_at(p, group.first) : seq) * p.max_blocks;
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
        const int page = page_at(p, table, j / p.page);
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
        ((T*)p.out)[row * p.d + c] = from_float<T>(l == 0.f ? 0.f : a / l);
    }
}

// ----------------------------------------------------------------------------- bfloat16, heads of up to 128 elements, pages of 64
// Two launches.  The first takes the shared keys of a group on tcgen05: a block has 128 of the rows (member, query head) of a kv head as the M of
// its products and walks a range of the pages,
//
//   S = Q K^T    Q and K in shared memory (K by TMA, 128-byte swizzle), S in tensor memory
//   P = 2^(S - m) as bfloat16 (the type of the values it is multiplied with), written over its scores in tensor memory
//   O += P V     P from tensor memory, V as an MN-major operand, O in tensor memory over the whole range
//
// one thread a row, so that maxima and sums need no exchange; O is rescaled only where a row's maximum moved by more than 2^8.  The second launch takes
// every member's own keys on mma.sync (the heads of a kv group are the 16 rows), a range a warp, and joins them with the first one's partial results.
constexpr int PAGE = 64;
constexpr int BQ = 128;
constexpr int TC_THREADS = 224;      // warp 0: TMA of K, warp 1: MMA and tensor memory, warps 2..5: Q and softmax, warp 6: TMA of V
constexpr float LOG2E = 1.4426950408889634f;
constexpr float RESCALE_STEP = 8.f;
constexpr uint32_t HALF_BYTES = BQ * 128;         // [128 rows][64 columns]
constexpr uint32_t KEY_HALF_BYTES = PAGE * 128;   // [64 keys][64 columns]

__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ uint64_t pair_f32(float lo, float hi) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
    return d;
}
__device__ __forceinline__ uint64_t pair_u32(uint32_t lo, uint32_t hi) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(hi));
    return d;
}
__device__ __forceinline__ void unpair_f32(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ void store_shared16(uint32_t addr, uint4 v) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// MN-major operand stored as [64-element MN blocks][K rows][64 elements], 128-byte swizzle (V: [key][dim]).
__device__ __forceinline__ uint64_t operand_desc_mn(uint32_t saddr, uint32_t mn_block_bytes) {
    uint64_t d = 0;
    d |= (uint64_t)((saddr & 0x3ffffu) >> 4);
    d |= (uint64_t)((mn_block_bytes >> 4) & 0x3fffu) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}

// Ranges of a group's shared pages: `per` pages each but the last; ranges from `used` on hold nothing and leave no partial result.
struct Ranges {
    int per, used;
    __device__ __forceinline__ Ranges(int tokens, int tile, int ranges) {
        const int tiles = (tokens + tile - 1) / tile;
        per = (tiles + ranges - 1) / ranges;
        used = per > 0 ? (tiles + per - 1) / per : 0;
    }
};

template <int HD>
__global__ void __launch_bounds__(TC_THREADS, 2) shared_prefix_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                                                                         const SharedParams p) {
    constexpr int HALVES = HD / 64;
    constexpr uint32_t Q_BYTES = HALVES * HALF_BYTES;
    constexpr uint32_t KV_BYTES = HALVES * KEY_HALF_BYTES;
    constexpr uint32_t TMEM_COLS = 256, O_COL = 2 * PAGE;
    constexpr uint32_t IDESC_QK = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(PAGE >> 3) << 17) | ((uint32_t)(BQ >> 4) << 24);
    constexpr uint32_t IDESC_PV = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(BQ >> 4) << 24);

    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    uint8_t* smem = smem_raw + (base - raw);
    const uint32_t q_s = base, k_s = q_s + Q_BYTES, v_s = k_s + 2 * KV_BYTES, bars = v_s + 2 * KV_BYTES;
    const uint32_t q_full = bars, k_full = bars + 8, k_empty = bars + 24, v_full = bars + 40, v_empty = bars + 56;
    const uint32_t s_full = bars + 72, p_full = bars + 88, pv_full = bars + 104;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + (bars - base) + 128);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int* status = p.status;

    if (threadIdx.x == 0) {
        prefetch_tensor_map(&map_k);
        prefetch_tensor_map(&map_v);
        mbar_init(q_full, 4);
        for (int i = 0; i < 2; ++i) {
            mbar_init(k_full + 8 * i, 1); mbar_init(k_empty + 8 * i, 1);
            mbar_init(v_full + 8 * i, 1); mbar_init(v_empty + 8 * i, 1);
            mbar_init(s_full + 8 * i, 1); mbar_init(p_full + 8 * i, 4);
            mbar_init(pv_full + 8 * i, 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_wait();
    const Group group = group_at(p, blockIdx.z);
    const int per = p.nq / p.nkv;
    const int kvh = blockIdx.y % p.nkv, row0 = blockIdx.y / p.nkv * BQ;
    const int rows = min(BQ, group.count * per - row0);
    const Ranges ranges(group.shared, PAGE, p.shared_ranges);
    const int tile_begin = (int)blockIdx.x * ranges.per;
    const int n_tiles = min(ranges.per, (group.shared + PAGE - 1) / PAGE - tile_begin);
    if (rows <= 0 || n_tiles <= 0) return;                    // uniform for the block, before tensor memory is taken
    const int* table = p.block_table + (size_t)member_at(p, group.first) * p.max_blocks;
    auto row_of_tile = [&](int j) { return (page_at(p, table, tile_begin + j) * p.nkv + kvh) * PAGE; };

    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    // The next kernel may start once every block is here.  Kernels before this one have then finished, so that it may read what they wrote ahead of
    // its own wait, which is for this kernel's partial results; and this kernel's tensor memory is taken, so that no later kernel can hold it
    // while it waits for this one.
    pdl_launch_dependents();

    if (warp == 0) {
        if (lane == 0) {
            for (int j = 0; j < n_tiles; ++j) {
                const int s = j & 1, row = row_of_tile(j);
                if (!mbar_wait(k_empty + 8 * s, ((uint32_t)(j >> 1) & 1u) ^ 1u, status, 1)) break;
                mbar_expect_tx(k_full + 8 * s, KV_BYTES);
                for (int h = 0; h < HALVES; ++h) tma_load_2d(k_s + s * KV_BYTES + h * KEY_HALF_BYTES, &map_k, k_full + 8 * s, h * 64, row);
            }
        }
    } else if (warp == 6) {
        for (int j = 0; j < n_tiles; ++j) {
            const int s = j & 1, row = row_of_tile(j);
            const int visible = min(PAGE, group.shared - (tile_begin + j) * PAGE);
            bool ok = true;
            if (lane == 0) ok = mbar_wait(v_empty + 8 * s, ((uint32_t)(j >> 1) & 1u) ^ 1u, status, 1);
            if (!__shfl_sync(0xffffffffu, (int)ok, 0)) break;
            if (visible == PAGE) {
                if (lane == 0) {
                    mbar_expect_tx(v_full + 8 * s, KV_BYTES);
                    for (int h = 0; h < HALVES; ++h) tma_load_2d(v_s + s * KV_BYTES + h * KEY_HALF_BYTES, &map_v, v_full + 8 * s, h * 64, row);
                }
            } else {
                // the page in which the shared tokens end: what lies behind them has weight zero and may be anything, infinities and NaN among
                // them, so zeros take its place
                const __nv_bfloat16* src = (const __nv_bfloat16*)p.v_cache + (size_t)row * p.d;
                for (int i = lane; i < PAGE * HD / 8; i += 32) {
                    const int key = i / (HD / 8), c = i % (HD / 8);
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (key < visible && c * 8 < p.d) v = *reinterpret_cast<const uint4*>(src + (size_t)key * p.d + c * 8);
                    store_shared16(v_s + s * KV_BYTES + (c >> 3) * KEY_HALF_BYTES + key * 128 + (((c & 7) ^ (key & 7)) << 4), v);
                }
                fence_async_shared();
                __syncwarp();
                if (lane == 0) mbar_arrive(v_full + 8 * s);
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            const uint64_t q_desc0 = operand_desc(q_s), k_desc0 = operand_desc(k_s), v_desc0 = operand_desc_mn(v_s, KEY_HALF_BYTES);
            bool ok = mbar_wait(q_full, 0, status, 2);
            auto issue_qk = [&](int i) {
                const int s = i & 1;
                if (!mbar_wait(k_full + 8 * s, (uint32_t)(i >> 1) & 1u, status, 2)) return false;
                // this buffer held P of tile i - 2, whose P V was issued before this; the tensor pipe runs its instructions in order
                tc_fence_after();
                const uint64_t k_desc = k_desc0 + (uint64_t)(s * (KV_BYTES >> 4));
#pragma unroll
                for (int ks = 0; ks < HD / 16; ++ks) {
                    const uint32_t in_half = (uint32_t)(ks & 3) * 32u;
                    umma_bf16(tmem_base + s * PAGE, q_desc0 + (uint64_t)(((uint32_t)(ks >> 2) * HALF_BYTES + in_half) >> 4),
                              k_desc + (uint64_t)(((uint32_t)(ks >> 2) * KEY_HALF_BYTES + in_half) >> 4), IDESC_QK, ks > 0 ? 1u : 0u);
                }
                umma_commit(s_full + 8 * s);
                umma_commit(k_empty + 8 * s);
                return true;
            };
            if (ok) ok = issue_qk(0);
            for (int j = 0; j < n_tiles && ok; ++j) {
                if (j + 1 < n_tiles) { ok = issue_qk(j + 1); if (!ok) break; }
                const int s = j & 1;
                const uint32_t phase = (uint32_t)(j >> 1) & 1u;
                if (!mbar_wait(p_full + 8 * s, phase, status, 2) || !mbar_wait(v_full + 8 * s, phase, status, 2)) break;
                tc_fence_after();
                const uint64_t v_desc = v_desc0 + (uint64_t)(s * (KV_BYTES >> 4));
#pragma unroll
                for (int ks = 0; ks < PAGE / 16; ++ks)
                    umma_bf16_a_tmem(tmem_base + O_COL, tmem_base + s * PAGE + (uint32_t)(ks * 8), v_desc + (uint64_t)(((uint32_t)ks * (16 * 128)) >> 4),
                                     IDESC_PV, (j > 0 || ks > 0) ? 1u : 0u);
                umma_commit(pv_full + 8 * s);
                umma_commit(v_empty + 8 * s);
            }
        }
    } else {
        const int quarter = warp & 3;
        const int r = quarter * 32 + lane;                     // this thread's row = its tensor-memory lane
        const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16);
        const bool live = r < rows, idle = quarter * 32 >= rows;    // an idle warp's rows of P are whatever is there, and go nowhere
        const int at = row0 + (live ? r : 0);
        const int seq = member_at(p, group.first + at / per), head = kvh * per + at % per;
        const int limit = live ? min(group.shared, p.seq_len[seq]) : 0;      // keys this row sees
        const float scale2 = p.scale * LOG2E;
        {
            const uint4* src = reinterpret_cast<const uint4*>((const __nv_bfloat16*)p.q + ((size_t)seq * p.nq + head) * p.d);
            uint4 v[HD / 8];
#pragma unroll
            for (int c = 0; c < HD / 8; ++c) v[c] = live && c * 8 < p.d ? src[c] : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int c = 0; c < HD / 8; ++c) store_shared16(q_s + (c >> 3) * HALF_BYTES + r * 128 + (((c & 7) ^ (r & 7)) << 4), v[c]);
            fence_async_shared();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
        }
        float m_run = -INFINITY, l_run = 0.f;                  // the maximum this row scales by (base 2) and its sum
        bool ok = true;
        for (int j = 0; j < n_tiles; ++j) {
            const int s = j & 1;
            ok = __all_sync(0xffffffffu, mbar_wait(s_full + 8 * s, (uint32_t)(j >> 1) & 1u, status, 3));      // the warp is together from here on
            if (!ok) break;
            if (idle) {
                if (lane == 0) mbar_arrive(p_full + 8 * s);
                continue;
            }
            tc_fence_after();
            const uint32_t s_addr = lane_addr + s * PAGE;
            uint32_t v[2][32];
            tmem_load32_start(s_addr, v[0]);
            tmem_load32_start(s_addr + 32, v[1]);
            tmem_wait_ld();
            const int seen = limit - (tile_begin + j) * PAGE;  // keys of this tile that the row sees
            if (seen < PAGE) {
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int c = 0; c < 32; ++c)
                        if (q * 32 + c >= seen) v[q][c] = 0xff800000u;
            }
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int c = 0; c < 32; c += 2) mx[(c >> 1) & 3] = max3(mx[(c >> 1) & 3], __uint_as_float(v[q][c]), __uint_as_float(v[q][c + 1]));
            const float m_tile = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale2;
            const bool moves = m_tile > m_run + RESCALE_STEP;
            const float m_new = moves ? m_tile : m_run;
            const float m_use = m_new == -INFINITY ? 0.f : m_new;
            const float alpha = moves ? fast_exp2(m_run - m_use) : 1.f;
            if (j > 0 && __any_sync(0xffffffffu, moves)) {
                // P V up to tile j - 2 is complete, since the scores of tile j exist; O may be scaled once that of tile j - 1 is
                ok = __all_sync(0xffffffffu, mbar_wait(pv_full + 8 * (s ^ 1), (uint32_t)((j - 1) >> 1) & 1u, status, 3));
                if (!ok) break;
                tc_fence_after();
#pragma unroll 1
                for (int c0 = 0; c0 < HD; c0 += 32) {
                    uint32_t o[32];
                    tmem_load32(lane_addr + O_COL + (uint32_t)c0, o);
#pragma unroll
                    for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * alpha);
                    tmem_store32(lane_addr + O_COL + (uint32_t)c0, o);
                }
                tmem_wait_st();
            }
            uint64_t sum2[2] = {0ull, 0ull};
            const uint64_t scale22 = pair_f32(scale2, scale2), neg_m2 = pair_f32(-m_use, -m_use);
            uint32_t packed[32];
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int c = 0; c < 32; c += 2) {
                    float x0, x1;
                    unpair_f32(fma2(pair_u32(v[q][c], v[q][c + 1]), scale22, neg_m2), x0, x1);
                    const float e0 = fast_exp2(x0), e1 = fast_exp2(x1);
                    sum2[(c >> 1) & 1] = add2(sum2[(c >> 1) & 1], pair_f32(e0, e1));
                    packed[q * 16 + (c >> 1)] = pack_bf16(e0, e1);
                }
            tmem_store32(s_addr, packed);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + 8 * s);
            float sum[4];
            unpair_f32(sum2[0], sum[0], sum[2]);
            unpair_f32(sum2[1], sum[1], sum[3]);
            l_run = l_run * alpha + (sum[0] + sum[1]) + (sum[2] + sum[3]);
            m_run = m_new;
        }
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(pv_full + 8 * ((n_tiles - 1) & 1), (uint32_t)((n_tiles - 1) >> 1) & 1u, status, 3));
        if (ok && !idle) {
            tc_fence_after();
            const size_t slot = ((size_t)seq * p.nq + head) * (p.shared_ranges + p.own_ranges) + blockIdx.x;
            float* dst = p.part_acc + slot * p.d;
#pragma unroll 1
            for (int c0 = 0; c0 < HD; c0 += 32) {
                uint32_t o[32];
                tmem_load32(lane_addr + O_COL + (uint32_t)c0, o);
                if (live) {
#pragma unroll
                    for (int c = 0; c < 32; c += 8)
                        if (c0 + c < p.d) {
                            *reinterpret_cast<uint4*>(dst + c0 + c) = make_uint4(o[c], o[c + 1], o[c + 2], o[c + 3]);
                            *reinterpret_cast<uint4*>(dst + c0 + c + 4) = make_uint4(o[c + 4], o[c + 5], o[c + 6], o[c + 7]);
                        }
                }
            }
            if (live) *reinterpret_cast<float2*>(p.part_ml + 2 * slot) = make_float2(m_run, l_run);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (*(volatile int*)status != 0) {                         // a wait gave up: let copies in flight land before the block leaves
        const unsigned long long t0 = global_timer();
        while (global_timer() - t0 < 2000000ull) __nanosleep(1000);
    }
    __syncwarp();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
}

// A member's own keys: the blocks of (16 query heads of a kv head, member) are a cluster along x, every warp of theirs walks tiles of 32 keys through a
// two-stage cp.async ring of its own, rows behind the last key filled with zeros.  Then the blocks hand their sums to the first one, which joins them with
// the shared ranges' and writes the result.
constexpr int OWN_TILE = 32;
constexpr int OWN_MAX_WARPS = 4;

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool take) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int HD> __host__ __device__ constexpr uint32_t own_tile_bytes() { return OWN_TILE * HD * 2; }
// Q; the warps' rings, where their sums go later; the cluster's inbox in the first block; what a row's partial results are multiplied by
template <int HD> __host__ __device__ constexpr uint32_t own_rings(int warps) { return (uint32_t)warps * 4 * own_tile_bytes<HD>(); }
template <int HD> constexpr size_t own_smem(int warps, int ranges, int rows) {
    return 16 * HD * 2 + own_rings<HD>(warps) + (ranges > 1 ? (size_t)ranges * rows * (HD + 4) * 4 : 0) + (size_t)16 * (MAX_RANGES + 8) * 4;
}

template <int HD>
__global__ void __launch_bounds__(32 * OWN_MAX_WARPS) shared_own_kernel(const SharedParams p) {
    constexpr int CHUNKS = HD / 8;                             // 16-byte pieces of a row
    constexpr uint32_t ROW = HD * 2, TILE = own_tile_bytes<HD>();
    extern __shared__ __align__(128) uint8_t smem_raw[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3, threads = blockDim.x, warps = threads >> 5;
    if (gridDim.x > 1) cluster_arrive_started();
    pdl_launch_dependents();
    const int per = p.nq / p.nkv, heads16 = (per + 15) / 16;
    const int kvh = blockIdx.y / heads16, h0 = blockIdx.y % heads16 * 16;
    const int rows = min(16, per - h0), head0 = kvh * per + h0;
    const int seq = member_at(p, blockIdx.z), shared = group_of(p, blockIdx.z).shared;
    const int len = max(0, min(p.seq_len[seq], p.max_blocks * PAGE));
    const int* table = p.block_table + (size_t)seq * p.max_blocks;
    const int first_tile = min(shared, len) / OWN_TILE;
    const int own_tiles = len > shared ? (len + OWN_TILE - 1) / OWN_TILE - first_tile : 0;
    const int streams = gridDim.x * warps, stream = blockIdx.x * warps + warp;
    const int per_stream = (own_tiles + streams - 1) / streams;
    const int tile_begin = first_tile + stream * per_stream;
    const int n_tiles = max(0, min(per_stream, first_tile + own_tiles - tile_begin));

    // swizzled rows: 16-byte piece c of row r lies at piece c ^ (r & 7), so that eight rows' pieces are in eight different banks' groups
    auto place = [](uint32_t row, uint32_t c) { return row * ROW + ((c ^ (row & 7u)) << 4); };
    const uint32_t q_s = smem_u32(smem_raw), ring = q_s + 16 * ROW + warp * 4 * TILE;
    for (int i = tid; i < 16 * CHUNKS; i += threads) {
        const int r = i / CHUNKS, c = i % CHUNKS;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (r < rows && c * 8 < p.d) v = *reinterpret_cast<const uint4*>((const __nv_bfloat16*)p.q + ((size_t)seq * p.nq + head0 + r) * p.d + c * 8);
        store_shared16(q_s + place(r, c), v);
    }
    auto issue = [&](int j) {
        if (j < n_tiles) {
            const int tile = tile_begin + j, pos0 = tile * OWN_TILE;
            const int page = page_at(p, table, pos0 / PAGE);
            const size_t off = (((size_t)page * p.nkv + kvh) * PAGE + pos0 % PAGE) * p.d;
            const __nv_bfloat16 *k = (const __nv_bfloat16*)p.k_cache + off, *v = (const __nv_bfloat16*)p.v_cache + off;
            const uint32_t dst = ring + (uint32_t)(j & 1) * 2 * TILE;
#pragma unroll
            for (int i = 0; i < OWN_TILE * CHUNKS / 32; ++i) {
                const int piece = i * 32 + lane, r = piece / CHUNKS, c = piece % CHUNKS;
                const bool take = pos0 + r < len && c * 8 < p.d;
                const size_t from = take ? (size_t)r * p.d + c * 8 : 0;
                cp_async16(dst + place(r, c), k + from, take);
                cp_async16(dst + TILE + place(r, c), v + from, take);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    issue(0);
    __syncthreads();
    uint32_t qf[HD / 16][4];
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) ldmatrix_x4(qf[ks], q_s + place((lane & 7) + ((lane >> 3) & 1) * 8, ks * 2 + (lane >> 4)));

    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[HD / 8][4] = {};
    const float scale2 = p.scale * LOG2E;
    const int mi = lane >> 3;
    for (int j = 0; j < n_tiles; ++j) {
        issue(j + 1);
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        __syncwarp();
        const uint32_t k_s = ring + (uint32_t)(j & 1) * 2 * TILE, v_s = k_s + TILE;
        const int pos0 = (tile_begin + j) * OWN_TILE;
        float s[4][4] = {};
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t b[4];
                ldmatrix_x4(b, k_s + place(half * 16 + (mi >> 1) * 8 + (lane & 7), ks * 2 + (mi & 1)));
                mma_bf16(s[2 * half], qf[ks], b[0], b[1]);
                mma_bf16(s[2 * half + 1], qf[ks], b[2], b[3]);
            }
        if (pos0 < shared || pos0 + OWN_TILE > len) {
#pragma unroll
            for (int nt = 0; nt < 4; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int pos = pos0 + nt * 8 + 2 * t + (e & 1);
                    if (pos < shared || pos >= len) s[nt][e] = -INFINITY;
                }
        }
        float alpha[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            float mx = fmaxf(fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1])),
                             fmaxf(fmaxf(s[2][2 * r], s[2][2 * r + 1]), fmaxf(s[3][2 * r], s[3][2 * r + 1])));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float m_new = fmaxf(m[r], mx * scale2), m_use = m_new == -INFINITY ? 0.f : m_new;
            alpha[r] = fast_exp2(m[r] - m_use);
            m[r] = m_new;
            float sum = 0.f;
#pragma unroll
            for (int nt = 0; nt < 4; ++nt)
#pragma unroll
                for (int e = 2 * r; e < 2 * r + 2; ++e) {
                    s[nt][e] = fast_exp2(fmaf(s[nt][e], scale2, -m_use));
                    sum += s[nt][e];
                }
            l[r] = l[r] * alpha[r] + sum;                      // this thread's share of the row's sum
        }
        uint32_t pa[2][4];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            pa[half][0] = pack_bf16(s[2 * half][0], s[2 * half][1]); pa[half][1] = pack_bf16(s[2 * half][2], s[2 * half][3]);
            pa[half][2] = pack_bf16(s[2 * half + 1][0], s[2 * half + 1][1]); pa[half][3] = pack_bf16(s[2 * half + 1][2], s[2 * half + 1][3]);
        }
#pragma unroll
        for (int n2 = 0; n2 < HD / 16; ++n2) {
#pragma unroll
            for (int i = 2 * n2; i < 2 * n2 + 2; ++i) { o[i][0] *= alpha[0]; o[i][1] *= alpha[0]; o[i][2] *= alpha[1]; o[i][3] *= alpha[1]; }
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t b[4];
                ldmatrix_x4_trans(b, v_s + place(half * 16 + (mi & 1) * 8 + (lane & 7), n2 * 2 + (mi >> 1)));
                mma_bf16(o[2 * n2], pa[half], b[0], b[1]);
                mma_bf16(o[2 * n2 + 1], pa[half], b[2], b[3]);
            }
        }
        __syncwarp();                                          // the stage may be overwritten by the next issue
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();

    // the warps' sums through shared memory (the rings are free now)
    float* sums = reinterpret_cast<float*>(smem_raw + 16 * ROW);              // [warps][16][HD]
    float* sums_ml = sums + warps * 16 * HD;                                  // [warps][16][2]
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        if (t == 0) { sums_ml[(warp * 16 + g + 8 * r) * 2] = m[r]; sums_ml[(warp * 16 + g + 8 * r) * 2 + 1] = l[r]; }
    }
#pragma unroll
    for (int i = 0; i < HD / 8; ++i) {
        const int c = i * 8 + 2 * t;
        *reinterpret_cast<float2*>(sums + (warp * 16 + g) * HD + c) = make_float2(o[i][0], o[i][1]);
        *reinterpret_cast<float2*>(sums + (warp * 16 + g + 8) * HD + c) = make_float2(o[i][2], o[i][3]);
    }
    __syncthreads();
    constexpr int QUADS = HD / 4, SLOT = HD + 4;                              // a row in fours; a row of the inbox: its sums, its maximum and its sum of weights
    float* inbox = reinterpret_cast<float*>(smem_raw + 16 * ROW + own_rings<HD>(warps));       // [blocks][rows][SLOT] in the first block
    float* factors = inbox + (gridDim.x > 1 ? gridDim.x * rows * SLOT : 0);   // [16][MAX_RANGES + 8]: by what partial results are multiplied
    if (gridDim.x > 1) {
        cluster_wait_started();
        for (int i = tid; i < rows * QUADS; i += threads) {
            const int r = i / QUADS, c = i % QUADS * 4;
            float m_all = -INFINITY, l_all = 0.f;
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int w = 0; w < warps; ++w) m_all = fmaxf(m_all, sums_ml[(w * 16 + r) * 2]);
            for (int w = 0; w < warps; ++w) {
                const float f = m_all == -INFINITY ? 0.f : fast_exp2(sums_ml[(w * 16 + r) * 2] - m_all);
                const float4 v = *reinterpret_cast<const float4*>(sums + (w * 16 + r) * HD + c);
                l_all += sums_ml[(w * 16 + r) * 2 + 1] * f;
                a.x += v.x * f; a.y += v.y * f; a.z += v.z * f; a.w += v.w * f;
            }
            float* slot = inbox + (size_t)(blockIdx.x * rows + r) * SLOT;
            cluster_store_float(slot + c, 0, a.x); cluster_store_float(slot + c + 1, 0, a.y);
            cluster_store_float(slot + c + 2, 0, a.z); cluster_store_float(slot + c + 3, 0, a.w);
            if (c == 0) { cluster_store_float(slot + HD, 0, m_all); cluster_store_float(slot + HD + 1, 0, l_all); }
        }
        cluster_barrier();
    }
    pdl_wait();                                                               // the shared ranges' partial results
    if (blockIdx.x > 0) return;
    // What is left in the first block: the own partial results (the cluster's in the inbox, else the warps' sums) and the shared ranges'.
    const int own = gridDim.x > 1 ? gridDim.x : warps, used = Ranges(shared, PAGE, p.shared_ranges).used, parts = own + used;
    const int stride = p.shared_ranges + p.own_ranges;
    auto own_ml = [&](int k, int r) { return gridDim.x > 1 ? inbox + (size_t)(k * rows + r) * SLOT + HD : sums_ml + (k * 16 + r) * 2; };
    auto own_row = [&](int k, int r) { return gridDim.x > 1 ? inbox + (size_t)(k * rows + r) * SLOT : sums + (k * 16 + r) * HD; };
    for (int r = warp; r < rows; r += warps) {                                // a warp a row: the maximum over the parts, then every part's factor
        const float* ml = p.part_ml + ((size_t)seq * p.nq + head0 + r) * stride * 2;
        float m_all = -INFINITY, l_all = 0.f;
        float mk[(MAX_RANGES + 8 + 31) / 32], lk[(MAX_RANGES + 8 + 31) / 32];
#pragma unroll
        for (int i = 0; i < (MAX_RANGES + 8 + 31) / 32; ++i) {
            const int k = i * 32 + lane;
            float2 both = make_float2(-INFINITY, 0.f);
            if (k < own) { const float* at = own_ml(k, r); both = make_float2(at[0], at[1]); }
            else if (k < parts) both = *reinterpret_cast<const float2*>(ml + 2 * (k - own));
            mk[i] = both.x; lk[i] = both.y;
            m_all = fmaxf(m_all, both.x);
        }
        m_all = warp_max(m_all);
#pragma unroll
        for (int i = 0; i < (MAX_RANGES + 8 + 31) / 32; ++i) {
            mk[i] = mk[i] == -INFINITY ? 0.f : fast_exp2(mk[i] - m_all);
            l_all += lk[i] * mk[i];
        }
        l_all = warp_sum(l_all);
        const float inv = l_all == 0.f ? 0.f : 1.f / l_all;
#pragma unroll
        for (int i = 0; i < (MAX_RANGES + 8 + 31) / 32; ++i)
            if (i * 32 + lane < parts) factors[r * (MAX_RANGES + 8) + i * 32 + lane] = mk[i] * inv;
    }
    __syncthreads();
    for (int i = tid; i < rows * QUADS; i += threads) {
        const int r = i / QUADS, c = i % QUADS * 4;
        if (c >= p.d) continue;
        const size_t row = (size_t)seq * p.nq + head0 + r;
        const float* f = factors + r * (MAX_RANGES + 8);
        const float* acc = p.part_acc + row * stride * p.d + c;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        auto add = [&](float4 v, float by) {                                  // a part without a key for this row may hold anything
            if (by != 0.f) { a.x += v.x * by; a.y += v.y * by; a.z += v.z * by; a.w += v.w * by; }
        };
        for (int k = 0; k < own; ++k) add(*reinterpret_cast<const float4*>(own_row(k, r) + c), f[k]);
#pragma unroll 8
        for (int k = 0; k < used; ++k) add(*reinterpret_cast<const float4*>(acc + (size_t)k * p.d), f[own + k]);
        uint2 packed = make_uint2(pack_bf16(a.x, a.y), pack_bf16(a.z, a.w));
        *reinterpret_cast<uint2*>((__nv_bfloat16*)p.out + row * p.d + c) = packed;
    }
}

// Tensor map of the cache as rows of d bfloat16, box 64 x 64, 128-byte swizzle, zeros beyond a row's end.
int cache_map(CUtensorMap* map, const void* ptr, uint64_t rows, uint64_t d) {
    EncodeFn encode = encode_fn();
    if (!encode) QT_FAIL(QT_ERR_LAUNCH, "attention_shared: the driver does not offer cuTensorMapEncodeTiled");
    const cuuint64_t dims[2] = {d, rows}, strides[1] = {d * 2};
    const cuuint32_t box[2] = {64, PAGE}, elem[2] = {1, 1};
    const CUresult rc = encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(ptr), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS) QT_FAIL(QT_ERR_LAUNCH, "attention_shared: cuTensorMapEncodeTiled failed with %d", (int)rc);
    return QT_OK;
}

template <int HD>
int launch_tc(const SharedParams& p, int most_members, cudaStream_t stream) {
    CUtensorMap map_k, map_v;
    int rc = cache_map(&map_k, p.k_cache, (uint64_t)p.n_pages * p.nkv * PAGE, p.d);
    if (rc == QT_OK) rc = cache_map(&map_v, p.v_cache, (uint64_t)p.n_pages * p.nkv * PAGE, p.d);
    if (rc != QT_OK) return rc;
    const int per = p.nq / p.nkv;
    const size_t smem = (HD / 64) * (HALF_BYTES + 4 * KEY_HALF_BYTES) + 1024 + 192, smem_own = own_smem<HD>(p.own_warps, p.own_ranges, per < 16 ? per : 16);
    cudaError_t raised = raise_shared<shared_prefix_tc_kernel<HD>>((int)smem);
    if (raised == cudaSuccess) raised = raise_shared<shared_own_kernel<HD>>((int)smem_own);
    if (raised != cudaSuccess) QT_FAIL(QT_ERR_LAUNCH, "attention_shared: cannot raise shared memory: %s", cudaGetErrorString(raised));
    const long long tiles = ((long long)most_members * per + BQ - 1) / BQ, y_own = (long long)p.nkv * ((per + 15) / 16);
    QT_REQUIRE(tiles * p.nkv <= 65535 && y_own <= 65535 && p.n_groups <= 65535 && p.n_seqs <= 65535, "attention_shared: too many rows for one launch");
    launch_kernel(shared_prefix_tc_kernel<HD>, dim3(p.shared_ranges, (unsigned)(tiles * p.nkv), p.n_groups), dim3(TC_THREADS), smem, stream, map_k, map_v, p);
    launch_kernel_cluster(shared_own_kernel<HD>, dim3(p.own_ranges, (unsigned)y_own, p.n_seqs), dim3(32 * p.own_warps), smem_own, stream,
                          (unsigned)p.own_ranges, p);
    QT_CHECK_LAUNCH("attention_shared");
    return QT_OK;
}

}  // namespace

// on_tc: bfloat16, d % 8 == 0 and at most 128, pages of 64, own_ranges at most 8.
extern "C" int qt_attention_decode_shared(const void* q, const void* k_cache, const void* v_cache, void* out, int dtype, const int* block_table,
                                          int max_blocks, const int* seq_len, const int* members, const int* share, int n_seqs, int n_groups,
                                          int most_members, int nq, int nkv, int d, int page_tokens, int n_pages, float scale, int shared_ranges,
                                          int own_ranges, int own_warps, int on_tc, float* part_acc, float* part_ml, int* status, void* stream) {
    QT_REQUIRE(n_seqs >= 0 && n_groups > 0 && nq > 0 && nkv > 0 && nq % nkv == 0, "attention_shared: bad head counts nq=%d nkv=%d (B=%d, %d groups)", nq, nkv, n_seqs, n_groups);
    QT_REQUIRE(d > 0 && d <= MAX_DIM && page_tokens > 0 && max_blocks > 0 && n_pages > 0, "attention_shared: bad sizes d=%d page=%d", d, page_tokens);
    QT_REQUIRE((long long)max_blocks * page_tokens <= 0x7fffffffll && most_members >= 0 && most_members <= n_seqs, "attention_shared: bad sizes: %d pages a sequence, %d members",
               max_blocks, most_members);
    QT_REQUIRE(shared_ranges > 0 && own_ranges > 0 && shared_ranges + own_ranges <= MAX_RANGES, "attention_shared: %d and %d ranges", shared_ranges, own_ranges);
    QT_REQUIRE(scale > 0.f && scale < INFINITY, "attention_shared: a score scale of %g (it must be positive)", (double)scale);
    if (n_seqs == 0) return QT_OK;
    const SharedParams p{q, k_cache, v_cache, out, block_table, max_blocks, seq_len, members, share, n_seqs, n_groups, nq, nkv, d, page_tokens, n_pages,
                         scale, shared_ranges, own_ranges, part_acc, part_ml, own_warps, status};
    cudaStream_t s = (cudaStream_t)stream;
    if (on_tc) {
        QT_REQUIRE(dtype == QT_BF16 && d % 8 == 0 && d <= 128 && page_tokens == PAGE && own_ranges <= 8 && own_warps > 0 && own_warps <= OWN_MAX_WARPS && status,
                   "attention_shared: the tensor-core kernels take bfloat16, heads of up to 128 in steps of 8, pages of 64 (d=%d, pages of %d)", d, page_tokens);
        QT_REQUIRE((long long)n_pages * nkv * PAGE <= 0x7fffffffll, "attention_shared: %d pages of %d heads are beyond a tensor map", n_pages, nkv);
        QT_REQUIRE((((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out | (uintptr_t)part_acc | (uintptr_t)part_ml) & 15) == 0,
                   "attention_shared: operands must be 16-byte aligned");
        return d <= 64 ? launch_tc<64>(p, most_members, s) : launch_tc<128>(p, most_members, s);
    }
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
