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
    int* status;                                // stays 0 unless a wait in a kernel ran out
    int row_tiles, own_tiles, shared_items, own_items, turn;        // filled in at the launch
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

// Ranges of a group's shared tiles: `per` tiles each but the last; ranges from `used` on hold nothing and leave no partial result.
struct Ranges {
    int per, used;
    __device__ __forceinline__ Ranges(int tokens, int tile, int ranges) {
        const int tiles = (tokens + tile - 1) / tile;
        per = (tiles + ranges - 1) / ranges;
        used = per > 0 ? (tiles + per - 1) / per : 0;
    }
};

// The ranges of a member's own keys, in tiles from the one on in which the shared keys end.
struct OwnRanges {
    int tile, tile0, per, used, shared, len;
    __device__ __forceinline__ OwnRanges(int tile_, int shared_, int len_, int ranges) : tile(tile_), shared(shared_), len(len_) {
        tile0 = shared / tile;
        const int tiles = len > shared ? (len + tile - 1) / tile - tile0 : 0;
        per = (tiles + ranges - 1) / ranges;
        used = per > 0 ? (tiles + per - 1) / per : 0;
    }
    __device__ __forceinline__ int begin(int i) const { return max(shared, (tile0 + i * per) * tile); }
    __device__ __forceinline__ int end(int i) const { return min(len, (tile0 + (i + 1) * per) * tile); }
};

// ----------------------------------------------------------------------------- any element type, heads of up to 256 elements, any page size
// A block has up to 32 rows (member, query head) of a kv head, of all members over a range of the group's shared keys or of one member over a range of its own,
// and walks the range 32 keys at a time through shared memory, as floats, the next tile's loads under way meanwhile.  Eight lanes have a row, a sixteenth or
// more of the dims each; where there are fewer rows, several groups of lanes share one's keys, each with a maximum, a sum and sums of its own, which meet at the
// end.  Five sequences of 900 shared and 60 own keys in float, 16 heads over 8 of 128: 22 us (a warp a row and range, a key at a time, 78 us).
constexpr int ANY_TILE = 32;
constexpr int ANY_THREADS = 256;
constexpr int ANY_ROWS = ANY_THREADS / 8;

template <typename T> __device__ __forceinline__ float4 load4(const T* p);
template <> __device__ __forceinline__ float4 load4<float>(const float* p) { return *reinterpret_cast<const float4*>(p); }
template <> __device__ __forceinline__ float4 load4<__nv_bfloat16>(const __nv_bfloat16* p) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v.x)), b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v.y));
    return make_float4(a.x, a.y, b.x, b.y);
}

inline size_t any_smem(int dims) { return (size_t)2 * ANY_TILE * (dims + 4) * sizeof(float); }

// FOURS: fours of dims a lane has, d <= 32 FOURS
template <typename T, int FOURS>
__global__ void __launch_bounds__(ANY_THREADS) shared_any_kernel(const SharedParams p) {
    pdl_wait();
    pdl_launch_dependents();
    extern __shared__ __align__(16) float any_tile[];
    constexpr int DIMS = 32 * FOURS, PITCH = DIMS + 4;
    float* k_s = any_tile;                                     // [ANY_TILE][PITCH]
    float* v_s = any_tile + ANY_TILE * PITCH;
    const int per = p.nq / p.nkv, ranges_all = p.shared_ranges + p.own_ranges;
    int index = blockIdx.x;
    const bool of_group = index < p.shared_items;
    if (!of_group) index -= p.shared_items;
    const int tiles = of_group ? p.row_tiles : p.own_tiles, n_ranges = of_group ? p.shared_ranges : p.own_ranges;
    const int row0 = index % tiles * ANY_ROWS, kvh = index / tiles % p.nkv, at = index / tiles / p.nkv / n_ranges;
    int range = index / tiles / p.nkv % n_ranges, rows, begin, end, first;
    if (of_group) {
        const Group group = group_at(p, at);
        const Ranges cut(group.shared, ANY_TILE, n_ranges);
        rows = min(ANY_ROWS, group.count * per - row0);
        begin = range * cut.per * ANY_TILE;
        end = min(group.shared, begin + cut.per * ANY_TILE);
        first = group.first;
    } else {
        const OwnRanges cut(ANY_TILE, group_of(p, at).shared, max(0, min(p.seq_len[member_at(p, at)], p.max_blocks * p.page)), n_ranges);
        rows = min(ANY_ROWS, per - row0);
        begin = cut.begin(range);
        end = cut.end(range);
        first = at;
        range += p.shared_ranges;
    }
    if (rows <= 0 || begin >= end) return;
    const int* table = p.block_table + (size_t)member_at(p, first) * p.max_blocks;
    int width = 1;                                             // rows, rounded up to a power of two: groups of lanes g, g + width, ... have row g
    while (width < rows) width *= 2;
    const int group = threadIdx.x >> 3, lane = threadIdx.x & 7, share = group / width, shares = ANY_ROWS / width, row = group % width;
    const bool live = row < rows;
    const int place = row0 + (live ? row : 0);
    const int seq = member_at(p, of_group ? first + place / per : first), head = kvh * per + (of_group ? place % per : place);
    const int limit = live ? min(end, p.seq_len[seq]) : 0;
    // fours of a row start on boundaries of theirs
    const bool wide = p.d % 4 == 0 && (((uintptr_t)p.q | (uintptr_t)p.k_cache | (uintptr_t)p.v_cache) & (4 * sizeof(T) - 1)) == 0;
    auto four = [&](const void* base, size_t row_at, int c) {  // dims c to c + 3 of a row, zeros beyond its end
        const T* at_row = (const T*)base + row_at;
        if (wide && c < p.d) return load4<T>(at_row + c);
        return make_float4(c < p.d ? to_float(at_row[c]) : 0.f, c + 1 < p.d ? to_float(at_row[c + 1]) : 0.f, c + 2 < p.d ? to_float(at_row[c + 2]) : 0.f,
                           c + 3 < p.d ? to_float(at_row[c + 3]) : 0.f);
    };
    float4 q[FOURS], o[FOURS];
#pragma unroll
    for (int i = 0; i < FOURS; ++i) {
        q[i] = four(p.q, ((size_t)seq * p.nq + head) * p.d, 4 * (lane + 8 * i));
        q[i].x *= p.scale; q[i].y *= p.scale; q[i].z *= p.scale; q[i].w *= p.scale;
        o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float m = -INFINITY, l = 0.f;
    // a thread brings FOURS fours of keys and of values: key threadIdx.x / 8, the dims that it also computes with
    const int my_key = threadIdx.x >> 3;
    float4 next_k[FOURS], next_v[FOURS];
    auto fetch = [&](int pos0) {
        const int pos = pos0 + my_key;
        const bool take = pos >= begin && pos < end;           // whatever else lies there counts for nothing
        const size_t at_row = take ? (((size_t)page_at(p, table, pos / p.page) * p.nkv + kvh) * p.page + pos % p.page) * p.d : 0;
#pragma unroll
        for (int i = 0; i < FOURS; ++i) {
            next_k[i] = take ? four(p.k_cache, at_row, 4 * (lane + 8 * i)) : make_float4(0.f, 0.f, 0.f, 0.f);
            next_v[i] = take ? four(p.v_cache, at_row, 4 * (lane + 8 * i)) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
    };
    const int tile0 = begin / ANY_TILE * ANY_TILE;
    fetch(tile0);
    for (int pos0 = tile0; pos0 < end; pos0 += ANY_TILE) {
        __syncthreads();                                       // the tile before has been read
#pragma unroll
        for (int i = 0; i < FOURS; ++i) {
            *reinterpret_cast<float4*>(k_s + my_key * PITCH + 4 * (lane + 8 * i)) = next_k[i];
            *reinterpret_cast<float4*>(v_s + my_key * PITCH + 4 * (lane + 8 * i)) = next_v[i];
        }
        __syncthreads();
        if (pos0 + ANY_TILE < end) fetch(pos0 + ANY_TILE);
        for (int j0 = share; j0 < ANY_TILE; j0 += 4 * shares) {
            float s[4];
            float top = m;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int j = j0 + u * shares;
                s[u] = 0.f;
                if (j < ANY_TILE) {
#pragma unroll
                    for (int i = 0; i < FOURS; ++i) {
                        const float4 k = *reinterpret_cast<const float4*>(k_s + j * PITCH + 4 * (lane + 8 * i));
                        s[u] = fmaf(q[i].x, k.x, fmaf(q[i].y, k.y, fmaf(q[i].z, k.z, fmaf(q[i].w, k.w, s[u]))));
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
#pragma unroll
                for (int off = 1; off < 8; off <<= 1) s[u] += __shfl_xor_sync(0xffffffffu, s[u], off);
                const int pos = pos0 + j0 + u * shares;
                if (j0 + u * shares >= ANY_TILE || pos < begin || pos >= limit) s[u] = -INFINITY;
                top = fmaxf(top, s[u]);
            }
            const float at_top = top == -INFINITY ? 0.f : top;
            if (top > m) {
                const float alpha = expf(m - at_top);
                l *= alpha;
#pragma unroll
                for (int i = 0; i < FOURS; ++i) { o[i].x *= alpha; o[i].y *= alpha; o[i].z *= alpha; o[i].w *= alpha; }
                m = top;
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int j = j0 + u * shares;
                const float w = expf(s[u] - at_top);           // 0 of -inf
                l += w;
                if (j < ANY_TILE) {
#pragma unroll
                    for (int i = 0; i < FOURS; ++i) {
                        const float4 v = *reinterpret_cast<const float4*>(v_s + j * PITCH + 4 * (lane + 8 * i));
                        o[i].x = fmaf(w, v.x, o[i].x); o[i].y = fmaf(w, v.y, o[i].y); o[i].z = fmaf(w, v.z, o[i].z); o[i].w = fmaf(w, v.w, o[i].w);
                    }
                }
            }
        }
    }
    __syncthreads();
    float* meet = any_tile;                                    // [ANY_ROWS][PITCH]: sums, then maximum and sum of weights behind them
#pragma unroll
    for (int i = 0; i < FOURS; ++i) *reinterpret_cast<float4*>(meet + group * PITCH + 4 * (lane + 8 * i)) = o[i];
    if (lane == 0) { meet[group * PITCH + DIMS] = m; meet[group * PITCH + DIMS + 1] = l; }
    __syncthreads();
    if (!live || share > 0) return;
    float top = -INFINITY, total = 0.f;
    for (int i = 0; i < shares; ++i) top = fmaxf(top, meet[(row + i * width) * PITCH + DIMS]);
#pragma unroll
    for (int i = 0; i < FOURS; ++i) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = 0; i < shares; ++i) {
        const float* part = meet + (row + i * width) * PITCH;
        const float f = part[DIMS] == -INFINITY ? 0.f : expf(part[DIMS] - top);
        total += part[DIMS + 1] * f;
#pragma unroll
        for (int c = 0; c < FOURS; ++c) {
            const float4 v = *reinterpret_cast<const float4*>(part + 4 * (lane + 8 * c));
            o[c].x = fmaf(v.x, f, o[c].x); o[c].y = fmaf(v.y, f, o[c].y); o[c].z = fmaf(v.z, f, o[c].z); o[c].w = fmaf(v.w, f, o[c].w);
        }
    }
    const size_t slot = ((size_t)seq * p.nq + head) * ranges_all + range;
#pragma unroll
    for (int i = 0; i < FOURS; ++i) {
        const float x[4] = {o[i].x, o[i].y, o[i].z, o[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (4 * (lane + 8 * i) + e < p.d) p.part_acc[slot * p.d + 4 * (lane + 8 * i) + e] = x[e];
    }
    if (lane == 0) { p.part_ml[2 * slot] = top; p.part_ml[2 * slot + 1] = total; }
}

// ----------------------------------------------------------------------------- bfloat16, heads of up to 128 elements, pages of 64
// Two launches.  In the first a block has up to 128 rows (member, query head) of a kv head as the M of products on tcgen05 and walks a range of pages: rows of
// all members over the group's shared keys, or one member's rows over keys of its own,
//
//   S = Q K^T    Q and K in shared memory (K by TMA, 128-byte swizzle), S in tensor memory
//   P = 2^(S - m) as bfloat16 (the type of the values it is multiplied with), written over its scores in tensor memory
//   O += P V     P from tensor memory, V as an MN-major operand, O in tensor memory over the whole range
//
// one thread a row, so that maxima and sums need no exchange; O is rescaled only where a row's maximum moved by more than 2^8.  A member's own keys give an M of a
// few rows and cost the tensor cores what 128 would, which is still less than what their keys' way from memory takes.  The second launch joins the ranges.
//
// Bound by the chain of a tile (scores, their 64 exponentials a row, P, O) where rows are many, and by memory where own keys are.  Measured, 32 heads over 8 of 128:
// eight sequences of 2,048 shared and 130 own keys 12.5 us, 48 of three prompts of up to 5,000 and 700 36 us, 64 of 16,384 and 512 46 us (146 MB and 18 GFLOP: 3.2 TB/s); 128
// sequences of 64 heads, 32,000 and 600 keys, 168 to 198 us by the clock that the power limit leaves (136 GFLOP: 0.8 to 0.7 PFLOP/s).
constexpr int PAGE = 64;
constexpr int BQ = 128;
constexpr int TC_THREADS = 224;      // warp 0: TMA of K, warp 1: MMA and tensor memory, warps 2..5: Q and softmax, warp 6: TMA of V
constexpr float LOG2E = 1.4426950408889634f;
constexpr float RESCALE_STEP = 8.f;
constexpr uint32_t HALF_BYTES = BQ * 128;         // [128 rows][64 columns]
constexpr uint32_t KEY_HALF_BYTES = PAGE * 128;   // [64 keys][64 columns]
constexpr int MAX_PARTS = MAX_RANGES;

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

// The products as a whole warp meets them: all lanes go through the same instructions, so that descriptors stay in the registers that a warp has in common, and one
// lane's are carried out.  Issued by a lane that runs alone, a product takes about 100 cycles to leave, 12 of them a tile: a tile of a
// block that is alone on its SM took 0.82 us so and takes 0.68.
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t elected;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(elected));
    return elected;
}
__device__ __forceinline__ void mma_one(uint32_t tmem_d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate, uint32_t one) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(tmem_d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(one) : "memory");
}
__device__ __forceinline__ void mma_one_a_tmem(uint32_t tmem_d, uint32_t tmem_a, uint64_t b_desc, uint32_t idesc, uint32_t accumulate, uint32_t one) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(tmem_d), "r"(tmem_a), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(one) : "memory");
}
__device__ __forceinline__ void commit_one(uint32_t bar, uint32_t one) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(one) : "memory");
}

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

template <int HD>
__global__ void __launch_bounds__(TC_THREADS, 2) shared_parts_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
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
    const uint32_t q_full = bars, k_full = bars + 8, v_full = bars + 24, s_full = bars + 40, p_full = bars + 56, pv_full = bars + 72;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + (bars - base) + 128);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int* status = p.status;

    if (threadIdx.x == 0) {
        prefetch_tensor_map(&map_k);
        prefetch_tensor_map(&map_v);
        mbar_init(q_full, 4);
        for (int i = 0; i < 2; ++i) {
            mbar_init(k_full + 8 * i, 1); mbar_init(v_full + 8 * i, 1);
            mbar_init(s_full + 8 * i, 1); mbar_init(p_full + 8 * i, 4);
            mbar_init(pv_full + 8 * i, 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_wait();
    const int per = p.nq / p.nkv, stride = p.shared_ranges + p.own_ranges;
    // Blocks of shared keys and blocks of own keys take turns by as many as there are multiprocessors, so that each of these has one of either kind: the
    // first are bound by the tensor cores and the exponentials, the second by memory.
    const int turns = min(p.shared_items, p.own_items) / p.turn;
    int index = blockIdx.x;
    bool of_group;
    if (index < 2 * turns * p.turn) {
        of_group = (index / p.turn & 1) == 0;
        index = index / p.turn / 2 * p.turn + index % p.turn;
    } else {
        index -= turns * p.turn;
        of_group = index < p.shared_items;
        if (!of_group) index -= p.shared_items - turns * p.turn;
    }
    // What this block has: `rows` rows from row0 on, of a group (member by member) or of one member, the keys [begin, end) of a page list.  Neighbours in
    // the grid share keys: the row tiles of a kv head and range.
    const int tiles_here = of_group ? p.row_tiles : p.own_tiles, ranges_here = of_group ? p.shared_ranges : p.own_ranges;
    const int row0 = index % tiles_here * BQ, kvh = index / tiles_here % p.nkv, at = index / tiles_here / p.nkv / ranges_here;
    int range = index / tiles_here / p.nkv % ranges_here, rows, begin, end, first;
    if (of_group) {
        const Group group = group_at(p, at);
        const Ranges ranges(group.shared, PAGE, p.shared_ranges);
        rows = min(BQ, group.count * per - row0);
        begin = range * ranges.per * PAGE;
        end = min(group.shared, begin + ranges.per * PAGE);
        first = group.first;
    } else {
        const OwnRanges own(PAGE, group_of(p, at).shared, max(0, min(p.seq_len[member_at(p, at)], p.max_blocks * PAGE)), p.own_ranges);
        rows = min(BQ, per - row0);
        begin = own.begin(range);
        end = own.end(range);
        first = at;
        range += p.shared_ranges;
    }
    const int tile_begin = begin / PAGE, n_tiles = (end + PAGE - 1) / PAGE - tile_begin;
    if (rows <= 0 || begin >= end) return;                    // uniform for the block, before tensor memory is taken
    const int* table = p.block_table + (size_t)member_at(p, first) * p.max_blocks;
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
                // the stage's last product has been formed: its scores were there
                if (!mbar_wait(s_full + 8 * s, ((uint32_t)(j >> 1) & 1u) ^ 1u, status, 1)) break;
                mbar_expect_tx(k_full + 8 * s, KV_BYTES);
                for (int h = 0; h < HALVES; ++h) tma_load_2d(k_s + s * KV_BYTES + h * KEY_HALF_BYTES, &map_k, k_full + 8 * s, h * 64, row);
            }
        }
    } else if (warp == 6) {
        if (lane == 0) {
            for (int j = 0; j < n_tiles; ++j) {
                const int s = j & 1, row = row_of_tile(j);
                if (!mbar_wait(pv_full + 8 * s, ((uint32_t)(j >> 1) & 1u) ^ 1u, status, 1)) break;
                mbar_expect_tx(v_full + 8 * s, KV_BYTES);
                for (int h = 0; h < HALVES; ++h) tma_load_2d(v_s + s * KV_BYTES + h * KEY_HALF_BYTES, &map_v, v_full + 8 * s, h * 64, row);
            }
        }
    } else if (warp == 1) {
        const uint64_t q_desc0 = operand_desc(q_s), k_desc0 = operand_desc(k_s), v_desc0 = operand_desc_mn(v_s, KEY_HALF_BYTES);
        const uint32_t one = elect_one();
        auto wait = [&](uint32_t bar, uint32_t phase) { return __all_sync(0xffffffffu, mbar_wait(bar, phase, status, 2)) != 0; };
        auto issue_qk = [&](int i) {
            const int s = i & 1;
            if (!wait(k_full + 8 * s, (uint32_t)(i >> 1) & 1u)) return false;
            // this buffer held P of tile i - 2, whose P V was issued before this; the tensor pipe runs its instructions in order
            tc_fence_after();
            const uint64_t k_desc = k_desc0 + (uint64_t)(s * (KV_BYTES >> 4));
#pragma unroll
            for (int ks = 0; ks < HD / 16; ++ks) {
                const uint32_t in_half = (uint32_t)(ks & 3) * 32u;
                mma_one(tmem_base + s * PAGE, q_desc0 + (uint64_t)(((uint32_t)(ks >> 2) * HALF_BYTES + in_half) >> 4),
                        k_desc + (uint64_t)(((uint32_t)(ks >> 2) * KEY_HALF_BYTES + in_half) >> 4), IDESC_QK, ks > 0 ? 1u : 0u, one);
            }
            commit_one(s_full + 8 * s, one);
            return true;
        };
        bool ok = wait(q_full, 0) && issue_qk(0);
        for (int j = 0; j < n_tiles && ok; ++j) {
            if (j + 1 < n_tiles) { ok = issue_qk(j + 1); if (!ok) break; }
            const int s = j & 1;
            const uint32_t phase = (uint32_t)(j >> 1) & 1u;
            if (!wait(p_full + 8 * s, phase) || !wait(v_full + 8 * s, phase)) break;
            tc_fence_after();
            const uint64_t v_desc = v_desc0 + (uint64_t)(s * (KV_BYTES >> 4));
#pragma unroll
            for (int ks = 0; ks < PAGE / 16; ++ks)
                mma_one_a_tmem(tmem_base + O_COL, tmem_base + s * PAGE + (uint32_t)(ks * 8), v_desc + (uint64_t)(((uint32_t)ks * (16 * 128)) >> 4), IDESC_PV,
                               (j > 0 || ks > 0) ? 1u : 0u, one);
            commit_one(pv_full + 8 * s, one);
        }
    } else {
        const int quarter = warp & 3;
        const int r = quarter * 32 + lane;                     // this thread's row = its tensor-memory lane
        const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16);
        const bool live = r < rows, idle = quarter * 32 >= rows;    // an idle warp's rows of P are whatever is there, and go nowhere
        const int mine = row0 + (live ? r : 0);
        const int seq = member_at(p, of_group ? first + mine / per : first), head = kvh * per + (of_group ? mine % per : mine);
        const int limit = live ? min(end, p.seq_len[seq]) : 0;               // the row sees the keys below this
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
        float m_run = -INFINITY;                               // the maximum this row scales by (base 2)
        uint64_t sum2[2] = {0ull, 0ull};                       // its sum, in two pairs
        bool ok = true;
        for (int j = 0; j < n_tiles; ++j) {
            const int s = j & 1;
            ok = __all_sync(0xffffffffu, mbar_wait(s_full + 8 * s, (uint32_t)(j >> 1) & 1u, status, 3));      // the warp is together from here on
            if (!ok) break;
            const int pos0 = (tile_begin + j) * PAGE;
            if (pos0 < begin || pos0 + PAGE > end) {
                // A page in which the keys begin or end: what lies outside has weight zero and may be anything, infinities and NaN among them, so
                // zeros take its values' place, a quarter of the page a warp, before the product may read it.
                ok = __all_sync(0xffffffffu, mbar_wait(v_full + 8 * s, (uint32_t)(j >> 1) & 1u, status, 3));
                if (!ok) break;
                for (int i = lane; i < PAGE / 4 * (HD / 8); i += 32) {
                    const int key = quarter * (PAGE / 4) + i / (HD / 8), c = i % (HD / 8);
                    if (pos0 + key < begin || pos0 + key >= end)
                        store_shared16(v_s + s * KV_BYTES + (c >> 3) * KEY_HALF_BYTES + key * 128 + (((c & 7) ^ (key & 7)) << 4), make_uint4(0, 0, 0, 0));
                }
                fence_async_shared();
                __syncwarp();
            }
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
            if (limit - pos0 < PAGE || pos0 < begin) {
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int c = 0; c < 32; ++c)
                        if (q * 32 + c >= limit - pos0 || q * 32 + c < begin - pos0) v[q][c] = 0xff800000u;
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
            if (__any_sync(0xffffffffu, moves)) {
                const uint64_t alpha2 = pair_f32(alpha, alpha);
                sum2[0] = fma2(sum2[0], alpha2, 0ull);
                sum2[1] = fma2(sum2[1], alpha2, 0ull);
            }
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
            m_run = m_new;
        }
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(pv_full + 8 * ((n_tiles - 1) & 1), (uint32_t)((n_tiles - 1) >> 1) & 1u, status, 3));
        if (ok && !idle) {
            tc_fence_after();
            const size_t slot = ((size_t)seq * p.nq + head) * stride + range;
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
            float sum[4];
            unpair_f32(sum2[0], sum[0], sum[2]);
            unpair_f32(sum2[1], sum[1], sum[3]);
            if (live) *reinterpret_cast<float2*>(p.part_ml + 2 * slot) = make_float2(m_run, (sum[0] + sum[1]) + (sum[2] + sum[3]));
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

// What rows' partial results are multiplied by: row r of `rows` has `parts` of them, ml(r, k) their maximum and sum; a warp a row.
template <bool BASE2, typename ML>
__device__ __forceinline__ void part_factors(float* factors, int rows, int parts, int warp, int warps, int lane, ML ml) {
    constexpr int TURNS = (MAX_PARTS + 31) / 32;
    for (int r = warp; r < rows; r += warps) {
        float m_all = -INFINITY, l_all = 0.f, mk[TURNS], lk[TURNS];
#pragma unroll
        for (int i = 0; i < TURNS; ++i) {
            const int k = i * 32 + lane;
            const float2 both = k < parts ? ml(r, k) : make_float2(-INFINITY, 0.f);
            mk[i] = both.x; lk[i] = both.y;
            m_all = fmaxf(m_all, both.x);
        }
        m_all = warp_max(m_all);
#pragma unroll
        for (int i = 0; i < TURNS; ++i) {
            mk[i] = mk[i] == -INFINITY ? 0.f : BASE2 ? fast_exp2(mk[i] - m_all) : expf(mk[i] - m_all);
            l_all += lk[i] * mk[i];
        }
        l_all = warp_sum(l_all);
        const float inv = l_all == 0.f ? 0.f : 1.f / l_all;    // a row without a key is zero
#pragma unroll
        for (int i = 0; i < TURNS; ++i)
            if (i * 32 + lane < parts) factors[r * MAX_PARTS + i * 32 + lane] = mk[i] * inv;
    }
}
__device__ __forceinline__ void add_part(float4& a, float4 v, float by) {      // a part without a key for the row may hold anything
    if (by != 0.f) { a.x += v.x * by; a.y += v.y * by; a.z += v.z * by; a.w += v.w * by; }
}

// Joins the partial results of up to 16 query heads of a member's kv head.  TILE: what ranges are cut in; BASE2: maxima are base 2, and the exponential may be
// approximate.
constexpr int JOIN_THREADS = 128;

template <typename T, int TILE, bool BASE2>
__global__ void __launch_bounds__(JOIN_THREADS) shared_join_kernel(const SharedParams p) {
    pdl_launch_dependents();
    __shared__ float factors[16 * MAX_PARTS];
    const int tid = threadIdx.x, per = p.nq / p.nkv, heads16 = (per + 15) / 16, stride = p.shared_ranges + p.own_ranges;
    const int h0 = blockIdx.x % heads16 * 16, rows = min(16, per - h0), head0 = blockIdx.x / heads16 * per + h0;
    // The kernel before this one lets it start once each of its blocks is past its own wait: what kernels before that one wrote (lists and lengths) is there.
    const int seq = member_at(p, blockIdx.y), shared = group_of(p, blockIdx.y).shared;
    const int of_group = Ranges(shared, TILE, p.shared_ranges).used;
    const int parts = of_group + OwnRanges(TILE, shared, max(0, min(p.seq_len[seq], p.max_blocks * p.page)), p.own_ranges).used;
    pdl_wait();                                                // the partial results
    const size_t row0 = (size_t)seq * p.nq + head0;
    auto slot_of = [&](int k) { return k < of_group ? k : p.shared_ranges + k - of_group; };
    part_factors<BASE2>(factors, rows, parts, tid >> 5, JOIN_THREADS / 32, tid & 31,
                        [&](int r, int k) { return *reinterpret_cast<const float2*>(p.part_ml + 2 * ((row0 + r) * stride + slot_of(k))); });
    __syncthreads();
    if (p.d % 4) {                                             // rows that are not whole fours
        for (int i = tid; i < rows * p.d; i += JOIN_THREADS) {
            const int r = i / p.d, c = i % p.d;
            float a = 0.f;
            for (int k = 0; k < parts; ++k) {
                const float f = factors[r * MAX_PARTS + k];
                if (f != 0.f) a += p.part_acc[((row0 + r) * stride + slot_of(k)) * p.d + c] * f;
            }
            ((T*)p.out)[(row0 + r) * p.d + c] = from_float<T>(a);
        }
        return;
    }
    const int quads = p.d / 4;
    for (int i = tid; i < rows * quads; i += JOIN_THREADS) {
        const int r = i / quads, c = i % quads * 4;
        const float* acc = p.part_acc + (row0 + r) * stride * p.d + c;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
        for (int k = 0; k < parts; ++k) add_part(a, *reinterpret_cast<const float4*>(acc + (size_t)slot_of(k) * p.d), factors[r * MAX_PARTS + k]);
        T* to = (T*)p.out + (row0 + r) * p.d + c;
        to[0] = from_float<T>(a.x); to[1] = from_float<T>(a.y); to[2] = from_float<T>(a.z); to[3] = from_float<T>(a.w);
    }
}

// One warp walks keys on mma.sync, the up to 16 query heads of a kv head as the rows, 16 keys at a time through a ring of four
// stages of its own (cp.async, three tiles ahead), so that nothing in the loop waits for another warp.  Keys outside [begin, end) are zeros in shared memory:
// their weight is zero, and what lies there may be anything, infinities and NaN among them.
constexpr int WALK_TILE = 16;
constexpr int WALK_STAGES = 4;

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

template <int HD> constexpr uint32_t WALK_BYTES = WALK_STAGES * 2 * WALK_TILE * HD * 2;      // a warp's ring

// What a warp has of its rows g and g + 8 (lane = 4 g + t): maximum (base 2), this lane's share of the sum, columns 8 i + 2 t and the next.
template <int HD> struct Walked { float m[2], l[2], o[HD / 8][4]; };

// `heads` query heads from head0 on; `first`: the page list for positions below `shared`, `mine`: from there on.
template <int HD>
__device__ __forceinline__ void walk_keys(const SharedParams& p, Walked<HD>& w, int seq, int kvh, int head0, int heads, const int* first, const int* mine,
                                          int shared, int begin, int end, uint32_t ring, int lane) {
    constexpr int CHUNKS = HD / 8;                             // 16-byte pieces of a row
    constexpr uint32_t ROW = HD * 2, TILE = WALK_TILE * ROW;
    const int g = lane >> 2, t = lane & 3, mi = lane >> 3;
    // swizzled rows: piece c of row r lies at piece c ^ (r & 7), so that the pieces that eight lanes of an ldmatrix name are in different banks
    auto place = [](uint32_t row, uint32_t c) { return row * ROW + ((c ^ (row & 7u)) << 4); };
    const int tile0 = begin / WALK_TILE, n_tiles = end > begin ? (end + WALK_TILE - 1) / WALK_TILE - tile0 : 0;
    // page numbers of 32 pages at a time, one a lane: a look into the page list in front of every tile would put a round trip on its path
    int pages_from = -1, page_first = 0, page_mine = 0;
    auto issue = [&](int j) {
        if (j < n_tiles) {
            const int pos0 = (tile0 + j) * WALK_TILE, index = pos0 / PAGE;
            if (pages_from < 0 || index >= pages_from + 32) {
                pages_from = index;
                const int at = min(index + lane, p.max_blocks - 1);
                page_first = at * PAGE < shared ? page_at(p, first, at) : 0;
                page_mine = (at + 1) * PAGE > shared ? page_at(p, mine, at) : 0;
            }
            const int of_first = __shfl_sync(0xffffffffu, page_first, index - pages_from), of_mine = __shfl_sync(0xffffffffu, page_mine, index - pages_from);
            const uint32_t dst = ring + (uint32_t)(j % WALK_STAGES) * 2 * TILE;
#pragma unroll
            for (int i = 0; i < WALK_TILE * CHUNKS / 32; ++i) {
                const int piece = i * 32 + lane, r = piece / CHUNKS, c = piece % CHUNKS, pos = pos0 + r;
                const bool take = pos >= begin && pos < end && c * 8 < p.d;
                const size_t from = take ? (((size_t)(pos < shared ? of_first : of_mine) * p.nkv + kvh) * PAGE + pos % PAGE) * p.d + c * 8 : 0;
                cp_async16(dst + place(r, c), (const __nv_bfloat16*)p.k_cache + from, take);
                cp_async16(dst + TILE + place(r, c), (const __nv_bfloat16*)p.v_cache + from, take);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int j = 0; j < WALK_STAGES - 1; ++j) issue(j);
    uint32_t qf[HD / 16][4];                                   // rows g and g + 8, columns 16 ks + 2 t, + 8: as the product takes them
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int r = g + (e & 1) * 8, c = ks * 16 + (e >> 1) * 8 + 2 * t;
            qf[ks][e] = r < heads && c < p.d ? *reinterpret_cast<const uint32_t*>((const __nv_bfloat16*)p.q + ((size_t)seq * p.nq + head0 + r) * p.d + c) : 0u;
        }
#pragma unroll
    for (int r = 0; r < 2; ++r) { w.m[r] = -INFINITY; w.l[r] = 0.f; }
#pragma unroll
    for (int i = 0; i < HD / 8; ++i) w.o[i][0] = w.o[i][1] = w.o[i][2] = w.o[i][3] = 0.f;
    const float scale2 = p.scale * LOG2E;
    for (int j = 0; j < n_tiles; ++j) {
        issue(j + WALK_STAGES - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(WALK_STAGES - 1) : "memory");
        __syncwarp();
        const uint32_t k_s = ring + (uint32_t)(j % WALK_STAGES) * 2 * TILE, v_s = k_s + TILE;
        const int pos0 = (tile0 + j) * WALK_TILE;
        float s[2][4] = {};
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks) {
            uint32_t b[4];
            ldmatrix_x4(b, k_s + place((mi >> 1) * 8 + (lane & 7), ks * 2 + (mi & 1)));
            mma_bf16(s[0], qf[ks], b[0], b[1]);
            mma_bf16(s[1], qf[ks], b[2], b[3]);
        }
        if (pos0 < begin || pos0 + WALK_TILE > end) {
#pragma unroll
            for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int pos = pos0 + nt * 8 + 2 * t + (e & 1);
                    if (pos < begin || pos >= end) s[nt][e] = -INFINITY;
                }
        }
        float alpha[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            float mx = fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float m_new = fmaxf(w.m[r], mx * scale2), m_use = m_new == -INFINITY ? 0.f : m_new;
            alpha[r] = fast_exp2(w.m[r] - m_use);
            w.m[r] = m_new;
            float sum = 0.f;
#pragma unroll
            for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                for (int e = 2 * r; e < 2 * r + 2; ++e) {
                    s[nt][e] = fast_exp2(fmaf(s[nt][e], scale2, -m_use));
                    sum += s[nt][e];
                }
            w.l[r] = w.l[r] * alpha[r] + sum;
        }
        const uint32_t pa[4] = {pack_bf16(s[0][0], s[0][1]), pack_bf16(s[0][2], s[0][3]), pack_bf16(s[1][0], s[1][1]), pack_bf16(s[1][2], s[1][3])};
#pragma unroll
        for (int n2 = 0; n2 < HD / 16; ++n2) {
#pragma unroll
            for (int i = 2 * n2; i < 2 * n2 + 2; ++i) { w.o[i][0] *= alpha[0]; w.o[i][1] *= alpha[0]; w.o[i][2] *= alpha[1]; w.o[i][3] *= alpha[1]; }
            uint32_t b[4];
            ldmatrix_x4_trans(b, v_s + place((mi & 1) * 8 + (lane & 7), n2 * 2 + (mi >> 1)));
            mma_bf16(w.o[2 * n2], pa, b[0], b[1]);
            mma_bf16(w.o[2 * n2 + 1], pa, b[2], b[3]);
        }
        __syncwarp();                                          // the stage may be overwritten by the next issue
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        w.l[r] += __shfl_xor_sync(0xffffffffu, w.l[r], 1);
        w.l[r] += __shfl_xor_sync(0xffffffffu, w.l[r], 2);
    }
}

// Everything in one launch, where so little is shared that a second launch costs more than reading it again (out of the L2 cache): the blocks of (16 query
// heads of a kv head, member) are a cluster along x whose warps each walk a range of all of the member's keys; the first block joins the ranges.  Its callers are those
// of the operator alone: steps of the engine share reading from sizes on that are beyond this form.  Bound by latency: two sequences of 199 shared and 40 own keys, 16
// heads over 8, 5.2 us (about 5 us more in two launches); 20 of 1,500 and 90, 5 heads of 64, 10 us.
constexpr int DIRECT_MAX_WARPS = 6;

template <int HD> constexpr size_t direct_smem(int warps, int ranges, int rows) {
    return (size_t)warps * WALK_BYTES<HD> + (ranges > 1 ? (size_t)ranges * rows * (HD + 4) * 4 : 0) + 16 * MAX_PARTS * 4;
}

template <int HD>
__global__ void __launch_bounds__(32 * DIRECT_MAX_WARPS) shared_direct_kernel(const SharedParams p) {
    extern __shared__ __align__(128) uint8_t smem_raw[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3, threads = blockDim.x, warps = threads >> 5;
    if (gridDim.x > 1) cluster_arrive_started();
    pdl_launch_dependents();
    const int per = p.nq / p.nkv, heads16 = (per + 15) / 16;
    const int kvh = blockIdx.y / heads16, h0 = blockIdx.y % heads16 * 16;
    const int rows = min(16, per - h0), head0 = kvh * per + h0;
    pdl_wait();
    const int seq = member_at(p, blockIdx.z);
    const Group group = group_of(p, blockIdx.z);
    const int len = max(0, min(p.seq_len[seq], p.max_blocks * PAGE));
    const OwnRanges all(WALK_TILE, 0, len, gridDim.x * warps);
    const int range = blockIdx.x * warps + warp;
    Walked<HD> w;
    walk_keys<HD>(p, w, seq, kvh, head0, rows, p.block_table + (size_t)member_at(p, group.first) * p.max_blocks, p.block_table + (size_t)seq * p.max_blocks,
                  group.shared, all.begin(range), all.end(range), smem_u32(smem_raw) + warp * WALK_BYTES<HD>, lane);
    __syncthreads();

    // the warps' sums through shared memory (the rings are free now), the blocks' through the first one's inbox
    constexpr int QUADS = HD / 4, SLOT = HD + 4;                              // a row in fours; with its maximum and its sum of weights
    float* sums = reinterpret_cast<float*>(smem_raw);                         // [warps][rows][SLOT]
    float* inbox = reinterpret_cast<float*>(smem_raw + warps * WALK_BYTES<HD>);                // [blocks][rows][SLOT] in the first block
    float* factors = inbox + (gridDim.x > 1 ? gridDim.x * rows * SLOT : 0);   // [16][MAX_PARTS]
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int row = g + 8 * r;
        if (row >= rows) continue;
        float* slot = sums + (warp * rows + row) * SLOT;
#pragma unroll
        for (int i = 0; i < HD / 8; ++i) *reinterpret_cast<float2*>(slot + i * 8 + 2 * t) = make_float2(w.o[i][2 * r], w.o[i][2 * r + 1]);
        if (t == 0) *reinterpret_cast<float2*>(slot + HD) = make_float2(w.m[r], w.l[r]);
    }
    __syncthreads();
    if (gridDim.x > 1) {
        cluster_wait_started();
        for (int i = tid; i < rows * QUADS; i += threads) {
            const int r = i / QUADS, c = i % QUADS * 4;
            float m_all = -INFINITY, l_all = 0.f;
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int k = 0; k < warps; ++k) m_all = fmaxf(m_all, sums[(k * rows + r) * SLOT + HD]);
            for (int k = 0; k < warps; ++k) {
                const float* slot = sums + (k * rows + r) * SLOT;
                const float f = m_all == -INFINITY ? 0.f : fast_exp2(slot[HD] - m_all);
                l_all += slot[HD + 1] * f;
                add_part(a, *reinterpret_cast<const float4*>(slot + c), f);
            }
            float* slot = inbox + (size_t)(blockIdx.x * rows + r) * SLOT;
            cluster_store_float(slot + c, 0, a.x); cluster_store_float(slot + c + 1, 0, a.y);
            cluster_store_float(slot + c + 2, 0, a.z); cluster_store_float(slot + c + 3, 0, a.w);
            if (c == 0) { cluster_store_float(slot + HD, 0, m_all); cluster_store_float(slot + HD + 1, 0, l_all); }
        }
        cluster_barrier();
        if (blockIdx.x > 0) return;
    }
    const float* from = gridDim.x > 1 ? inbox : sums;
    const int parts = gridDim.x > 1 ? gridDim.x : warps;
    part_factors<true>(factors, rows, parts, warp, warps, lane, [&](int r, int k) { return *reinterpret_cast<const float2*>(from + (size_t)(k * rows + r) * SLOT + HD); });
    __syncthreads();
    for (int i = tid; i < rows * QUADS; i += threads) {
        const int r = i / QUADS, c = i % QUADS * 4;
        if (c >= p.d) continue;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int k = 0; k < parts; ++k) add_part(a, *reinterpret_cast<const float4*>(from + (size_t)(k * rows + r) * SLOT + c), factors[r * MAX_PARTS + k]);
        *reinterpret_cast<uint2*>((__nv_bfloat16*)p.out + ((size_t)seq * p.nq + head0 + r) * p.d + c) = make_uint2(pack_bf16(a.x, a.y), pack_bf16(a.z, a.w));
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

template <typename T, int FOURS>
int launch_any(SharedParams p, int most_members, cudaStream_t stream) {
    const size_t smem = any_smem(32 * FOURS);
    const cudaError_t raised = raise_shared<shared_any_kernel<T, FOURS>>((int)smem);
    if (raised != cudaSuccess) QT_FAIL(QT_ERR_LAUNCH, "attention_shared: cannot raise shared memory: %s", cudaGetErrorString(raised));
    const int per = p.nq / p.nkv;
    const long long tiles = ((long long)most_members * per + ANY_ROWS - 1) / ANY_ROWS, own_tiles = (per + ANY_ROWS - 1) / ANY_ROWS;
    const long long shared = tiles * p.nkv * p.shared_ranges * p.n_groups, own = own_tiles * p.nkv * p.own_ranges * p.n_seqs;
    const long long heads = (long long)p.nkv * ((per + 15) / 16);
    QT_REQUIRE(shared + own <= 0x3fffffffll && heads <= 0x7fffffffll && p.n_seqs <= 65535, "attention_shared: too many rows for one launch");
    p.row_tiles = (int)tiles; p.own_tiles = (int)own_tiles; p.shared_items = (int)shared; p.own_items = (int)own;
    launch_kernel(shared_any_kernel<T, FOURS>, dim3((unsigned)(shared + own)), dim3(ANY_THREADS), smem, stream, p);
    launch_kernel(shared_join_kernel<T, ANY_TILE, false>, dim3((unsigned)heads, p.n_seqs), dim3(JOIN_THREADS), 0, stream, p);
    QT_CHECK_LAUNCH("attention_shared");
    return QT_OK;
}

template <int HD>
int launch_parts(SharedParams p, int most_members, cudaStream_t stream) {
    CUtensorMap map_k, map_v;
    int rc = cache_map(&map_k, p.k_cache, (uint64_t)p.n_pages * p.nkv * PAGE, p.d);
    if (rc == QT_OK) rc = cache_map(&map_v, p.v_cache, (uint64_t)p.n_pages * p.nkv * PAGE, p.d);
    if (rc != QT_OK) return rc;
    const size_t smem = (HD / 64) * (HALF_BYTES + 4 * KEY_HALF_BYTES) + 1024 + 192;
    const cudaError_t raised = raise_shared<shared_parts_kernel<HD>>((int)smem);
    if (raised != cudaSuccess) QT_FAIL(QT_ERR_LAUNCH, "attention_shared: cannot raise shared memory: %s", cudaGetErrorString(raised));
    const int per = p.nq / p.nkv;
    const long long tiles = ((long long)most_members * per + BQ - 1) / BQ, own_tiles = (per + BQ - 1) / BQ, heads = (long long)p.nkv * ((per + 15) / 16);
    const long long shared = tiles * p.nkv * p.shared_ranges * p.n_groups, own = own_tiles * p.nkv * p.own_ranges * p.n_seqs;
    QT_REQUIRE(shared + own <= 0x3fffffffll && p.n_seqs <= 65535, "attention_shared: too many rows for one launch");
    p.row_tiles = (int)tiles; p.own_tiles = (int)own_tiles; p.shared_items = (int)shared; p.own_items = (int)own; p.turn = sm_count();
    launch_kernel(shared_parts_kernel<HD>, dim3((unsigned)(shared + own)), dim3(TC_THREADS), smem, stream, map_k, map_v, p);
    launch_kernel(shared_join_kernel<__nv_bfloat16, PAGE, true>, dim3((unsigned)heads, p.n_seqs), dim3(JOIN_THREADS), 0, stream, p);
    QT_CHECK_LAUNCH("attention_shared");
    return QT_OK;
}

template <int HD>
int launch_direct(const SharedParams& p, int warps, cudaStream_t stream) {
    const int per = p.nq / p.nkv;
    const size_t smem = direct_smem<HD>(warps, p.own_ranges, per < 16 ? per : 16);
    QT_REQUIRE(smem <= 227 * 1024, "attention_shared: %d blocks of %d warps want %zu bytes of shared memory a block", p.own_ranges, warps, smem);
    const cudaError_t raised = raise_shared<shared_direct_kernel<HD>>((int)smem);
    if (raised != cudaSuccess) QT_FAIL(QT_ERR_LAUNCH, "attention_shared: cannot raise shared memory: %s", cudaGetErrorString(raised));
    const long long heads = (long long)p.nkv * ((per + 15) / 16);
    QT_REQUIRE(heads <= 65535 && p.n_seqs <= 65535, "attention_shared: too many rows for one launch");
    launch_kernel_cluster(shared_direct_kernel<HD>, dim3(p.own_ranges, (unsigned)heads, p.n_seqs), dim3(32 * warps), smem, stream, (unsigned)p.own_ranges, p);
    QT_CHECK_LAUNCH("attention_shared");
    return QT_OK;
}

}  // namespace

// A call's arguments as one structure, which its caller lays out field by field.
struct SharedCall {
    const void *q, *k_cache, *v_cache;
    void* out;
    const int *block_table, *seq_len, *members, *share;
    float *part_acc, *part_ml;
    int* status;
    void* stream;
    double scale;
    int dtype, n_seqs, n_groups, most_members, nq, nkv, d, page_tokens, shared_ranges, own_ranges, direct_warps, on_tc, max_blocks, n_pages;
};
static_assert(sizeof(SharedCall) == 13 * 8 + 14 * 4, "12 addresses, a number of 64 bits and 14 of 32, without gaps");

// on_tc: bfloat16, d % 8 == 0 and at most 128, pages of 64.  With shared_ranges = 0 (on_tc) one launch walks all of a member's keys, by own_ranges <= 8
// blocks of direct_warps warps a member and kv head.
extern "C" int qt_attention_decode_shared(const SharedCall* call) {
    const SharedCall& c = *call;
    const int n_seqs = c.n_seqs, n_groups = c.n_groups, most_members = c.most_members, nq = c.nq, nkv = c.nkv, d = c.d, page_tokens = c.page_tokens, n_pages = c.n_pages,
              max_blocks = c.max_blocks, shared_ranges = c.shared_ranges, own_ranges = c.own_ranges, direct_warps = c.direct_warps;
    const float scale = (float)c.scale;
    QT_REQUIRE(n_seqs >= 0 && n_groups > 0 && nq > 0 && nkv > 0 && nq % nkv == 0, "attention_shared: bad head counts nq=%d nkv=%d (B=%d, %d groups)", nq, nkv, n_seqs, n_groups);
    QT_REQUIRE(d > 0 && d <= MAX_DIM && page_tokens > 0 && max_blocks > 0 && n_pages > 0, "attention_shared: bad sizes d=%d page=%d", d, page_tokens);
    QT_REQUIRE((long long)max_blocks * page_tokens <= 0x7fffffffll && most_members >= 0 && most_members <= n_seqs, "attention_shared: bad sizes: %d pages a sequence, %d members",
               max_blocks, most_members);
    QT_REQUIRE(shared_ranges >= 0 && own_ranges > 0 && shared_ranges + own_ranges <= MAX_RANGES, "attention_shared: %d and %d ranges", shared_ranges, own_ranges);
    QT_REQUIRE(scale > 0.f && scale < INFINITY, "attention_shared: a score scale of %g (it must be positive)", (double)scale);
    if (n_seqs == 0) return QT_OK;
    const SharedParams p{c.q, c.k_cache, c.v_cache, c.out, c.block_table, max_blocks, c.seq_len, c.members, c.share, n_seqs, n_groups, nq, nkv, d, page_tokens, n_pages,
                         scale, shared_ranges, own_ranges, c.part_acc, c.part_ml, c.status, 0, 0, 0, 0, 0};
    QT_REQUIRE((((uintptr_t)c.part_acc | (uintptr_t)c.part_ml) & 15) == 0, "attention_shared: scratch must be 16-byte aligned");
    cudaStream_t s = (cudaStream_t)c.stream;
    if (c.on_tc) {
        QT_REQUIRE(c.dtype == QT_BF16 && d % 8 == 0 && d <= 128 && page_tokens == PAGE && c.status,
                   "attention_shared: the tensor-core kernels take bfloat16, heads of up to 128 in steps of 8, pages of 64 (d=%d, pages of %d)", d, page_tokens);
        QT_REQUIRE((long long)n_pages * nkv * PAGE <= 0x7fffffffll, "attention_shared: %d pages of %d heads are beyond a tensor map", n_pages, nkv);
        QT_REQUIRE((((uintptr_t)c.q | (uintptr_t)c.k_cache | (uintptr_t)c.v_cache | (uintptr_t)c.out) & 15) == 0, "attention_shared: operands must be 16-byte aligned");
        if (shared_ranges == 0) {
            QT_REQUIRE(own_ranges <= 8 && direct_warps > 0 && direct_warps <= DIRECT_MAX_WARPS, "attention_shared: %d blocks of %d warps", own_ranges, direct_warps);
            return d <= 64 ? launch_direct<64>(p, direct_warps, s) : launch_direct<128>(p, direct_warps, s);
        }
        return d <= 64 ? launch_parts<64>(p, most_members, s) : launch_parts<128>(p, most_members, s);
    }
    QT_REQUIRE(shared_ranges > 0, "attention_shared: %d ranges of shared keys", shared_ranges);
    return QT_DISPATCH_DTYPE(c.dtype, "attention_shared", {
        if (d <= 64) return launch_any<T, 2>(p, most_members, s);
        if (d <= 128) return launch_any<T, 4>(p, most_members, s);
        return launch_any<T, 8>(p, most_members, s);
    });
}

QT_DEFINE_LAST_ERROR(attention_shared)
