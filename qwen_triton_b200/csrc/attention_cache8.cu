// Attention over a cache held in 8 bits: pages [pages, kv_heads, 64, d] of e4m3 numbers with a scale for each page and head (cache8.cu writes them).
//
//   out_i = sum_j softmax_j(scale q_i . k_j) v_j,     k_j = s_k[page of j] k8_j,     v_j = s_v[page of j] v8_j
//
// A block takes eight rows (query token, head of a kv head's group) and a range of pages; each of its warps walks portions of 32 keys of its own (16 for heads
// beyond 128) through a ring of its own in shared memory, which it fills with cp.async: no warp waits for another before the end.  S^T = K q^T and O^T += V^T P^T on
// mma.sync have keys and values as the operand with 16 rows and the eight query rows as the other.  Which keys and elements a lane's share of a fragment is, is free as
// long as both operands agree, so a lane reads 16 neighbouring bytes; the 16-byte pieces of a row lie where the row's number xored with theirs says, so that the lanes
// that read together meet all banks.
//
// Every e4m3 number is a half.  Queries are brought to halves with a power of two for each row (its largest element lies in [2^14, 2^15), so no digit
// of it is lost but below 2^-38 of that); FLOAT queries are two halves, and so is P then.  A weight is p_j s_v[j] relative to the largest such: the running
// maximum is that of the score plus log2 s_v, so that halves hold the weights whatever scales the pages have; the sum of the p_j takes the scale back out.
// Weights are held times 2^11, at most 2^15, so that one down to 2^-25 of the largest keeps a half's eleven digits, and what is smaller is off by at most 2^-36 of the
// largest.  FLOAT: the second half is what the first one leaves, times 2^11 and with sums of its own, so that it too has its digits: 2^-24 of a weight, or 2^-47 of the largest.
//
// A value that is not a number, of a key that not every row sees, is taken out and noted: its element becomes NaN in the rows that see it, and in no other.
//
// Ranges of a sequence join in the cluster that they form (up to eight), or through memory and a second launch.
//
// Bound by the cache's way from memory for many keys (128 sequences of 4,096 tokens, 32 heads over 8 of 128: 181 us, 5.9 TB/s; 48 of 3,000 to 12,000: 130 us, 5.6 TB/s), by the
// latency of a warp's ring and the join for few (one sequence of 700 tokens, 16 heads over 8: 5.1 us; 8 of 2,048: 13, 5 of them the bytes); in float32, twice the products, by these
// (5 sequences of 1,500, 16 heads of 96: 12.4 us).  Prompts, eight rows a block, walk all keys again for every eight rows: 1,000 tokens behind 2,000, 16 heads over 4, take 404 us with
// heads of 256 (24 are the products at the rate of 16-bit ones), in float32 232 with heads of 128 and 534 with heads of 256, where a few registers spill (on tcgen05 heads of 128 take
// 46 in bfloat16).
#include "cache8_call.h"
#include "fp8.cuh"

#include <algorithm>
#include <math.h>

using namespace qt;
using namespace qt_fp8;

namespace {

constexpr int PAGE = 64;
constexpr int WARPS = 4;
constexpr int ROWS = 8;                                    // query rows of a block
constexpr int MAX_CLUSTER = 8, MAX_RANGES = 64;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float RESCALE_STEP = 4.f;                        // a row's maximum moves when the true one is more than 2^4 above it
constexpr float LIFT = 11.f;                               // weights are held times 2^11: halves end at 2^16
constexpr float REST = 2048.f;                             // FLOAT: and what a half leaves of one times 2^11 again

struct Params {
    const void* q; void* out;
    const uint8_t* k; const uint8_t* v; const float* k_scale; const float* v_scale;
    const int* block_table; int max_blocks, n_pages;
    const int* seq_start; const int* seq_past;             // prompts
    const int* seq_len;                                    // one query a sequence
    int nq, nkv, d;
    float scale;
    int ranges, range_pages;                               // a block walks range_pages pages of its sequence
    int clusters;                                          // ranges join in clusters (up to eight), else through memory
    float* part_acc; float* part_ml;
};

__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ uint32_t shared_address(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
// 16 bytes on their way to shared memory; zeros where `there` is false
__device__ __forceinline__ void copy16(void* to, const void* from, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(shared_address(to)), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(void* to, const void* from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(shared_address(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
template <int WORDS> __device__ __forceinline__ void load_words(uint32_t* w, const uint8_t* at) {
    if constexpr (WORDS == 4) {
        const uint4 x = *reinterpret_cast<const uint4*>(at);
        w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
    } else {
        const uint2 x = *reinterpret_cast<const uint2*>(at);
        w[0] = x.x; w[1] = x.y;
    }
}

// D: the head size rounded up to 64, 128 or 256; what lies between d and D is zero.
template <int D> struct Ring {
    static constexpr int SUBS = D > 128 ? 1 : 2, KEYS = 16 * SUBS, PER_PAGE = PAGE / KEYS;      // 16 keys each, at a time
    static constexpr int STAGES = 2, PIECES = D / 16;                  // 16-byte pieces of a row
    static constexpr int HALF = KEYS * D, STAGE = 2 * HALF + 16;       // keys, values, their scales
    static constexpr size_t SMEM = (size_t)WARPS * STAGES * STAGE;
    static_assert(SMEM >= (size_t)WARPS * ROWS * (D + 2) * 4 + ROWS * (D + 2) * 4, "the warps' results and the block's lie over the rings");
    // where piece c of row r lies
    __device__ static int at(int r, int c) { return r * D + ((D == 64 ? c ^ ((r >> 1) & 3) : c ^ (r & 7)) << 4); }
};

// Of a warp's values of a portion from key `key0` on, rows `from` to `to`: NaN become zeros, and the first key of each element is noted.
template <int D> __device__ __forceinline__ void take_out_nan(uint8_t* values, int from, int to, int key0, int* first_nan) {
#pragma unroll 1
    for (int i = from * Ring<D>::PIECES + (threadIdx.x & 31); i < to * Ring<D>::PIECES; i += 32) {
        uint32_t* words = reinterpret_cast<uint32_t*>(values + Ring<D>::at(i / Ring<D>::PIECES, i % Ring<D>::PIECES));
        const uint4 w = *reinterpret_cast<const uint4*>(words);
        if (!(any_nan(w.x) | any_nan(w.y) | any_nan(w.z) | any_nan(w.w))) continue;
#pragma unroll 1
        for (int b = 0; b < 16; ++b) {
            const uint32_t word = words[b >> 2];
            if ((word >> (8 * (b & 3)) & 0x7f) != 0x7f) continue;
            words[b >> 2] = word & ~(0xffu << (8 * (b & 3)));
            first_nan[D] = 1;
            atomicMin(first_nan + i % Ring<D>::PIECES * 16 + b, key0 + i / Ring<D>::PIECES);
        }
    }
    __syncwarp();
}

// JOIN: how ranges meet.  ALONE: there is one; CLUSTER: the blocks of a cluster along x; MEMORY: parts for the second launch.
constexpr int ALONE = 0, CLUSTER = 1, MEMORY = 2;

template <int D, int JOIN, typename T>
__global__ void __launch_bounds__(32 * WARPS, sizeof(T) == 4 || D > 128 ? 2 : 3) attention_cache8_kernel(const Params p) {
    using R = Ring<D>;
    constexpr bool FLOAT = sizeof(T) == 4;
    constexpr int STEPS = D / 16, SUBS = R::SUBS, KEYS = R::KEYS, PER_PAGE = R::PER_PAGE, STAGES = R::STAGES;
    constexpr int KPIECES = D / 64;                        // of a key row, a lane's pieces: KPIECES t + c (of 64 elements: t)
    constexpr int VBYTES = D / 8;                          // of a value row, a lane's neighbouring elements
    extern __shared__ __align__(128) uint8_t shared[];
    __shared__ int first_nan[D + 1];                       // prompts: of each element, the first key taken out; whether there is one
    pdl_launch_dependents();
    if (p.seq_start) {
        for (int i = threadIdx.x; i <= D; i += 32 * WARPS) first_nan[i] = i < D ? 0x7fffffff : 0;
        __syncthreads();
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int seq = blockIdx.z, kvh = blockIdx.y % p.nkv, group = p.nq / p.nkv;
    const int tile = p.seq_start ? blockIdx.x / p.ranges : blockIdx.y / p.nkv, range = JOIN == ALONE ? 0 : p.seq_start ? blockIdx.x % p.ranges : blockIdx.x;
    uint8_t* ring = shared + warp * STAGES * R::STAGE;
    if (p.d < D) {                                         // what no copy reaches
        for (int i = lane; i < STAGES * R::STAGE / 16; i += 32) *reinterpret_cast<uint4*>(ring + 16 * i) = make_uint4(0, 0, 0, 0);
        __syncwarp();
    }
    pdl_wait();
    const int* table = p.block_table + (size_t)seq * p.max_blocks;
    int range_pages = p.range_pages;
    if (JOIN == CLUSTER && p.seq_start)                    // prompts: equal ranges of what the tile's last row sees
        range_pages = max(1, (p.seq_past[seq] + (min((tile + 1) * ROWS, (p.seq_start[seq + 1] - p.seq_start[seq]) * group) - 1) / group + PAGE) / PAGE + p.ranges - 1) / p.ranges;
    const int page_begin = (int)min((long long)range * range_pages, (long long)p.max_blocks), begin = page_begin * PER_PAGE + warp;
    // the first pages are asked for together with the lengths that say whether they are needed
    int first[STAGES];
#pragma unroll
    for (int s = 0; s < STAGES; ++s) first[s] = table[min((begin + s * WARPS) / PER_PAGE, p.max_blocks - 1)];
    const int capacity = p.max_blocks * PAGE;
    int token0 = seq, tokens = 1, past;
    if (p.seq_start) {
        token0 = p.seq_start[seq];
        tokens = p.seq_start[seq + 1] - token0;
        past = p.seq_past[seq];
    } else {
        past = min(p.seq_len[seq], capacity) - 1;
    }
    const int row0 = tile * ROWS, rows = tokens * group;
    if (row0 >= rows) return;                              // prompts only, and the same for a whole cluster
    const int last_row = min(row0 + ROWS, rows) - 1;
    const int end = min(past + last_row / group + 1, capacity);          // keys that any row sees
    const int pages = (end + PAGE - 1) / PAGE;
    const int page_end = range == p.ranges - 1 ? pages : min(pages, page_begin + range_pages);        // the last range takes what is left
    if (JOIN == MEMORY && page_begin >= page_end && range > 0) return;   // the join knows from the length

    const int stop = (min(end, page_end * PAGE) + KEYS - 1) / KEYS;      // portions; the warp's are begin, begin + WARPS, ...
    auto page_number = [&](int u) { return u < stop ? min(max(table[u / PER_PAGE], 0), p.n_pages - 1) : 0; };
    // portion u on its way to stage s
    auto fetch = [&](int u, int s, int page) {
        uint8_t* to = ring + s * R::STAGE;
        if (u < stop) {
            const size_t block = (size_t)page * p.nkv + kvh;
            const int key = u % PER_PAGE * KEYS, there = end - u * KEYS;
            const uint8_t* k = p.k + (block * PAGE + key) * p.d;
            const uint8_t* v = p.v + (block * PAGE + key) * p.d;
            const int pieces = p.d >> 4;
            if (p.d == D) {
#pragma unroll
                for (int i = lane; i < KEYS * R::PIECES; i += 32) {
                    const int r = i / R::PIECES, c = i % R::PIECES;
                    copy16(to + R::at(r, c), k + 16 * i, true);
                    copy16(to + R::HALF + R::at(r, c), v + 16 * i, r < there);
                }
            } else {
                for (int i = lane; i < KEYS * pieces; i += 32) {
                    const int r = i / pieces, c = i % pieces;
                    copy16(to + R::at(r, c), k + 16 * i, true);
                    copy16(to + R::HALF + R::at(r, c), v + 16 * i, r < there);
                }
            }
            if (lane < 2) copy4(to + 2 * R::HALF + 4 * lane, (lane ? p.v_scale : p.k_scale) + block);
        }
        copies_end();
    };
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) fetch(begin + s * WARPS, s, min(max(first[s], 0), p.n_pages - 1));
    int page = min(max(first[STAGES - 1], 0), p.n_pages - 1);      // of the next portion to fetch

    // queries: row g of the block; of key rows, lane t has the elements from 16 KPIECES t on (instruction 4 c + j: 4 of them from 16 c + 4 j on)
    uint32_t qh[STEPS][2], ql[FLOAT ? STEPS : 1][2];
    float factor;
    {
        const int row = row0 + g;
        const bool here = row <= last_row;
        const T* q = (const T*)p.q + ((size_t)(token0 + row / group) * p.nq + kvh * group + row % group) * p.d;
        float x[STEPS][4], most = 0.f;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const int at = 16 * KPIECES * t + 4 * s;
            if (here && at < p.d) {
                if constexpr (FLOAT) {
                    const float4 f = *reinterpret_cast<const float4*>(q + at);
                    x[s][0] = f.x; x[s][1] = f.y; x[s][2] = f.z; x[s][3] = f.w;
                } else {
                    const uint2 f = *reinterpret_cast<const uint2*>(q + at);
                    const float2 lo = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&f.x)), hi = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&f.y));
                    x[s][0] = lo.x; x[s][1] = lo.y; x[s][2] = hi.x; x[s][3] = hi.y;
                }
            } else {
                x[s][0] = x[s][1] = x[s][2] = x[s][3] = 0.f;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) most = fmaxf(most, fabsf(x[s][i]));
        }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        // 2^-shift brings the largest to [2^14, 2^15); none for rows of zeros or with infinities
        int shift = (__float_as_int(most) >> 23) - 127 - 14;
        if (!(most >= 0x1p-100f && most < INFINITY)) shift = 0;
        const float by = exp2f((float)-shift);
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            float y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = x[s][i] * by;
            qh[s][0] = pack_half(y[0], y[1]);
            qh[s][1] = pack_half(y[2], y[3]);
            if (FLOAT) {
                const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&qh[s][0])), b = __half22float2(*reinterpret_cast<const __half2*>(&qh[s][1]));
                ql[FLOAT ? s : 0][0] = pack_half(y[0] - a.x, y[1] - a.y);
                ql[FLOAT ? s : 0][1] = pack_half(y[2] - b.x, y[3] - b.y);
            }
        }
        factor = exp2f((float)shift) * p.scale * LOG2E;
    }
    // of scores, lane (g, t) has rows 2 t and 2 t + 1
    const float factor0 = __shfl_sync(0xffffffffu, factor, 8 * t), factor1 = __shfl_sync(0xffffffffu, factor, 8 * t + 4);
    const int limit0 = row0 + 2 * t <= last_row ? past + (row0 + 2 * t) / group + 1 : 0;
    const int limit1 = row0 + 2 * t + 1 <= last_row ? past + (row0 + 2 * t + 1) / group + 1 : 0;
    const int least = past + row0 / group + 1;             // keys below are seen by every row that is there

    float acc[STEPS][4] = {}, rest[FLOAT ? STEPS : 1][4] = {};
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    int s_at = 0;
    for (int u = begin; u < stop; u += WARPS) {
        // the stage that the portion before this one left is the next to fill
        fetch(u + (STAGES - 1) * WARPS, s_at == 0 ? STAGES - 1 : s_at - 1, page);
        page = page_number(u + STAGES * WARPS);
        copies_wait<STAGES - 1>();
        __syncwarp();
        const uint8_t* stage = ring + s_at * R::STAGE;
        const int key0 = u * KEYS;
        s_at = s_at == STAGES - 1 ? 0 : s_at + 1;
        const float2 scales = *reinterpret_cast<const float2*>(stage + 2 * R::HALF);
        const float f0 = factor0 * scales.x, f1 = factor1 * scales.x, lift = log2f(scales.y), out_of = 1.f / scales.y;
        float s[SUBS][4];
#pragma unroll
        for (int v = 0; v < SUBS; ++v) {
            float c[2][4] = {};                            // two chains of half as many dependent instructions
#pragma unroll
            for (int i = 0; i < KPIECES; ++i) {
                uint32_t a[4], b[4];
                load_words<4>(a, stage + R::at(16 * v + g, KPIECES * t + i));
                load_words<4>(b, stage + R::at(16 * v + 8 + g, KPIECES * t + i));
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t a0 = halves(a[j]), a1 = halves(b[j]), a2 = halves(a[j] >> 16), a3 = halves(b[j] >> 16);
                    mma(c[j & 1], a0, a1, a2, a3, qh[4 * i + j][0], qh[4 * i + j][1]);
                    if (FLOAT) mma(c[j & 1], a0, a1, a2, a3, ql[FLOAT ? 4 * i + j : 0][0], ql[FLOAT ? 4 * i + j : 0][1]);
                }
            }
            s[v][0] = fmaf(c[0][0] + c[1][0], f0, lift); s[v][1] = fmaf(c[0][1] + c[1][1], f1, lift);
            s[v][2] = fmaf(c[0][2] + c[1][2], f0, lift); s[v][3] = fmaf(c[0][3] + c[1][3], f1, lift);
        }
        if (key0 + KEYS > least || last_row < row0 + ROWS - 1) {
#pragma unroll
            for (int v = 0; v < SUBS; ++v)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (key0 + 16 * v + g + 8 * (i >> 1) >= ((i & 1) ? limit1 : limit0)) s[v][i] = -INFINITY;
            if (p.seq_start && key0 + KEYS > least)         // (a value that every row sees makes its element NaN in all of them by itself)
                take_out_nan<D>(const_cast<uint8_t*>(stage) + R::HALF, max(least - key0, 0), min(end - key0, KEYS), key0, first_nan);
        }
        float top0 = -INFINITY, top1 = -INFINITY;
#pragma unroll
        for (int v = 0; v < SUBS; ++v) {
            top0 = fmaxf(top0, fmaxf(s[v][0], s[v][2]));
            top1 = fmaxf(top1, fmaxf(s[v][1], s[v][3]));
        }
        if (__any_sync(0xffffffffu, top0 > m0 + RESCALE_STEP || top1 > m1 + RESCALE_STEP)) {
#pragma unroll
            for (int off = 4; off < 32; off *= 2) {
                top0 = fmaxf(top0, __shfl_xor_sync(0xffffffffu, top0, off));
                top1 = fmaxf(top1, __shfl_xor_sync(0xffffffffu, top1, off));
            }
            const float n0 = fmaxf(m0, top0), n1 = fmaxf(m1, top1);
            const float a0 = n0 == -INFINITY ? 1.f : fast_exp2(m0 - n0), a1 = n1 == -INFINITY ? 1.f : fast_exp2(m1 - n1);
            l0 *= a0; l1 *= a1;
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
                acc[i][0] *= a0; acc[i][1] *= a1; acc[i][2] *= a0; acc[i][3] *= a1;
                if (FLOAT) { float (&r)[4] = rest[FLOAT ? i : 0]; r[0] *= a0; r[1] *= a1; r[2] *= a0; r[3] *= a1; }
            }
            m0 = n0; m1 = n1;
        }
        const float u0 = m0 == -INFINITY ? 0.f : m0 - LIFT, u1 = m1 == -INFINITY ? 0.f : m1 - LIFT;
#pragma unroll
        for (int v = 0; v < SUBS; ++v) {
            const float w0 = fast_exp2(s[v][0] - u0), w1 = fast_exp2(s[v][1] - u1), w2 = fast_exp2(s[v][2] - u0), w3 = fast_exp2(s[v][3] - u1);
            l0 = fmaf(w0 + w2, out_of, l0);
            l1 = fmaf(w1 + w3, out_of, l1);
            const uint32_t h0 = pack_half(w0, w1), h1 = pack_half(w2, w3);
            const uint32_t b0 = transposed(h0), b1 = transposed(h1);
            uint32_t r0 = 0, r1 = 0;
            if (FLOAT) {
                const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&h0)), y = __half22float2(*reinterpret_cast<const __half2*>(&h1));
                r0 = transposed(pack_half((w0 - x.x) * REST, (w1 - x.y) * REST));
                r1 = transposed(pack_half((w2 - y.x) * REST, (w3 - y.y) * REST));
            }
            const uint8_t* values = stage + R::HALF;
#pragma unroll
            for (int c = 0; c < (VBYTES + 15) / 16; ++c) {
                constexpr int WORDS = VBYTES < 16 ? VBYTES / 4 : 4;
                uint32_t vw[4][WORDS];                     // keys 16 v + 2 t, + 1, + 8, + 9
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int byte = g * VBYTES + 16 * c;
                    load_words<WORDS>(vw[i], values + R::at(16 * v + 2 * t + (i & 1) + 8 * (i >> 1), byte >> 4) + (byte & 15));
                }
#pragma unroll
                for (int w = 0; w < WORDS; ++w) {
                    // bytes of neighbouring keys side by side: an element's two keys are one half2
                    const uint32_t a01 = __byte_perm(vw[0][w], vw[1][w], 0x5140), a23 = __byte_perm(vw[0][w], vw[1][w], 0x7362);
                    const uint32_t b01 = __byte_perm(vw[2][w], vw[3][w], 0x5140), b23 = __byte_perm(vw[2][w], vw[3][w], 0x7362);
                    const uint32_t x0 = halves(a01), x1 = halves(a01 >> 16), x2 = halves(b01), x3 = halves(b01 >> 16);
                    const uint32_t y0 = halves(a23), y1 = halves(a23 >> 16), y2 = halves(b23), y3 = halves(b23 >> 16);
                    mma(acc[8 * c + 2 * w], x0, x1, x2, x3, b0, b1);
                    mma(acc[8 * c + 2 * w + 1], y0, y1, y2, y3, b0, b1);
                    if (FLOAT) {
                        mma(rest[FLOAT ? 8 * c + 2 * w : 0], x0, x1, x2, x3, r0, r1);
                        mma(rest[FLOAT ? 8 * c + 2 * w + 1 : 0], y0, y1, y2, y3, r0, r1);
                    }
                }
            }
        }
        __syncwarp();                                      // the stage may be filled again
    }
    // the warps' results, then the block's, over the rings
    copies_wait<0>();
    __syncthreads();
#pragma unroll
    for (int off = 4; off < 32; off *= 2) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, off);
        l1 += __shfl_xor_sync(0xffffffffu, l1, off);
    }
    float* parts = reinterpret_cast<float*>(shared);       // [WARPS][ROWS][D]
    float* sums = parts + WARPS * ROWS * D;                // [WARPS][ROWS][2]
    float* block_part = sums + WARPS * ROWS * 2;           // CLUSTER: [ROWS][D], [ROWS][2]
    float* block_sums = block_part + ROWS * D;
    if (g == 0) {
        sums[(warp * ROWS + 2 * t) * 2] = m0; sums[(warp * ROWS + 2 * t) * 2 + 1] = l0;
        sums[(warp * ROWS + 2 * t + 1) * 2] = m1; sums[(warp * ROWS + 2 * t + 1) * 2 + 1] = l1;
    }
    float* own = parts + warp * ROWS * D + g * VBYTES;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {                      // elements 2 i and 2 i + 1 of the lane's
        if (FLOAT) {
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(rest[FLOAT ? i : 0][j], 1.f / REST, acc[i][j]);
        }
        *reinterpret_cast<float2*>(own + (2 * t) * D + 2 * i) = make_float2(acc[i][0], acc[i][2]);
        *reinterpret_cast<float2*>(own + (2 * t + 1) * D + 2 * i) = make_float2(acc[i][1], acc[i][3]);
    }
    __syncthreads();
    const bool some_nan = p.seq_start && first_nan[D];
    for (int i = threadIdx.x; i < ROWS * p.d; i += 32 * WARPS) {
        const int r = i / p.d, c = i % p.d, row = row0 + r;
        if (row > last_row) break;
        float m = -INFINITY, l = 0.f, a = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) m = fmaxf(m, sums[(w * ROWS + r) * 2]);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float mw = sums[(w * ROWS + r) * 2];
            // a warp without keys has nothing; one whose sums are NaN hands that on
            const float by = mw == -INFINITY ? 1.f : fast_exp2(mw - m);
            l = fmaf(sums[(w * ROWS + r) * 2 + 1], by, l);
            a = fmaf(parts[(w * ROWS + r) * D + c], by, a);
        }
        const int head = kvh * group + row % group;
        if (some_nan && first_nan[c] <= past + row / group) a = NAN;
        if (JOIN == ALONE) {
            ((T*)p.out)[((size_t)(token0 + row / group) * p.nq + head) * p.d + c] = from_float<T>(l == 0.f ? 0.f : a / l);
        } else if (JOIN == MEMORY) {
            const size_t part = ((size_t)seq * p.nq + head) * p.ranges + range;
            p.part_acc[part * p.d + c] = a;
            if (c == 0) { p.part_ml[part * 2] = m; p.part_ml[part * 2 + 1] = l; }
        } else {
            block_part[r * D + c] = a;
            if (c == 0) { block_sums[2 * r] = m; block_sums[2 * r + 1] = l; }
        }
    }
    if (JOIN == CLUSTER) {
        cluster_barrier();
        const int ranks = p.ranges, live = last_row - row0 + 1;
        const uint32_t part0 = shared_address(block_part), sums0 = shared_address(block_sums);
        auto remote = [](uint32_t at, int rank) {
            uint32_t there;
            float v;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(rank));
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(there) : "memory");
            return v;
        };
        for (int i = range * 32 * WARPS + threadIdx.x; i < live * p.d; i += ranks * 32 * WARPS) {
            const int r = i / p.d, c = i % p.d;
            float mr[MAX_CLUSTER], lr[MAX_CLUSTER], ar[MAX_CLUSTER], m = -INFINITY, l = 0.f, a = 0.f;
#pragma unroll
            for (int k = 0; k < MAX_CLUSTER; ++k)
                if (k < ranks) {
                    mr[k] = remote(sums0 + 8 * r, k);
                    lr[k] = remote(sums0 + 8 * r + 4, k);
                    ar[k] = remote(part0 + 4 * (r * D + c), k);
                }
#pragma unroll
            for (int k = 0; k < MAX_CLUSTER; ++k)
                if (k < ranks) m = fmaxf(m, mr[k]);
#pragma unroll
            for (int k = 0; k < MAX_CLUSTER; ++k)
                if (k < ranks) {
                    const float by = mr[k] == -INFINITY ? 1.f : fast_exp2(mr[k] - m);
                    l = fmaf(lr[k], by, l);
                    a = fmaf(ar[k], by, a);
                }
            const int row = row0 + r;
            ((T*)p.out)[((size_t)(token0 + row / group) * p.nq + kvh * group + row % group) * p.d + c] = from_float<T>(l == 0.f ? 0.f : a / l);
        }
        cluster_barrier();                                 // nobody leaves while its part is read
    }
}

// The ranges of a (sequence, head): sum of l and acc, each at its distance from the largest maximum.  GROUPS of threads (four for more than 16 ranges) take every
// GROUPS-th range, so that sixteen parts are on their way at a time (32 ranges of one sequence of 8,192: 11.5 us with four groups, 12.3 with one; but 4 ranges of 128
// sequences of 4,096, whose blocks are many: 191 and 180).
constexpr int JOIN_WIDTH = 128;
template <int GROUPS, typename T>
__global__ void __launch_bounds__(GROUPS * JOIN_WIDTH) join_cache8_kernel(const Params p) {
    __shared__ float by[MAX_RANGES], parts[GROUPS][JOIN_WIDTH];
    pdl_launch_dependents();
    pdl_wait();
    const int head = blockIdx.x, seq = blockIdx.y, lane = threadIdx.x & 31, member = threadIdx.x % JOIN_WIDTH, of = threadIdx.x / JOIN_WIDTH;
    const int pages = (min(p.seq_len[seq], p.max_blocks * PAGE) + PAGE - 1) / PAGE;
    const int used = min(max(1, (pages + p.range_pages - 1) / p.range_pages), p.ranges);
    const size_t first = ((size_t)seq * p.nq + head) * p.ranges;
    const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + first;
    // every warp the same
    const float2 a = lane < used ? ml[lane] : make_float2(-INFINITY, 0.f), b = lane + 32 < used ? ml[lane + 32] : make_float2(-INFINITY, 0.f);
    const float m = warp_max(fmaxf(a.x, b.x));
    const float fa = a.x == -INFINITY ? 1.f : fast_exp2(a.x - m), fb = b.x == -INFINITY ? 1.f : fast_exp2(b.x - m);
    const float l = warp_sum(fmaf(a.y, fa, b.y * fb));
    if (threadIdx.x < 32) { by[lane] = fa; by[lane + 32] = fb; }
    __syncthreads();
    for (int c0 = 0; c0 < p.d; c0 += JOIN_WIDTH) {         // the same for every thread
        const int c = c0 + member;
        float sum = 0.f;
        if (c < p.d) {
#pragma unroll 4
            for (int r = of; r < used; r += GROUPS) sum = fmaf(p.part_acc[(first + r) * p.d + c], by[r], sum);
        }
        if (GROUPS > 1) {
            parts[of][member] = sum;
            __syncthreads();
            sum = 0.f;
#pragma unroll
            for (int i = 0; i < GROUPS; ++i) sum += parts[i][member];
        }
        if (of == 0 && c < p.d) {
            ((T*)p.out)[((size_t)seq * p.nq + head) * p.d + c] = from_float<T>(l == 0.f ? 0.f : sum / l);
        }
        __syncthreads();
    }
}

template <int D, int JOIN, typename T> int launch(const Params& p, dim3 grid, cudaStream_t stream) {
    const cudaError_t raised = raise_shared<attention_cache8_kernel<D, JOIN, T>>((int)Ring<D>::SMEM);
    if (raised != cudaSuccess) QT_FAIL(QT_ERR_LAUNCH, "attention_cache8: cannot raise shared memory: %s", cudaGetErrorString(raised));
    if (JOIN == CLUSTER) launch_kernel_cluster(attention_cache8_kernel<D, JOIN, T>, grid, dim3(32 * WARPS), Ring<D>::SMEM, stream, (unsigned)p.ranges, p);
    else launch_kernel(attention_cache8_kernel<D, JOIN, T>, grid, dim3(32 * WARPS), Ring<D>::SMEM, stream, p);
    QT_CHECK_LAUNCH("attention_cache8");
    if (JOIN == MEMORY) {
        if (p.ranges > 16) launch_kernel(join_cache8_kernel<4, T>, dim3(p.nq, grid.z), dim3(4 * JOIN_WIDTH), 0, stream, p);
        else launch_kernel(join_cache8_kernel<1, T>, dim3(p.nq, grid.z), dim3(JOIN_WIDTH), 0, stream, p);
        QT_CHECK_LAUNCH("attention_cache8 join");
    }
    return QT_OK;
}
template <int D, typename T> int launch_join(const Params& p, dim3 grid, cudaStream_t stream) {
    if (p.ranges == 1) return launch<D, ALONE, T>(p, grid, stream);
    if (p.clusters) return launch<D, CLUSTER, T>(p, grid, stream);
    return launch<D, MEMORY, T>(p, grid, stream);
}
template <typename T> int launch_size(const Params& p, dim3 grid, cudaStream_t stream) {
    if (p.d <= 64) return launch_join<64, T>(p, grid, stream);
    if (p.d <= 128) return launch_join<128, T>(p, grid, stream);
    return launch_join<256, T>(p, grid, stream);
}

int check(const char* name, int dtype, int nq, int nkv, int d, int max_blocks, int n_pages, const void* q, const void* k, const void* v, const void* out) {
    QT_REQUIRE(dtype == QT_F32 || dtype == QT_BF16, "%s: unknown element type %d", name, dtype);
    QT_REQUIRE(nq > 0 && nkv > 0 && nq % nkv == 0 && max_blocks > 0 && max_blocks <= 0x7fffffff / PAGE && n_pages > 0, "%s: bad sizes nq=%d nkv=%d", name, nq, nkv);
    QT_REQUIRE(d > 0 && d <= 256 && d % 16 == 0, "%s: head_dim=%d is not a multiple of 16 up to 256", name, d);
    QT_REQUIRE((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & 15) == 0, "%s: operands must be 16-byte aligned", name);
    return QT_OK;
}

}  // namespace

// One query a sequence: q and out [n_seqs, nq, d], seq_len [n_seqs] keys each (none: zeros).  Ranges join in clusters of blocks (at most eight,
// with `clusters`) or through memory: part_acc holds n_seqs nq ranges d floats and part_ml n_seqs nq ranges 2.  A block walks range_pages pages of its
// sequence, the last range whatever is left.
extern "C" int qt_attention_decode_cache8(const Cache8Call* call) {
    const Cache8Call& c = *call;
    if (c.n_seqs == 0) return QT_OK;
    const int rc = check("attention_decode_cache8", c.dtype, c.nq, c.nkv, c.d, c.max_blocks, c.n_pages, c.q, c.k, c.v, c.out);
    if (rc) return rc;
    const int tiles = (c.nq / c.nkv + ROWS - 1) / ROWS;
    QT_REQUIRE(c.n_seqs > 0 && c.n_seqs <= 65535 && (long long)c.nkv * tiles <= 65535, "attention_decode_cache8: %d sequences of %d heads", c.n_seqs, c.nq);
    const int clusters = c.clusters && c.ranges <= MAX_CLUSTER;
    QT_REQUIRE(c.ranges >= 1 && c.ranges <= MAX_RANGES && c.range_pages >= 1 && (c.ranges == 1 || clusters || (c.part_acc && c.part_ml && (uintptr_t)c.part_ml % 8 == 0)),
               "attention_decode_cache8: %d ranges of %d pages", c.ranges, c.range_pages);
    const Params p{c.q, c.out, (const uint8_t*)c.k, (const uint8_t*)c.v, c.k_scale, c.v_scale, c.block_table, c.max_blocks, c.n_pages, nullptr, nullptr, c.seq_len, c.nq, c.nkv, c.d,
                   (float)c.scale, c.ranges, std::min(c.range_pages, c.max_blocks), clusters, c.part_acc, c.part_ml};
    const dim3 grid(c.ranges, c.nkv * tiles, c.n_seqs);
    return c.dtype == QT_F32 ? launch_size<float>(p, grid, (cudaStream_t)c.stream) : launch_size<__nv_bfloat16>(p, grid, (cudaStream_t)c.stream);
}

// Packed queries [n_tokens, nq, d] of sequences whose keys, this call's own among them, are in the cache; causal.  A tile's keys are walked by a cluster of `ranges`
// blocks.
extern "C" int qt_attention_prefill_cache8(const Cache8Call* call) {
    const Cache8Call& c = *call;
    if (c.n_seqs == 0 || c.max_q_len == 0) return QT_OK;
    const int rc = check("attention_prefill_cache8", c.dtype, c.nq, c.nkv, c.d, c.max_blocks, c.n_pages, c.q, c.k, c.v, c.out);
    if (rc) return rc;
    QT_REQUIRE(c.n_seqs > 0 && c.n_seqs <= 65535 && c.nkv <= 65535 && c.max_q_len > 0 && (long long)c.max_q_len * (c.nq / c.nkv) <= 0x7fffffff - ROWS,
               "attention_prefill_cache8: %d sequences of up to %d tokens", c.n_seqs, c.max_q_len);
    const Params p{c.q, c.out, (const uint8_t*)c.k, (const uint8_t*)c.v, c.k_scale, c.v_scale, c.block_table, c.max_blocks, c.n_pages, c.seq_start, c.seq_past, nullptr, c.nq, c.nkv, c.d,
                   (float)c.scale, c.ranges, c.max_blocks, c.ranges > 1, nullptr, nullptr};
    const long long blocks = (((long long)c.max_q_len * (c.nq / c.nkv) + ROWS - 1) / ROWS) * c.ranges;
    QT_REQUIRE(c.ranges >= 1 && c.ranges <= MAX_CLUSTER && blocks <= 0x7fffffff, "attention_prefill_cache8: %d ranges", c.ranges);
    const dim3 grid((unsigned)blocks, c.nkv, c.n_seqs);
    return c.dtype == QT_F32 ? launch_size<float>(p, grid, (cudaStream_t)c.stream) : launch_size<__nv_bfloat16>(p, grid, (cudaStream_t)c.stream);
}

QT_DEFINE_LAST_ERROR(attention_cache8)
