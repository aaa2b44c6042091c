// Attention of prompts over a cache held in 8 bits on the fifth-generation tensor cores (bfloat16 queries, heads in steps of 16 up to 128, pages of 64).
//
//   S = Q K^T        tcgen05.mma kind::f8f6f4.  The keys are 8-bit numbers as they lie in the cache.  A query row times a power of two is the sum of two such numbers:
//                    the nearest one and the nearest to what is left, which hold a bfloat16 number's eight digits but for elements below 2^-8 of the row's
//                    largest (these are off by at most 2^-17 of it: the largest lies from 2^7 on, the second number ends at 2^-9 and may be off by 2^-10).  Twice the products at twice the rate of 16-bit ones, and no key is converted.
//   P = softmax(S)   a thread a row, in registers; the powers of two and the page's scales are factors on the scores
//   O += P V         tcgen05.mma kind::f16.  P is halves in tensor memory; the values are brought to halves, which hold every 8-bit number, by four warps on their way
//                    from one shared-memory tile to another, once for the block's 256 rows.  (Both as 8-bit numbers, P in two, would need no conversion of
//                    values, but P's small weights would end at 2^-18 of the largest, and the conversions of P are more.)
//
// A weight is p_j s_v[j] relative to the largest such, as in attention_cache8.cu: the maximum is that of the score plus log2 s_v, and the row's sum takes the scale out.  Weights are
// held times 2^11, at most 2^15: one down to 2^-25 of the largest keeps a half's eleven digits, and what is smaller is off by at most 2^-36 of the largest.
//
// A block takes 256 rows (query token, head of a kv head's group; a token's heads are neighbours) as two tiles of 128 and walks the keys page by page.  S of a
// page is double buffered, P lies over the scores it came from, O stays in tensor memory and is scaled only where a row's maximum runs 2^4 ahead of the one it is
// scaled by (at 2^14, which leaves the weights no room to be lifted, 758 us in the place of 779 and with heads of 64 153 in the place of 161; but all below 2^-25 of the largest are
// lost then, however many).  512 threads: warp 0 copies (TMA tiles of keys, bulk copies of values), warp 1 issues, warps 4 to 7 convert values, warps 8 to 11 and 12 to 15 are the
// softmax of the two tiles, with most of the registers: 88 + 88 + 168 + 168 = 4 * 128.  Every mbarrier wait is bounded and reports through a status word.
//
// A value that is not a number, in a page that not every row sees, becomes zero as it is converted, and the first key of each element is noted: that element is NaN in the rows
// that see it, and in no other.
//
// Few blocks behind many keys: the pages of a block are cut into ranges for a cluster of up to eight, whose sums meet in distributed shared memory, laid over the
// operands (256 tokens of 32 heads over 8 of 128 behind 8,000: 158 us in one range, 56 in four; 64 tokens 154 and, in eight, 37).
//
// What bounds it: a page of a block takes some 1,950 cycles, of which the tensor cores are asked for 1,600: the products of scores run at half their rate, their queries on the way
// from shared memory (66 cycles for 128 x 64 x 32, of which the tensor cores need 32).  4,096 tokens behind 8,192, 32 heads over 8 of 128: 744-791 us as clocks are, 925-870
// TFLOP/s; the same over a 16-bit cache, attention_tc.cu, 734.  What was tried on it (figures of before the weights were lifted): two pages at a time, which halve the queries' way, but leave room for one sum a row, so
// that the two threads of a row walk in step (739 in the place of 712); half of the queries in tensor memory, with scores buffered once (810 in the place of 729, and with
// heads of 64 695 in the place of 620); an eighth of the exponentials on the FMA pipe (no change, more of them slower); other orders of the products than a tile's next
// scores, then its values, tile by tile (both tiles' scores first 785, values first 850, whatever is ready 758).
#include "cache8_call.h"
#include "fp8.cuh"
#include "tc_common.cuh"

#include <math.h>

using namespace qt;
using namespace qt_fp8;
using namespace qt_tc;

namespace {

constexpr int PAGE = 64;
constexpr int BQ = 128, TILES = 2;                         // rows of a tile = the instruction's M; tiles of a block
constexpr int THREADS = 512;
constexpr int K_STAGES = 3, RAW_STAGES = 3, V_STAGES = 3;
constexpr int MAX_RANGES = 8, LEAST_PAGES = 4;              // blocks of a cluster; pages that a block walks before another one has any
constexpr float RESCALE_STEP = 4.f, LIFT = 11.f, LOG2E = 1.4426950408889634f;       // weights are held times 2^LIFT: 2^15 at most, halves end at 2^16

struct TcParams {
    const __nv_bfloat16* q; __nv_bfloat16* out;
    const uint8_t* v; const float* k_scale; const float* v_scale;
    const int* block_table; int max_blocks, n_pages;
    const int* seq_start; const int* seq_past;
    int nq, nkv, d, ranges;
    float scale;
    int* status;
};

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
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// A whole warp goes through the same instructions and one lane's are carried out: descriptors stay in the registers that a warp has in common.
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t elected;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(elected));
    return elected;
}
__device__ __forceinline__ void mma_scores(uint32_t tmem_d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate, uint32_t one) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(tmem_d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(one) : "memory");
}
__device__ __forceinline__ void mma_values(uint32_t tmem_d, uint32_t tmem_a, uint64_t b_desc, uint32_t idesc, uint32_t accumulate, uint32_t one) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(tmem_d), "r"(tmem_a), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(one) : "memory");
}
__device__ __forceinline__ void commit_one(uint32_t bar, uint32_t one) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(one) : "memory");
}
// mbar_wait without a call: where warps have different numbers of registers, ptxas finds none for a function that all of them call.
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, int* status, int code) {
    unsigned long long since = 0;
#pragma unroll 1
    for (uint32_t spins = 1; !mbar_try_wait(bar, parity); ++spins)
        if ((spins & 0x3ffu) == 0) {
            if (*(volatile int*)status != 0) return false;
            const unsigned long long now = global_timer();
            if (since == 0) since = now;
            else if (now - since > WAIT_LIMIT_NS) { atomicCAS(status, 0, code); return false; }
        }
    return true;
}
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, int* status, int code) { return __all_sync(0xffffffffu, wait(bar, parity, status, code)); }
// `bytes` (a multiple of 16) from global to shared memory, counted on a barrier
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
// K-major tile of 64-byte rows, 64-byte swizzle: groups of 8 rows lie 512 bytes apart
__device__ __forceinline__ uint64_t operand_desc_64(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3ffffu) >> 4) | (uint64_t)1 << 16 | (uint64_t)(512 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)4 << 61;
}
// MN-major tile stored as [blocks of 64 elements][keys][64 elements] halves, 128-byte swizzle
__device__ __forceinline__ uint64_t operand_desc_mn(uint32_t saddr, uint32_t block_bytes) {
    return (uint64_t)((saddr & 0x3ffffu) >> 4) | (uint64_t)((block_bytes >> 4) & 0x3fffu) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
__device__ __forceinline__ void store16(uint32_t addr, uint4 v) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint4 load16(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
// Sixteen values of a key, in shared memory or in registers: NaN become zeros, and the first key of each element is noted.  (Not functions that are called: see `wait`.)
__device__ __forceinline__ void take_out_nan(uint32_t addr, int* first_nan, int key) {
#pragma unroll 1
    for (int b = 0; b < 16; ++b) {
        uint32_t byte;
        asm volatile("ld.shared.u8 %0, [%1];" : "=r"(byte) : "r"(addr + b) : "memory");
        if ((byte & 0x7f) != 0x7f) continue;
        asm volatile("st.shared.u8 [%0], %1;" ::"r"(addr + b), "r"(0) : "memory");
        atomicMin(first_nan + b, key);
    }
}
__device__ __forceinline__ void take_out_nan(uint4& v, int* first_nan, int key) {
    uint32_t* words[4] = {&v.x, &v.y, &v.z, &v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll 1
        for (int b = 0; b < 32; b += 8)
            if ((*words[k] >> b & 0x7f) == 0x7f) {
                *words[k] &= ~(0xffu << b);
                atomicMin(first_nan + 4 * k + b / 8, key);
            }
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

template <int HD> struct Shape {
    static constexpr uint32_t Q_TILE = BQ * 2 * HD;        // both parts of a tile's queries: HD 128 part by part, HD 64 side by side in a row of 128 bytes
    static constexpr uint32_t PAGE_BYTES = PAGE * HD, V_BYTES = 2 * PAGE_BYTES, V_BLOCK = PAGE * 128;
    static constexpr uint32_t Q0 = 0, K0 = TILES * Q_TILE, V0 = K0 + K_STAGES * PAGE_BYTES, RAW0 = V0 + V_STAGES * V_BYTES, BARS = RAW0 + RAW_STAGES * PAGE_BYTES;
    static constexpr int N_BARS = TILES + 2 * K_STAGES + 2 * RAW_STAGES + 2 * V_STAGES + 3 * 2 * TILES;
    static constexpr uint32_t NANS = BARS + 8 * N_BARS + 16;          // of each element, the first key taken out; whether there is one at all
    static constexpr size_t SMEM = NANS + 4 * HD + 16 + 1024;
    // SPLIT: a block's sums, over everything before the barriers; rows begin four banks apart
    static constexpr int PARK_ROW = HD + 4;
    static constexpr uint32_t PARK_ML = TILES * BQ * PARK_ROW * 4;
    static_assert(PARK_ML + TILES * BQ * 8 <= BARS, "the sums lie over the operands");
};

// HD: the head size, or (not FULL) what it is rounded up to.  Keys and queries have zeros behind d, values anything: their products are columns of O that nobody reads.
// SPLIT: the pages are walked by a cluster of blocks (along x), a range each, whose sums meet in distributed shared memory.
template <int HD, bool FULL, bool SPLIT>
__global__ void __launch_bounds__(THREADS, 1) attention_cache8_tc_kernel(const __grid_constant__ CUtensorMap map_k, const TcParams p) {
    using S = Shape<HD>;
    const int d = FULL ? HD : p.d;
    const uint32_t v_page = FULL ? S::PAGE_BYTES : (uint32_t)(PAGE * p.d);
    constexpr uint32_t IDESC_QK = (1u << 4) | ((uint32_t)(PAGE >> 3) << 17) | ((uint32_t)(BQ >> 4) << 24);                      // e4m3, both K-major
    constexpr uint32_t IDESC_PV = (1u << 4) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(BQ >> 4) << 24);           // halves, V MN-major
    constexpr uint32_t O_COL = TILES * 2 * PAGE;           // S of tile t, buffer b at (2 t + b) * 64; O of tile t behind them
    extern __shared__ uint8_t smem_raw[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_wait();                                            // before tensor memory is taken: a block of an earlier kernel never waits for what this one holds
    const int seq = blockIdx.z, ranges = SPLIT ? p.ranges : 1, kvh = SPLIT ? blockIdx.x / ranges : blockIdx.x, range = SPLIT ? blockIdx.x % ranges : 0, group = p.nq / p.nkv;
    const int start = p.seq_start[seq], rows_all = (p.seq_start[seq + 1] - start) * group, past = p.seq_past[seq];
    const int row0 = ((int)gridDim.y - 1 - (int)blockIdx.y) * (TILES * BQ);              // the longest walks first
    if (row0 >= rows_all) return;                          // uniform for the block
    const int capacity = p.max_blocks * PAGE;
    int rows[TILES], n_tiles[TILES];                       // of each tile: rows that are there, pages they see
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
        rows[t] = max(0, min(BQ, rows_all - row0 - t * BQ));
        n_tiles[t] = rows[t] ? (min(past + (row0 + t * BQ + rows[t] - 1) / group + 1, capacity) + PAGE - 1) / PAGE : 0;
    }
    int page0 = 0;                                         // the block's first page; what follows counts from there
    if (SPLIT) {
        const int each = max(LEAST_PAGES, (max(n_tiles[0], n_tiles[1]) + ranges - 1) / ranges);
        page0 = range * each;
#pragma unroll
        for (int t = 0; t < TILES; ++t) n_tiles[t] = max(0, min(each, n_tiles[t] - page0));
    }
    const int n = max(n_tiles[0], n_tiles[1]);
    const int end = min(past + (min(rows_all, row0 + TILES * BQ) - 1) / group + 1, capacity);          // keys that any row sees
    const int* table = p.block_table + (size_t)seq * p.max_blocks;
    auto block_of = [&](int j) { return (size_t)min(max(table[page0 + j], 0), p.n_pages - 1) * p.nkv + kvh; };

    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    const uint32_t bars = base + S::BARS;
    const uint32_t q_full = bars, k_full = q_full + 8 * TILES, k_empty = k_full + 8 * K_STAGES, raw_full = k_empty + 8 * K_STAGES, raw_empty = raw_full + 8 * RAW_STAGES;
    const uint32_t v_full = raw_empty + 8 * RAW_STAGES, v_empty = v_full + 8 * V_STAGES, s_full = v_empty + 8 * V_STAGES, p_full = s_full + 16 * TILES, pv_full = p_full + 16 * TILES;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem_raw + (base - raw) + S::BARS + 8 * S::N_BARS);
    int* first_nan = reinterpret_cast<int*>(smem_raw + (base - raw) + S::NANS);
    volatile int* some_nan = first_nan + HD;
    for (int i = threadIdx.x; i <= HD; i += THREADS) first_nan[i] = i < HD ? 0x7fffffff : 0;
    int* status = p.status;
    if (threadIdx.x == 0) {
        prefetch_tensor_map(&map_k);
        for (int i = 0; i < TILES; ++i) mbar_init(q_full + 8 * i, 4);
        for (int i = 0; i < K_STAGES; ++i) { mbar_init(k_full + 8 * i, 1); mbar_init(k_empty + 8 * i, 1); }
        for (int i = 0; i < RAW_STAGES; ++i) { mbar_init(raw_full + 8 * i, 1); mbar_init(raw_empty + 8 * i, 4); }
        for (int i = 0; i < V_STAGES; ++i) { mbar_init(v_full + 8 * i, 4); mbar_init(v_empty + 8 * i, 1); }
        for (int i = 0; i < 2 * TILES; ++i) { mbar_init(s_full + 8 * i, 1); mbar_init(p_full + 8 * i, 4); mbar_init(pv_full + 8 * i, 1); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    pdl_launch_dependents();

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp == 0) {
            if (lane == 0) {
                for (int j = 0; j < n; ++j) {
                    const size_t block = block_of(j);
                    const int ks = j % K_STAGES, rs = j % RAW_STAGES;
                    if (!wait(k_empty + 8 * ks, ((uint32_t)(j / K_STAGES) & 1u) ^ 1u, status, 1)) break;
                    mbar_expect_tx(k_full + 8 * ks, S::PAGE_BYTES);
                    tma_load_2d(base + S::K0 + ks * S::PAGE_BYTES, &map_k, k_full + 8 * ks, 0, (int)(block * PAGE));
                    if (!wait(raw_empty + 8 * rs, ((uint32_t)(j / RAW_STAGES) & 1u) ^ 1u, status, 1)) break;
                    mbar_expect_tx(raw_full + 8 * rs, v_page);
                    bulk_load(base + S::RAW0 + rs * S::PAGE_BYTES, p.v + block * v_page, v_page, raw_full + 8 * rs);
                }
            }
        } else if (warp == 1) {
            const uint32_t one = elect_one();
            const uint64_t q_desc0 = operand_desc(base + S::Q0), k_desc0 = HD == 128 ? operand_desc(base + S::K0) : operand_desc_64(base + S::K0);
            const uint64_t v_desc0 = operand_desc_mn(base + S::V0, S::V_BLOCK);
            auto issue_scores = [&](int t, int j) {
                const int s = j % K_STAGES;
                tc_fence_after();
                const uint32_t acc = tmem_base + (uint32_t)((2 * t + (j & 1)) * PAGE);
#pragma unroll
                for (int part = 0; part < 2; ++part)
#pragma unroll
                    for (int ks = 0; ks < HD / 32; ++ks)
                        mma_scores(acc, q_desc0 + (uint64_t)((t * S::Q_TILE + part * (HD == 128 ? BQ * 128 : 64) + ks * 32) >> 4),
                                   k_desc0 + (uint64_t)((s * S::PAGE_BYTES + ks * 32) >> 4), IDESC_QK, part + ks > 0 ? 1u : 0u, one);
                commit_one(s_full + 8 * (2 * t + (j & 1)), one);
            };
            bool ok = n > 0 && wait_warp(k_full, 0, status, 2);
#pragma unroll
            for (int t = 0; t < TILES; ++t)
                if (ok && n_tiles[t] > 0) {
                    ok = wait_warp(q_full + 8 * t, 0, status, 2);
                    if (ok) issue_scores(t, 0);
                }
            if (ok) commit_one(k_empty, one);
            for (int j = 0; j < n && ok; ++j) {
                const int s = j % V_STAGES, b = j & 1, next = (j + 1) % K_STAGES;
                if (j + 1 < n) ok = wait_warp(k_full + 8 * next, (uint32_t)((j + 1) / K_STAGES) & 1u, status, 2);
#pragma unroll
                for (int t = 0; t < TILES; ++t) {
                    if (ok && j + 1 < n_tiles[t]) {
                        // the buffer holds P of page j - 1 until its P V is complete
                        if (j > 0) ok = wait_warp(pv_full + 8 * (2 * t + (b ^ 1)), (uint32_t)((j - 1) >> 1) & 1u, status, 2);
                        if (ok) issue_scores(t, j + 1);
                    }
                    if (ok && j < n_tiles[t]) {
                        ok = wait_warp(p_full + 8 * (2 * t + b), (uint32_t)(j >> 1) & 1u, status, 2) && wait_warp(v_full + 8 * s, (uint32_t)(j / V_STAGES) & 1u, status, 2);
                        if (!ok) continue;
                        tc_fence_after();
#pragma unroll
                        for (int ks = 0; ks < PAGE / 16; ++ks)
                            mma_values(tmem_base + O_COL + (uint32_t)(t * HD), tmem_base + (uint32_t)((2 * t + b) * PAGE + ks * 8),
                                       v_desc0 + (uint64_t)((s * S::V_BYTES + ks * (16 * 128)) >> 4), IDESC_PV, j + ks > 0 ? 1u : 0u, one);
                        commit_one(pv_full + 8 * (2 * t + b), one);
                    }
                }
                if (!ok) break;
                if (j + 1 < n) commit_one(k_empty + 8 * next, one);
                commit_one(v_empty + 8 * s, one);
            }
        }
    } else if (warp < 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        // 16 bytes of a key's values become 32: two 16-byte pieces of the row's 128 bytes in a block of 64 elements.  Neighbours take the pieces in turns, so that the
        // lanes that write together meet all banks.
        const int thread = threadIdx.x - 128;
        constexpr int EACH = PAGE * (HD / 16) / 128;       // pieces of a page that a thread converts, at most
        const int pieces = d / 16;                         // of a key
        int keys[EACH], columns[EACH];
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            keys[i] = (thread + i * 128) / pieces;         // PAGE or more: none
            columns[i] = (thread + i * 128) % pieces;
        }
        const int all_see = past + row0 / group + 1;       // keys that every row sees
        bool ok = true;
        for (int j = 0; j < n && ok; ++j) {
            const int rs = j % RAW_STAGES, vs = j % V_STAGES;
            ok = wait_warp(raw_full + 8 * rs, (uint32_t)(j / RAW_STAGES) & 1u, status, 4) && wait_warp(v_empty + 8 * vs, ((uint32_t)(j / V_STAGES) & 1u) ^ 1u, status, 4);
            if (!ok) break;
            uint4 v[EACH];
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                if (!FULL) v[i] = make_uint4(0, 0, 0, 0);
                if (!FULL && keys[i] >= PAGE) continue;
                v[i] = load16(base + S::RAW0 + rs * S::PAGE_BYTES + (thread + i * 128) * 16);
                if ((page0 + j) * PAGE + keys[i] >= end) v[i] = make_uint4(0, 0, 0, 0);       // behind the last key lies anything, NaN too
            }
            if ((page0 + j) * PAGE + PAGE > all_see) {
                // FULL: piece by piece, through shared memory; the others: all at once, in registers.  What never runs decides how the rest is scheduled: 4,096 tokens of heads of
                // 128 take 752 us so, the other way 821; 2 x 2,000 of heads of 96 take 94 us, the other way 107.
                uint32_t some = 0;
#pragma unroll
                for (int i = 0; i < EACH; ++i) {
                    const uint32_t here = any_nan(v[i].x) | any_nan(v[i].y) | any_nan(v[i].z) | any_nan(v[i].w);
                    some |= here;
                    if (FULL && here) {
                        const uint32_t at = base + S::RAW0 + rs * S::PAGE_BYTES + (thread + i * 128) * 16;
                        take_out_nan(at, first_nan + 16 * columns[i], (page0 + j) * PAGE + keys[i]);
                        v[i] = load16(at);
                        *some_nan = 1;
                    }
                }
                if (!FULL && some) {
#pragma unroll
                    for (int i = 0; i < EACH; ++i) take_out_nan(v[i], first_nan + 16 * columns[i], (page0 + j) * PAGE + keys[i]);
                    *some_nan = 1;
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(raw_empty + 8 * rs);
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                if (!FULL && keys[i] >= PAGE) continue;
                const int key = keys[i], c = columns[i], swap = (c >> 2) & 1;
                const uint32_t row = base + S::V0 + vs * S::V_BYTES + (c >> 2) * S::V_BLOCK + key * 128;
                const uint4 lo = make_uint4(halves(v[i].x), halves(v[i].x >> 16), halves(v[i].y), halves(v[i].y >> 16));
                const uint4 hi = make_uint4(halves(v[i].z), halves(v[i].z >> 16), halves(v[i].w), halves(v[i].w >> 16));
                const int at = 2 * (c & 3);
                store16(row + (uint32_t)(((at + swap) ^ (key & 7)) << 4), swap ? hi : lo);
                store16(row + (uint32_t)(((at + 1 - swap) ^ (key & 7)) << 4), swap ? lo : hi);
            }
            fence_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(v_full + 8 * vs);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
        const int t = (warp - 8) >> 2, quarter = warp & 3, r = quarter * 32 + lane, my_rows = t ? rows[1] : rows[0], my_tiles = t ? n_tiles[1] : n_tiles[0];
        const int mine = row0 + t * BQ + min(r, max(my_rows - 1, 0));        // rows beyond the last act as the last
        const int token = start + mine / group, head = kvh * group + mine % group;
        const int qpos = past + mine / group, first_qpos = past + (row0 + t * BQ) / group;
        const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16);
        float factor = 0.f;
        if (my_rows) {
            // the row as two 8-bit numbers an element, 2^-shift of it: its largest lies in [2^7, 2^8)
            const uint4* src = reinterpret_cast<const uint4*>(p.q + ((size_t)token * p.nq + head) * d);
            uint4 x[HD / 8];
            float most = 0.f;
#pragma unroll
            for (int i = 0; i < HD / 8; ++i) {
                x[i] = FULL || 8 * i < d ? src[i] : make_uint4(0, 0, 0, 0);
                const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[k]));
                    most = max3(most, fabsf(f.x), fabsf(f.y));
                }
            }
            int shift = (__float_as_int(most) >> 23) - 127 - 7;
            if (!(most >= 0x1p-100f && most < INFINITY)) shift = 0;
            const float by = exp2f((float)-shift);
            factor = exp2f((float)shift) * p.scale * LOG2E;
            const uint32_t row = base + S::Q0 + t * S::Q_TILE + r * 128;
#pragma unroll
            for (int c = 0; c < HD / 16; ++c) {            // 16 elements: 16 bytes of each part
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    const uint4 y = x[2 * c + (h >> 1)];
                    const uint32_t w0 = (h & 1) ? y.z : y.x, w1 = (h & 1) ? y.w : y.y;
                    const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w0)), b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w1));
                    const float f[4] = {nan_if_infinite(a.x * by), nan_if_infinite(a.y * by), nan_if_infinite(b.x * by), nan_if_infinite(b.y * by)};
                    hi[h] = pack4(f[0], f[1], f[2], f[3]);
                    const float2 g0 = floats(hi[h]), g1 = floats(hi[h] >> 16);
                    lo[h] = pack4(f[0] - g0.x, f[1] - g0.y, f[2] - g1.x, f[3] - g1.y);
                }
                const uint32_t at0 = (uint32_t)((c ^ (r & 7)) << 4), at1 = HD == 128 ? (uint32_t)(BQ * 128) + at0 : (uint32_t)(((c + 4) ^ (r & 7)) << 4);
                store16(row + at0, make_uint4(hi[0], hi[1], hi[2], hi[3]));
                store16(row + at1, make_uint4(lo[0], lo[1], lo[2], lo[3]));
            }
            fence_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full + 8 * t);
        }
        float m_run = -INFINITY, l_run = 0.f;
        bool ok = true;
        size_t block = my_tiles > 0 ? block_of(0) : 0;
        float k_scale = my_tiles > 0 ? p.k_scale[block] : 1.f, v_scale = my_tiles > 0 ? p.v_scale[block] : 1.f;
        for (int j = 0; j < my_tiles && ok; ++j) {
            const int b = j & 1;
            const float scale2 = fmaxf(factor * k_scale, 0x1p-125f), lift = log2f(v_scale), out_of = 1.f / v_scale;
            if (j + 1 < my_tiles) {                      // the next page's scales on their way
                block = block_of(j + 1);
                k_scale = p.k_scale[block];
                v_scale = p.v_scale[block];
            }
            ok = wait_warp(s_full + 8 * (2 * t + b), (uint32_t)(j >> 1) & 1u, status, 3);
            if (!ok) break;
            tc_fence_after();
            const uint32_t s_addr = lane_addr + (uint32_t)((2 * t + b) * PAGE);
            uint32_t v[2][32];
            tmem_load32_start(s_addr, v[0]);
            tmem_load32_start(s_addr + 32, v[1]);
            tmem_wait_ld();
            const int pos0 = (page0 + j) * PAGE;
            if (pos0 + PAGE - 1 > first_qpos) {            // some row of the tile does not see the whole page
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int c = 0; c < 32; ++c)
                        if (pos0 + q * 32 + c > qpos) v[q][c] = 0xff800000u;   // -inf
            }
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            const uint64_t scale22 = pair_f32(scale2, scale2);
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int c = 0; c < 32; c += 2) mx[(c >> 1) & 3] = max3(mx[(c >> 1) & 3], __uint_as_float(v[q][c]), __uint_as_float(v[q][c + 1]));
            const float m_tile = fmaf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), scale2, lift);
            const bool moves = m_tile > m_run + RESCALE_STEP;
            const float m_new = moves ? m_tile : m_run, m_use = m_new == -INFINITY ? 0.f : m_new;
            const float alpha = moves ? fast_exp2(m_run - m_use) : 1.f;
            if (j > 0 && __any_sync(0xffffffffu, moves)) {
                // O may be scaled once P V of the page before is complete; a softmax warp waits for P V only here and at the end
                ok = wait_warp(pv_full + 8 * (2 * t + ((j - 1) & 1)), (uint32_t)((j - 1) >> 1) & 1u, status, 3);
                if (!ok) break;
                tc_fence_after();
#pragma unroll 1
                for (int c0 = 0; c0 < d; c0 += 32) {
                    uint32_t o[32];
                    tmem_load32(lane_addr + O_COL + (uint32_t)(t * HD + c0), o);
#pragma unroll
                    for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * alpha);
                    tmem_store32(lane_addr + O_COL + (uint32_t)(t * HD + c0), o);
                }
                tmem_wait_st();
            }
            // P as halves, two keys to a column, over this row's scores (they are in registers)
            uint64_t sum2[2] = {0ull, 0ull};
            const float below = lift - m_use + LIFT;
            const uint64_t below2 = pair_f32(below, below);
            uint32_t packed[32];
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int c = 0; c < 32; c += 2) {
                    float x0, x1;
                    unpair_f32(fma2(pair_u32(v[q][c], v[q][c + 1]), scale22, below2), x0, x1);
                    const float e0 = fast_exp2(x0), e1 = fast_exp2(x1);
                    sum2[(c >> 1) & 1] = add2(sum2[(c >> 1) & 1], pair_f32(e0, e1));
                    packed[q * 16 + (c >> 1)] = pack_half(e0, e1);
                }
            tmem_store32(s_addr, packed);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + 8 * (2 * t + b));
            float sum[4];
            unpair_f32(sum2[0], sum[0], sum[2]);
            unpair_f32(sum2[1], sum[1], sum[3]);
            l_run = fmaf((sum[0] + sum[1]) + (sum[2] + sum[3]), out_of, l_run * alpha);
            m_run = m_new;
        }
        const int last = my_tiles - 1;
        // the elements of this row that a value which is no number reaches
        auto hand_on_nan = [&](uint32_t (&o)[32], int c0) {
            if (*some_nan)
#pragma unroll
                for (int c = 0; c < 32; ++c)
                    if (first_nan[c0 + c] <= qpos) o[c] = 0x7fffffffu;
        };
        const bool done = last >= 0 && ok && wait_warp(pv_full + 8 * (2 * t + (last & 1)), (uint32_t)(last >> 1) & 1u, status, 3);
        if (SPLIT) asm volatile("bar.sync 1, 256;" ::: "memory");      // both tiles' products are complete: the operands' place is free
        if (SPLIT) {
            tc_fence_after();
            float* park = reinterpret_cast<float*>(smem_raw + (base - raw)) + (t * BQ + r) * S::PARK_ROW;
            float* ml = reinterpret_cast<float*>(smem_raw + (base - raw) + S::PARK_ML) + 2 * (t * BQ + r);
            ml[0] = done ? m_run : -INFINITY;
            ml[1] = done ? l_run : 0.f;
#pragma unroll 1
            for (int c0 = 0; c0 < HD; c0 += 32) {
                uint32_t o[32];
                if (done) {
                    tmem_load32(lane_addr + O_COL + (uint32_t)(t * HD + c0), o);
                    hand_on_nan(o, c0);
                } else {
#pragma unroll
                    for (int c = 0; c < 32; ++c) o[c] = 0u;
                }
#pragma unroll
                for (int c = 0; c < 32; c += 4) *reinterpret_cast<uint4*>(park + c0 + c) = make_uint4(o[c], o[c + 1], o[c + 2], o[c + 3]);
                __syncwarp();
            }
        } else if (done) {
            tc_fence_after();
            const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
            __nv_bfloat16* dst = p.out + ((size_t)token * p.nq + head) * d;
#pragma unroll 1
            for (int c0 = 0; c0 < d; c0 += 32) {
                uint32_t o[32];
                tmem_load32(lane_addr + O_COL + (uint32_t)(t * HD + c0), o);
                hand_on_nan(o, c0);
                if (r < my_rows) {
#pragma unroll
                    for (int c = 0; c < 32; c += 8) {
                        if (!FULL && c0 + c >= d) break;
                        uint4 w;
                        w.x = pack_bf16(__uint_as_float(o[c]) * inv, __uint_as_float(o[c + 1]) * inv);
                        w.y = pack_bf16(__uint_as_float(o[c + 2]) * inv, __uint_as_float(o[c + 3]) * inv);
                        w.z = pack_bf16(__uint_as_float(o[c + 4]) * inv, __uint_as_float(o[c + 5]) * inv);
                        w.w = pack_bf16(__uint_as_float(o[c + 6]) * inv, __uint_as_float(o[c + 7]) * inv);
                        *reinterpret_cast<uint4*>(dst + c0 + c) = w;
                    }
                }
                __syncwarp();
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (*(volatile int*)status != 0) {                     // a wait gave up: let copies in flight land before the block leaves
        const unsigned long long t0 = global_timer();
        while (global_timer() - t0 < 2000000ull) __nanosleep(1000);
    }
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512) : "memory");
    if (SPLIT) {
        cluster_sync_all();
        // the block of rank i finishes rows i, i + ranges, ...: LANES lanes a row, four columns each
        constexpr int LANES = HD / 4, AT_ONCE = THREADS / LANES;
        const int c = threadIdx.x % LANES * 4;
        for (int i = threadIdx.x / LANES; i * ranges + range < TILES * BQ; i += AT_ONCE) {
            const int r = i * ranges + range, mine = row0 + r;
            if (mine >= rows_all) break;
            float m = -INFINITY, l = 0.f, mk[MAX_RANGES], lk[MAX_RANGES], sum[4] = {};
            float4 o[MAX_RANGES];
#pragma unroll
            for (int k = 0; k < MAX_RANGES; ++k)
                if (k < ranges) {
                    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(mk[k]), "=f"(lk[k]) : "r"(map_to_cta(base + S::PARK_ML + 8 * r, k)) : "memory");
                    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(o[k].x), "=f"(o[k].y), "=f"(o[k].z), "=f"(o[k].w)
                                 : "r"(map_to_cta(base + (uint32_t)(r * S::PARK_ROW + c) * 4, k)) : "memory");
                }
#pragma unroll
            for (int k = 0; k < MAX_RANGES; ++k)
                if (k < ranges) m = fmaxf(m, mk[k]);
#pragma unroll
            for (int k = 0; k < MAX_RANGES; ++k)
                if (k < ranges) {
                    // a range without keys has nothing; one whose sums are NaN hands that on
                    const float by = mk[k] == -INFINITY ? 1.f : fast_exp2(mk[k] - m);
                    l = fmaf(lk[k], by, l);
                    sum[0] = fmaf(o[k].x, by, sum[0]); sum[1] = fmaf(o[k].y, by, sum[1]); sum[2] = fmaf(o[k].z, by, sum[2]); sum[3] = fmaf(o[k].w, by, sum[3]);
                }
            const float inv = l == 0.f ? 0.f : 1.f / l;
            if (FULL || c < d)
                *reinterpret_cast<uint2*>(p.out + ((size_t)(start + mine / group) * p.nq + kvh * group + mine % group) * d + c) =
                    make_uint2(pack_bf16(sum[0] * inv, sum[1] * inv), pack_bf16(sum[2] * inv, sum[3] * inv));
        }
        cluster_sync_all();                                // nobody leaves while its sums are read
    }
}

template <int HD, bool FULL, bool SPLIT> int launch(const void* k, const TcParams& p, int n_seqs, int max_q_len, cudaStream_t stream) {
    EncodeFn encode = encode_fn();
    if (!encode) QT_FAIL(QT_ERR_LAUNCH, "attention_cache8_tc: the driver does not offer cuTensorMapEncodeTiled");
    CUtensorMap map_k;
    const cuuint64_t dims[2] = {(cuuint64_t)p.d, (cuuint64_t)p.n_pages * p.nkv * PAGE}, strides[1] = {(cuuint64_t)p.d};      // zeros behind d
    const cuuint32_t box[2] = {HD, PAGE}, elem[2] = {1, 1};
    const CUresult rc = encode(&map_k, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(k), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                               HD == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS) QT_FAIL(QT_ERR_LAUNCH, "attention_cache8_tc: cuTensorMapEncodeTiled failed with %d", (int)rc);
    const cudaError_t raised = raise_shared<attention_cache8_tc_kernel<HD, FULL, SPLIT>>((int)Shape<HD>::SMEM);
    if (raised != cudaSuccess) QT_FAIL(QT_ERR_LAUNCH, "attention_cache8_tc: cannot raise shared memory: %s", cudaGetErrorString(raised));
    const long long blocks = ((long long)max_q_len * (p.nq / p.nkv) + TILES * BQ - 1) / (TILES * BQ);
    QT_REQUIRE(blocks <= 65535, "attention_cache8_tc: %d tokens of a sequence are too many", max_q_len);
    const dim3 grid((unsigned)(p.nkv * p.ranges), (unsigned)blocks, n_seqs);
    if (SPLIT) launch_kernel_cluster(attention_cache8_tc_kernel<HD, FULL, SPLIT>, grid, dim3(THREADS), Shape<HD>::SMEM, stream, (unsigned)p.ranges, map_k, p);
    else launch_kernel(attention_cache8_tc_kernel<HD, FULL, SPLIT>, grid, dim3(THREADS), Shape<HD>::SMEM, stream, map_k, p);
    QT_CHECK_LAUNCH("attention_cache8_tc");
    return QT_OK;
}

template <int HD, bool FULL> int launch_ranges(const void* k, const TcParams& p, int n_seqs, int max_q_len, cudaStream_t stream) {
    return p.ranges > 1 ? launch<HD, FULL, true>(k, p, n_seqs, max_q_len, stream) : launch<HD, FULL, false>(k, p, n_seqs, max_q_len, stream);
}

}  // namespace

// Packed bfloat16 queries [n_tokens, nq, d] of sequences whose keys, this call's own among them, are in the cache; causal.  d is a multiple of 16 up to 128.  A block's
// pages are walked by a cluster of `ranges` blocks.
extern "C" int qt_attention_prefill_cache8_tc(const Cache8Call* call) {
    const Cache8Call& c = *call;
    if (c.n_seqs == 0 || c.max_q_len == 0) return QT_OK;
    QT_REQUIRE(c.dtype == QT_BF16 && c.d > 0 && c.d <= 128 && c.d % 16 == 0, "attention_prefill_cache8_tc: bfloat16 heads in steps of 16 up to 128, not %d (type %d)", c.d, c.dtype);
    QT_REQUIRE(c.nq > 0 && c.nkv > 0 && c.nq % c.nkv == 0 && c.ranges >= 1 && c.ranges <= MAX_RANGES && c.nkv <= 0x7fffffff / MAX_RANGES && c.max_blocks > 0 && c.max_blocks <= 0x7fffffff / PAGE && c.n_pages > 0 && c.n_seqs > 0 &&
                   c.n_seqs <= 65535 && c.max_q_len > 0 && (long long)c.max_q_len * (c.nq / c.nkv) <= 0x7fffffff - TILES * BQ &&
                   (long long)c.n_pages * c.nkv <= 0x7fffffff / PAGE,
               "attention_prefill_cache8_tc: bad sizes nq=%d nkv=%d, %d pages, %d sequences of up to %d tokens", c.nq, c.nkv, c.n_pages, c.n_seqs, c.max_q_len);
    QT_REQUIRE(c.status != nullptr && c.scale > 0., "attention_prefill_cache8_tc: a status word and a positive scale are required");
    QT_REQUIRE((((uintptr_t)c.q | (uintptr_t)c.k | (uintptr_t)c.v | (uintptr_t)c.out) & 15) == 0, "attention_prefill_cache8_tc: operands must be 16-byte aligned");
    const TcParams p{(const __nv_bfloat16*)c.q, (__nv_bfloat16*)c.out, (const uint8_t*)c.v, c.k_scale, c.v_scale, c.block_table, c.max_blocks, c.n_pages, c.seq_start, c.seq_past,
                     c.nq, c.nkv, c.d, c.ranges, (float)c.scale, c.status};
    cudaStream_t s = (cudaStream_t)c.stream;
    if (c.d == 64) return launch_ranges<64, true>(c.k, p, c.n_seqs, c.max_q_len, s);
    if (c.d == 128) return launch_ranges<128, true>(c.k, p, c.n_seqs, c.max_q_len, s);
    return c.d < 64 ? launch_ranges<64, false>(c.k, p, c.n_seqs, c.max_q_len, s) : launch_ranges<128, false>(c.k, p, c.n_seqs, c.max_q_len, s);
}

QT_DEFINE_LAST_ERROR(attention_cache8_tc)
