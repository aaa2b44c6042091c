// y = x W^T for a weight of 8-bit numbers with a scale for each block of 128 x 128, and what makes rows and weights such numbers.
//
//   s_x[g, m] = max(amax_{k in g} |x[m, k]| * r, 2^-100),  x8[m, k] = e4m3(x[m, k] / s_x[g, m])        g: 128 columns, r: the float next to 1 / 448
//   y[m, n]   = sum_g s_x[g, m] s_w[n / 128, g] sum_{k in g} x8[m, k] w8[n, k]
//
// Sums are held in 32 bits; y is rounded once.
#include "fp8.cuh"
#include "tc_common.cuh"

#include <algorithm>

using namespace qt;
using namespace qt_fp8;
using namespace qt_tc;

namespace {

constexpr float LEAST_SCALE = 0x1p-100f, PER_TOP = 1.f / TOP;

// ----------------------------------------------------------------------------- rows in 8 bits
// A warp a row and 128 columns, four columns a lane.  Scales as [group, row].
template <typename T>
__global__ void __launch_bounds__(256) quantise_rows_kernel(const T* x, uint8_t* values, float* scales, int rows, int k, int groups) {
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const long long unit = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (unit >= (long long)rows * groups) return;
    const int m = (int)(unit / groups), g = (int)(unit % groups), c0 = g * GROUP + lane * 4;
    const T* row = x + (size_t)m * k;
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = c0 + i < k ? to_float(row[c0 + i]) : 0.f;
    const float largest = warp_max(fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3]))));
    const float scale = fmaxf(__fmul_rn(largest, PER_TOP), LEAST_SCALE);
    if (lane == 0) scales[(size_t)g * rows + m] = scale;
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        const uint32_t two = pack2(__fdiv_rn(v[i], scale), __fdiv_rn(v[i + 1], scale));
        if (c0 + i < k) values[(size_t)m * k + c0 + i] = (uint8_t)two;
        if (c0 + i + 1 < k) values[(size_t)m * k + c0 + i + 1] = (uint8_t)(two >> 8);
    }
}

// A block a weight's block of 128 x 128: the same with one scale for all of it.
template <typename T>
__global__ void __launch_bounds__(256) quantise_weight_kernel(const T* w, uint8_t* values, float* scales, int n, int k) {
    __shared__ float most[8];
    pdl_launch_dependents();
    pdl_wait();
    const int n0 = blockIdx.y * GROUP, k0 = blockIdx.x * GROUP, col = k0 + (threadIdx.x & 127);
    float largest = 0.f;
    for (int r = n0 + (threadIdx.x >> 7); r < min(n, n0 + GROUP); r += 2)
        if (col < k) largest = fmaxf(largest, fabsf(to_float(w[(size_t)r * k + col])));
    largest = warp_max(largest);
    if ((threadIdx.x & 31) == 0) most[threadIdx.x >> 5] = largest;
    __syncthreads();
    largest = warp_max(most[threadIdx.x & 7]);
    const float scale = fmaxf(__fmul_rn(largest, PER_TOP), LEAST_SCALE);
    if (threadIdx.x == 0) scales[(size_t)blockIdx.y * gridDim.x + blockIdx.x] = scale;
    for (int r = n0 + (threadIdx.x >> 7); r < min(n, n0 + GROUP); r += 2)
        if (col < k) values[(size_t)r * k + col] = (uint8_t)pack2(__fdiv_rn(to_float(w[(size_t)r * k + col]), scale), 0.f);
}

// ----------------------------------------------------------------------------- the product, any sizes
// 64 x 64 outputs a block, 4 x 4 a thread, a group of K at a time in shared memory as floats.
template <typename T>
__global__ void __launch_bounds__(256) gemm_fp8_any_kernel(const uint8_t* x8, const float* x_scale, const uint8_t* w8, const float* w_scale, T* out, int rows,
                                                           int n, int k, int groups) {
    __shared__ float xs[32][65], ws[32][65];
    pdl_launch_dependents();
    pdl_wait();
    const int m0 = blockIdx.y * 64, n0 = blockIdx.x * 64, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    float total[4][4] = {};
    for (int g = 0; g < groups; ++g) {
        float part[4][4] = {};
        for (int k0 = g * GROUP; k0 < min(k, (g + 1) * GROUP); k0 += 32) {
            for (int i = threadIdx.x; i < 64 * 32; i += 256) {
                const int r = i >> 5, c = i & 31;
                xs[c][r] = m0 + r < rows && k0 + c < k ? floats(x8[(size_t)(m0 + r) * k + k0 + c]).x : 0.f;
                ws[c][r] = n0 + r < n && k0 + c < k ? floats(w8[(size_t)(n0 + r) * k + k0 + c]).x : 0.f;
            }
            __syncthreads();
            for (int c = 0; c < 32; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) part[i][j] = fmaf(xs[c][ty + 16 * i], ws[c][tx + 16 * j], part[i][j]);
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (m0 + ty + 16 * i < rows && n0 + tx + 16 * j < n)
                    total[i][j] = fmaf(part[i][j], x_scale[(size_t)g * rows + m0 + ty + 16 * i] * w_scale[(size_t)((n0 + tx + 16 * j) / GROUP) * groups + g], total[i][j]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (m0 + ty + 16 * i < rows && n0 + tx + 16 * j < n) out[(size_t)(m0 + ty + 16 * i) * n + n0 + tx + 16 * j] = from_float<T>(total[i][j]);
}

// ----------------------------------------------------------------------------- the product on tcgen05
// Both operands are K-major tiles of 128-byte rows (one group of K), four tcgen05.mma of 32 elements a group.  The scales belong to the sums of a group: these
// go to one of two accumulators in tensor memory, and while the next group's are formed in the other, the epilogue's threads read them and add them, times both
// scales, to sums in their registers.
constexpr int BM = 128;                                     // the instruction's M
constexpr uint32_t A_BYTES = BM * GROUP;

__device__ __forceinline__ void umma_fp8(uint32_t tmem_d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void prefetch_2d(const CUtensorMap* map, int c_inner, int c_outer) {
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global [%0, {%1, %2}];" ::"l"(map), "r"(c_inner), "r"(c_outer) : "memory");
}
// float accumulator, e4m3 operands, both K-major
template <int N> constexpr uint32_t FP8_IDESC = (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);

__device__ __forceinline__ void tmem_load16_start(uint32_t taddr, uint32_t (&v)[16]) {     // results are valid after tmem_wait_ld()
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr));
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
__device__ __forceinline__ float2 unpair(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}

struct GemmParams {
    const float* x_scale; const float* w_scale; void* out;
    int rows, n, groups;
    int groups_per_split;
    int wide;                                               // rows of the output begin at 32-byte boundaries
    int* status;
};

// Few rows.  The weight's rows are the instruction's M (a tile is one row of scale blocks), BX rows of x its N; a cluster's blocks take a range of K each and add
// their sums through distributed shared memory in the order of their ranks.  192 threads: warp 0 copies, warp 1 issues, warps 2 to 5 add up, a weight row a thread.
constexpr int FEW_THREADS = 192, PREFETCH = 16;
template <int BX> struct Few {
    static constexpr uint32_t STAGE_BYTES = A_BYTES + BX * GROUP;
    static constexpr int PARK = BM + 1;                     // floats from one column of parked sums to the next
    static size_t smem(int stages) { return (size_t)stages * STAGE_BYTES + 2 * BX * 4 + 8 * (2 * stages + 4) + 16 + 1024; }
};

template <int BX, typename TO>
__global__ void __launch_bounds__(FEW_THREADS) gemm_fp8_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const GemmParams p,
                                                                   int stages) {
    constexpr uint32_t STAGE_BYTES = Few<BX>::STAGE_BYTES, TMEM_COLS = 2 * BX < 32 ? 32 : 2 * BX, IDESC = FP8_IDESC<BX>;
    constexpr int PARK = Few<BX>::PARK;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t* smem = smem_raw + (base - raw);
    const uint32_t scales_at = stages * STAGE_BYTES, bars = base + scales_at + 2 * BX * 4;
    const uint32_t full0 = bars, empty0 = bars + 8 * stages, acc_full = empty0 + 8 * stages, acc_empty = acc_full + 16;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + (acc_empty + 16 - base));
    float* column_scale = reinterpret_cast<float*>(smem + scales_at);                       // [2][BX]

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = blockIdx.x, splits = gridDim.x, w0 = blockIdx.y * BM, x0 = blockIdx.z * BX;
    const int g_begin = split * p.groups_per_split, count = min(p.groups, g_begin + p.groups_per_split) - g_begin;      // >= 1: the host cuts so
    int* status = p.status;
    if (threadIdx.x == 0) {
        prefetch_tensor_map(&map_w);
        prefetch_tensor_map(&map_x);
        for (int s = 0; s < stages; ++s) { mbar_init(full0 + 8 * s, 1); mbar_init(empty0 + 8 * s, 1); }
        for (int s = 0; s < 2; ++s) { mbar_init(acc_full + 8 * s, 1); mbar_init(acc_empty + 8 * s, 4); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    pdl_launch_dependents();                                // not before the columns are this block's: a dependent's block must not take them first and wait
    float acc[BX];
#pragma unroll
    for (int c = 0; c < BX; ++c) acc[c] = 0.f;

    if (warp == 0) {
        if (lane == 0) {
            // while the kernels before this one run, the weight comes as far as the L2 cache (where they may still write it)
            for (int i = 0; i < min(count, PREFETCH); ++i) prefetch_2d(&map_w, (g_begin + i) * GROUP, w0);
            pdl_wait();
            for (int i = 0; i < count; ++i) {
                const int s = i % stages;
                if (i >= stages && !mbar_wait(empty0 + 8 * s, (uint32_t)(i / stages - 1) & 1u, status, 1)) break;
                mbar_expect_tx(full0 + 8 * s, STAGE_BYTES);
                const uint32_t dst = base + s * STAGE_BYTES;
                tma_load_2d(dst, &map_w, full0 + 8 * s, (g_begin + i) * GROUP, w0);
                tma_load_2d(dst + A_BYTES, &map_x, full0 + 8 * s, (g_begin + i) * GROUP, x0);
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            const uint64_t a_desc0 = operand_desc(base), b_desc0 = operand_desc(base + A_BYTES);
            for (int i = 0; i < count; ++i) {
                const int s = i % stages, b = i & 1;
                if (i >= 2 && !mbar_wait(acc_empty + 8 * b, (uint32_t)(i / 2 - 1) & 1u, status, 2)) break;
                if (!mbar_wait(full0 + 8 * s, (uint32_t)(i / stages) & 1u, status, 2)) break;
                tc_fence_after();
                const uint64_t step = (uint64_t)(s * (STAGE_BYTES >> 4));
#pragma unroll
                for (int k = 0; k < GROUP / 32; ++k) umma_fp8(tmem_base + b * BX, a_desc0 + step + 2 * k, b_desc0 + step + 2 * k, IDESC, k > 0 ? 1u : 0u);
                umma_commit(empty0 + 8 * s);
                umma_commit(acc_full + 8 * b);
            }
        }
    } else {
        const int quarter = warp & 3, column = (warp - 2) * 32 + lane;
        pdl_wait();                                         // the rows' scales come from the kernel before; the output may still be read by one
        const float* w_scale = p.w_scale + (size_t)blockIdx.y * p.groups;
        auto scale_of = [&](int g) { return column < BX && x0 + column < p.rows ? p.x_scale[(size_t)g * p.rows + x0 + column] * w_scale[g] : 0.f; };
        float mine = scale_of(g_begin);
        bool ok = true;                                     // a wait that gave up ends the work, not the way through the barriers
        for (int i = 0; i < count; ++i) {
            const int b = i & 1;
            float* scale = column_scale + b * BX;
            if (column < BX) scale[column] = mine;
            if (i + 1 < count) mine = scale_of(g_begin + i + 1);
            asm volatile("bar.sync 1, 128;" ::: "memory");
            ok = ok && mbar_wait(acc_full + 8 * b, (uint32_t)(i / 2) & 1u, status, 3);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) continue;
            tc_fence_after();
            const uint32_t at = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(b * BX);
#pragma unroll
            for (int c0 = 0; c0 < BX; c0 += 16) {
                uint32_t v[16];
                tmem_load16(at + (uint32_t)c0, v);
                if (c0 + 16 == BX) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(acc_empty + 8 * b);
                }
#pragma unroll
                for (int c = 0; c < 16; c += 4) {
                    const float4 by = *reinterpret_cast<const float4*>(scale + c0 + c);
                    acc[c0 + c] = fmaf(__uint_as_float(v[c]), by.x, acc[c0 + c]);
                    acc[c0 + c + 1] = fmaf(__uint_as_float(v[c + 1]), by.y, acc[c0 + c + 1]);
                    acc[c0 + c + 2] = fmaf(__uint_as_float(v[c + 2]), by.z, acc[c0 + c + 2]);
                    acc[c0 + c + 3] = fmaf(__uint_as_float(v[c + 3]), by.w, acc[c0 + c + 3]);
                }
            }
        }
        const int row = quarter * 32 + lane;
        if (splits == 1) {
            if (w0 + row < p.n) {
#pragma unroll
                for (int c = 0; c < BX; ++c)
                    if (x0 + c < p.rows) ((TO*)p.out)[(size_t)(x0 + c) * p.n + w0 + row] = from_float<TO>(acc[c]);
            }
        } else {
            float* park = reinterpret_cast<float*>(smem);   // over the ring: every product that read it is complete
#pragma unroll
            for (int c = 0; c < BX; ++c) park[c * PARK + row] = acc[c];
        }
    }
    tc_fence_before();
    __syncthreads();
    if (*(volatile int*)status != 0) {                      // a wait gave up: let copies in flight land before the block leaves
        const unsigned long long t0 = global_timer();
        while (global_timer() - t0 < 2000000ull) __nanosleep(1000);
    }
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
    if (splits > 1) {
        cluster_sync_all();
        // the block of rank r finishes columns r, r + splits, ...: the ranks' sums one after the other
        const uint32_t park = base;
        for (int i = threadIdx.x; i < (BX / splits + 1) * BM; i += FEW_THREADS) {
            const int c = (i >> 7) * splits + split, row = i & (BM - 1);
            if (c >= BX || x0 + c >= p.rows) break;
            float sum = 0.f;
            for (int r = 0; r < splits; ++r) {
                float v;
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(map_to_cta(park + (uint32_t)(c * PARK + row) * 4, r)) : "memory");
                sum += v;
            }
            if (w0 + row < p.n) ((TO*)p.out)[(size_t)(x0 + c) * p.n + w0 + row] = from_float<TO>(sum);
        }
        cluster_sync_all();                                 // nobody leaves while its sums are read
    }
}

// Many rows.  128 rows of x are the instruction's M, 256 weight rows its N; eight warps add up, a row of x and 128 weight rows (one scale block) a thread.  One block
// an SM walks tiles; 320 threads: warp 0 copies, warp 1 issues, warps 2 to 9 add up and store.
constexpr int BN = 256, MANY_THREADS = 320, MANY_STAGES = 4;
constexpr uint32_t B_BYTES = BN * GROUP, MANY_STAGE_BYTES = A_BYTES + B_BYTES;
constexpr int RASTER = 8;

__device__ __forceinline__ void tile_of(int t, int w_tiles, int x_tiles, int& w, int& x) {     // groups of RASTER weight tiles, in a group rows of tiles
    const int per_group = RASTER * x_tiles, group = t / per_group, r = t % per_group, first = group * RASTER, width = min(RASTER, w_tiles - first);
    w = first + r % width;
    x = r / width;
}

template <typename TO>
__global__ void __launch_bounds__(MANY_THREADS, 1) gemm_fp8_many_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const GemmParams p) {
    constexpr uint32_t IDESC = FP8_IDESC<BN>, TMEM_COLS = 2 * BN;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t* smem = smem_raw + (base - raw);
    const uint32_t bars = base + MANY_STAGES * MANY_STAGE_BYTES;
    const uint32_t full0 = bars, empty0 = bars + 8 * MANY_STAGES, acc_full = empty0 + 8 * MANY_STAGES, acc_empty = acc_full + 16;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + (acc_empty + 16 - base));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int w_tiles = (p.n + BN - 1) / BN, x_tiles = (p.rows + BM - 1) / BM, tiles = w_tiles * x_tiles;
    int* status = p.status;
    if (threadIdx.x == 0) {
        prefetch_tensor_map(&map_w);
        prefetch_tensor_map(&map_x);
        for (int s = 0; s < MANY_STAGES; ++s) { mbar_init(full0 + 8 * s, 1); mbar_init(empty0 + 8 * s, 1); }
        for (int s = 0; s < 2; ++s) { mbar_init(acc_full + 8 * s, 1); mbar_init(acc_empty + 8 * s, 8); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    pdl_launch_dependents();                                // not before the columns are this block's: a dependent's block must not take them first and wait
    if (warp == 0) {
        if (lane == 0) {
            pdl_wait();
            int s = 0;
            uint32_t phase = 1;
            bool ok = true;
            for (int tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
                int w, x;
                tile_of(tile, w_tiles, x_tiles, w, x);
                for (int g = 0; g < p.groups; ++g) {
                    ok = mbar_wait(empty0 + 8 * s, phase, status, 1);
                    if (!ok) break;
                    mbar_expect_tx(full0 + 8 * s, MANY_STAGE_BYTES);
                    const uint32_t dst = base + s * MANY_STAGE_BYTES;
                    tma_load_2d(dst, &map_x, full0 + 8 * s, g * GROUP, x * BM);
                    tma_load_2d(dst + A_BYTES, &map_w, full0 + 8 * s, g * GROUP, w * BN);
                    if (++s == MANY_STAGES) { s = 0; phase ^= 1u; }
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            const uint64_t a_desc0 = operand_desc(base), b_desc0 = operand_desc(base + A_BYTES);
            int s = 0, b = 0;
            uint32_t phase = 0, acc_phase = 1;
            bool ok = true;
            for (int tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x)
                for (int g = 0; g < p.groups; ++g) {
                    ok = mbar_wait(acc_empty + 8 * b, acc_phase, status, 2) && mbar_wait(full0 + 8 * s, phase, status, 2);
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t step = (uint64_t)(s * (MANY_STAGE_BYTES >> 4));
#pragma unroll
                    for (int k = 0; k < GROUP / 32; ++k) umma_fp8(tmem_base + b * BN, a_desc0 + step + 2 * k, b_desc0 + step + 2 * k, IDESC, k > 0 ? 1u : 0u);
                    umma_commit(empty0 + 8 * s);
                    umma_commit(acc_full + 8 * b);
                    if (++s == MANY_STAGES) { s = 0; phase ^= 1u; }
                    if ((b ^= 1) == 0) acc_phase ^= 1u;
                }
        }
    } else {
        const int quarter = warp & 3, half = (warp - 2) >> 2, row = quarter * 32 + lane;
        pdl_wait();
        const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(half * 128);
        int b = 0;
        uint32_t acc_phase = 0;
        bool ok = true;
        for (int tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
            int w, x;
            tile_of(tile, w_tiles, x_tiles, w, x);
            const int m = x * BM + row, n0 = w * BN + half * 128;
            const float* x_scale = p.x_scale + min(m, p.rows - 1);
            const float* w_scale = p.w_scale + (size_t)min(n0 / GROUP, (p.n - 1) / GROUP) * p.groups;
            uint64_t acc[64];
#pragma unroll
            for (int c = 0; c < 64; ++c) acc[c] = 0ull;
            float by = x_scale[0] * w_scale[0];
            for (int g = 0; g < p.groups; ++g) {
                const float now = by;
                if (g + 1 < p.groups) by = x_scale[(size_t)(g + 1) * p.rows] * w_scale[g + 1];
                ok = __all_sync(0xffffffffu, mbar_wait(acc_full + 8 * b, acc_phase, status, 3));
                if (!ok) break;
                tc_fence_after();
                const uint32_t at = lane_addr + (uint32_t)(b * BN);
                const uint64_t by2 = pair_f32(now, now);
                uint32_t v[2][16];
                tmem_load16_start(at, v[0]);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    tmem_wait_ld();
                    if (i < 7) tmem_load16_start(at + 16 * (i + 1), v[(i + 1) & 1]);
#pragma unroll
                    for (int c = 0; c < 8; ++c) acc[8 * i + c] = fma2(pair_u32(v[i & 1][2 * c], v[i & 1][2 * c + 1]), by2, acc[8 * i + c]);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(acc_empty + 8 * b);
                if ((b ^= 1) == 0) acc_phase ^= 1u;
            }
            TO* dst = (TO*)p.out + (size_t)m * p.n + n0;
            if (!ok || m >= p.rows) {
            } else if (p.wide && n0 + 128 <= p.n) {
                constexpr int PER = 32 / sizeof(TO);       // numbers in 32 bytes
#pragma unroll
                for (int c = 0; c < 128; c += PER) {
                    uint32_t word[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if constexpr (sizeof(TO) == 2) {
                            const float2 y = unpair(acc[c / 2 + i]);
                            const __nv_bfloat162 two = __floats2bfloat162_rn(y.x, y.y);
                            word[i] = *reinterpret_cast<const uint32_t*>(&two);
                        } else {
                            const float2 y = unpair(acc[c / 2 + i / 2]);
                            word[i] = __float_as_uint((i & 1) ? y.y : y.x);
                        }
                    }
                    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst + c), "r"(word[0]), "r"(word[1]), "r"(word[2]), "r"(word[3]), "r"(word[4]),
                                 "r"(word[5]), "r"(word[6]), "r"(word[7]) : "memory");
                }
            } else {
#pragma unroll
                for (int c = 0; c < 64; ++c) {
                    const float2 y = unpair(acc[c]);
                    if (n0 + 2 * c < p.n) dst[2 * c] = from_float<TO>(y.x);
                    if (n0 + 2 * c + 1 < p.n) dst[2 * c + 1] = from_float<TO>(y.y);
                }
            }
            __syncwarp();
        }
    }
    tc_fence_before();
    __syncthreads();
    if (*(volatile int*)status != 0) {
        const unsigned long long t0 = global_timer();
        while (global_timer() - t0 < 2000000ull) __nanosleep(1000);
    }
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
}

// ----------------------------------------------------------------------------- host side
// [rows, k] bytes, box 128 x box_rows, 128-byte swizzle, zeros outside.
int byte_map(CUtensorMap* map, const void* ptr, uint64_t rows, uint64_t k, uint32_t box_rows) {
    EncodeFn encode = encode_fn();
    if (!encode) QT_FAIL(QT_ERR_LAUNCH, "gemm_fp8: the driver does not offer cuTensorMapEncodeTiled");
    const cuuint64_t dims[2] = {k, rows}, strides[1] = {k};
    const cuuint32_t box[2] = {GROUP, box_rows}, elem[2] = {1, 1};
    const CUresult rc = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS) QT_FAIL(QT_ERR_LAUNCH, "gemm_fp8: cuTensorMapEncodeTiled failed with %d for [%llu, %llu]", (int)rc, (unsigned long long)rows, (unsigned long long)k);
    return QT_OK;
}

template <int BX, typename TO>
int launch_few(const void* x8, const void* w8, GemmParams p, int k, int splits, cudaStream_t stream) {
    CUtensorMap map_w, map_x;
    int rc = byte_map(&map_w, w8, p.n, k, BM);
    if (rc) return rc;
    rc = byte_map(&map_x, x8, p.rows, k, BX);
    if (rc) return rc;
    p.groups_per_split = (p.groups + splits - 1) / splits;
    splits = (p.groups + p.groups_per_split - 1) / p.groups_per_split;
    int stages = std::min(BX <= 32 ? 4 : 5, p.groups_per_split);
    const int park = splits > 1 ? (int)((BX * Few<BX>::PARK * 4 + Few<BX>::STAGE_BYTES - 1) / Few<BX>::STAGE_BYTES) : 1;
    stages = std::max(std::max(stages, park), 2);
    const cudaError_t raised = raise_shared<gemm_fp8_few_kernel<BX, TO>>(227 * 1024);
    if (raised != cudaSuccess) QT_FAIL(QT_ERR_LAUNCH, "gemm_fp8: cannot raise shared memory: %s", cudaGetErrorString(raised));
    launch_kernel_cluster(gemm_fp8_few_kernel<BX, TO>, dim3(splits, (p.n + BM - 1) / BM, (p.rows + BX - 1) / BX), dim3(FEW_THREADS), Few<BX>::smem(stages), stream, splits, map_w,
                          map_x, p, stages);
    QT_CHECK_LAUNCH("gemm_fp8 few");
    return QT_OK;
}

template <typename TO> int launch_many(const void* x8, const void* w8, const GemmParams& p, int k, cudaStream_t stream) {
    CUtensorMap map_w, map_x;
    int rc = byte_map(&map_w, w8, p.n, k, BN);
    if (rc) return rc;
    rc = byte_map(&map_x, x8, p.rows, k, BM);
    if (rc) return rc;
    const cudaError_t raised = raise_shared<gemm_fp8_many_kernel<TO>>(227 * 1024);
    if (raised != cudaSuccess) QT_FAIL(QT_ERR_LAUNCH, "gemm_fp8: cannot raise shared memory: %s", cudaGetErrorString(raised));
    const long long tiles = (long long)((p.n + BN - 1) / BN) * ((p.rows + BM - 1) / BM);
    QT_REQUIRE(tiles <= 0x7fffffff / RASTER, "gemm_fp8: %d x %d outputs are too many", p.rows, p.n);
    launch_kernel(gemm_fp8_many_kernel<TO>, dim3((unsigned)std::min<long long>(tiles, sm_count())), dim3(MANY_THREADS),
                  (size_t)MANY_STAGES * MANY_STAGE_BYTES + 8 * (2 * MANY_STAGES + 4) + 16 + 1024, stream, map_w, map_x, p);
    QT_CHECK_LAUNCH("gemm_fp8 many");
    return QT_OK;
}

}  // namespace

// x [rows, k] -> values [rows, k] e4m3, scales [ceil(k / 128), rows].
extern "C" int qt_quantise_rows(const void* x, int dtype, void* values, float* scales, int rows, int k, void* stream) {
    QT_REQUIRE(rows >= 0 && k > 0, "quantise_rows: bad sizes %d x %d", rows, k);
    if (rows == 0) return QT_OK;
    const int groups = (k + GROUP - 1) / GROUP;
    const long long blocks = ((long long)rows * groups + 7) / 8;
    QT_REQUIRE(blocks <= 0x7fffffff, "quantise_rows: %d x %d is too large", rows, k);
    return QT_DISPATCH_DTYPE(dtype, "quantise_rows", {
        launch_kernel(quantise_rows_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, (cudaStream_t)stream, (const T*)x, (uint8_t*)values, scales, rows, k, groups);
        QT_CHECK_LAUNCH("quantise_rows");
        return QT_OK;
    });
}

// w [n, k] -> values [n, k] e4m3, scales [ceil(n / 128), ceil(k / 128)].
extern "C" int qt_quantise_weight(const void* w, int dtype, void* values, float* scales, int n, int k, void* stream) {
    QT_REQUIRE(n > 0 && k > 0 && (n + GROUP - 1) / GROUP <= 65535, "quantise_weight: bad sizes %d x %d", n, k);
    return QT_DISPATCH_DTYPE(dtype, "quantise_weight", {
        launch_kernel(quantise_weight_kernel<T>, dim3((k + GROUP - 1) / GROUP, (n + GROUP - 1) / GROUP), dim3(256), 0, (cudaStream_t)stream, (const T*)w, (uint8_t*)values,
                      scales, n, k);
        QT_CHECK_LAUNCH("quantise_weight");
        return QT_OK;
    });
}

// x8 [rows, k], x_scale [groups, rows], w8 [n, k], w_scale [ceil(n / 128), groups], out [rows, n].  `form`: -1 chooses; 0 any sizes; 16, 32, 64, 128: few rows in
// tiles of so many, with `splits` ranges of K; 256: many rows.
extern "C" int qt_gemm_fp8(const void* x8, const float* x_scale, const void* w8, const float* w_scale, void* out, int dtype, int rows, int n, int k, int form, int splits,
                           int* status, void* stream) {
    QT_REQUIRE(rows >= 0 && n > 0 && k > 0 && (rows + 63) / 64 <= 65535, "gemm_fp8: bad sizes M=%d N=%d K=%d", rows, n, k);
    QT_REQUIRE(status != nullptr, "gemm_fp8: a status word is required");
    if (rows == 0) return QT_OK;
    const int size = dtype == QT_F32 ? 4 : 2;
    GemmParams p{x_scale, w_scale, out, rows, n, (k + GROUP - 1) / GROUP, 0, (uintptr_t)out % 32 == 0 && (size_t)n * size % 32 == 0, status};
    cudaStream_t s = (cudaStream_t)stream;
    const bool aligned = k % 16 == 0 && (((uintptr_t)x8 | (uintptr_t)w8) & 15) == 0;
    if (!aligned) form = 0;
    return QT_DISPATCH_DTYPE(dtype, "gemm_fp8", {
        if (form == 16) return launch_few<16, T>(x8, w8, p, k, splits, s);
        if (form == 32) return launch_few<32, T>(x8, w8, p, k, splits, s);
        if (form == 64) return launch_few<64, T>(x8, w8, p, k, splits, s);
        if (form == 128) return launch_few<128, T>(x8, w8, p, k, splits, s);
        if (form == 256) return launch_many<T>(x8, w8, p, k, s);
        launch_kernel(gemm_fp8_any_kernel<T>, dim3((n + 63) / 64, (rows + 63) / 64), dim3(256), 0, s, (const uint8_t*)x8, x_scale, (const uint8_t*)w8, w_scale, (T*)out, rows, n,
                      k, p.groups);
        QT_CHECK_LAUNCH("gemm_fp8");
        return QT_OK;
    });
}

QT_DEFINE_LAST_ERROR(gemm_fp8)
