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
// Four neighbouring columns a lane.  WIDE: rows begin where four elements do.
template <typename T> __device__ __forceinline__ void load4(float (&v)[4], const T* row, int c0, int k, bool wide) {
    if (wide && c0 + 4 <= k) {
        if constexpr (sizeof(T) == 2) {
            const uint2 two = *reinterpret_cast<const uint2*>(row + c0);
            const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&two.x)), b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&two.y));
            v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
        } else {
            const float4 f = *reinterpret_cast<const float4*>(row + c0);
            v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = c0 + i < k ? to_float(row[c0 + i]) : 0.f;
    }
}
// A warp's 128 columns in 8 bits, four a lane, and their scale.
__device__ __forceinline__ uint32_t quantise4(const float (&v)[4], float& scale) {
    const float largest = warp_max(fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3]))));
    scale = fmaxf(__fmul_rn(largest, PER_TOP), LEAST_SCALE);
    return pack4(__fdiv_rn(v[0], scale), __fdiv_rn(v[1], scale), __fdiv_rn(v[2], scale), __fdiv_rn(v[3], scale));
}
// x / s for many x: the correctly rounded quotient by P. Markstein's method (IBM J. Res. Dev. 34, 1990): with r = 1 / s correctly rounded, a step from x r gives a
// quotient within an ulp, whose remainder is exact, and q + remainder r rounds as x / s does.  Scales whose remainders could leave float's range are divided by.
struct Divisor {
    float s, r;
    bool near;
    __device__ __forceinline__ float operator()(float x) const {
        if (!near) return __fdiv_rn(x, s);
        float q = __fmul_rn(x, r);
        q = __fmaf_rn(__fmaf_rn(q, s, -x), -r, q);          // the remainder's signs keep those of zeros
        return __fmaf_rn(__fmaf_rn(q, s, -x), -r, q);
    }
};
// N neighbours that begin at a boundary of 16 bytes.
template <int N, typename T> __device__ __forceinline__ void load_neighbours(float (&v)[N], const T* at) {
    constexpr int PIECES = N * (int)sizeof(T) / 16;
    uint4 raw[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) raw[i] = reinterpret_cast<const uint4*>(at)[i];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const uint32_t words[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (sizeof(T) == 2) {
                v[8 * i + 2 * j] = __uint_as_float(words[j] << 16);
                v[8 * i + 2 * j + 1] = __uint_as_float(words[j] & 0xffff0000u);
            } else {
                v[4 * i + j] = __uint_as_float(words[j]);
            }
        }
    }
}
// A lane's N columns from c0 on of row m (zeros and not `inside` behind the row's end), GROUP / N lanes a group: every lane of the warp calls.
template <int N> __device__ __forceinline__ void quantise_neighbours(const float (&v)[N], uint8_t* values, float* scales, int rows, int k, int m, int c0, bool inside) {
    float largest = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) largest = fmaxf(largest, fabsf(v[i]));
#pragma unroll
    for (int d = 1; d < GROUP / N; d *= 2) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, d));
    const float scale = fmaxf(__fmul_rn(largest, PER_TOP), LEAST_SCALE);
    const Divisor over{scale, __frcp_rn(scale), scale > 0x1p-60f && scale < 0x1p60f};
    if (!inside) return;
    if (c0 % GROUP == 0) scales[(size_t)(c0 / GROUP) * rows + m] = scale;
    uint32_t out[N / 4];
#pragma unroll
    for (int i = 0; i < N / 4; ++i) out[i] = pack4(over(v[4 * i]), over(v[4 * i + 1]), over(v[4 * i + 2]), over(v[4 * i + 3]));
    uint8_t* to = values + (size_t)m * k + c0;
    if constexpr (N == 16) *reinterpret_cast<uint4*>(to) = make_uint4(out[0], out[1], out[2], out[3]);
    else *reinterpret_cast<uint2*>(to) = make_uint2(out[0], out[1]);
}
// Rows in 8 bits, scales as [group, row], bound by instructions (73 % of the issue slots) where there are many: a lane 16 columns, eight lanes a group, a warp 512 columns of a row, a block eight
// rows, whose scales lie side by side.  4096 rows of 12288 in bfloat16: 33 us (4.6 TB/s), where four columns a lane, a warp a group and CUDA's division took 76; 333 of
// 8192: 3.1 (5.1); 8 of 4096: 1.8 (1.6); with eight columns a lane 41, 3.3 and 1.6.
template <typename T>
__global__ void __launch_bounds__(256) quantise_rows_wide_kernel(const T* x, uint8_t* values, float* scales, int rows, int k) {
    pdl_launch_dependents();
    pdl_wait();
    const int m = blockIdx.y * 8 + (threadIdx.x >> 5), c0 = blockIdx.x * 512 + (threadIdx.x & 31) * 16;
    if (m >= rows) return;
    float v[16] = {};
    if (c0 < k) load_neighbours(v, x + (size_t)m * k + c0);
    quantise_neighbours(v, values, scales, rows, k, m, c0, c0 < k);
}
// The same of act(gate) * up, rounded to T first as the activation by itself leaves it: of a row of 2 k numbers, gate then up (group 0) or `group` of each in turns.
// Eight columns a lane: its instructions (76 % of the issue slots) and exponentials (55 % of their pipe) bound it more than memory (4096 rows of 2 * 12288 in bfloat16 71 us, 3.6 TB/s, where the activation and the rows to
// 8 bits take 97 in two launches; 8 rows 2.6 and 3.7; with 16 columns a lane 88 and 4.7).
template <typename T>
__global__ void __launch_bounds__(256) gated_rows_kernel(const T* gate_up, uint8_t* values, float* scales, int rows, int k, int group, int act, float limit) {
    pdl_launch_dependents();
    pdl_wait();
    const int m = blockIdx.y * 8 + (threadIdx.x >> 5), c0 = blockIdx.x * 256 + (threadIdx.x & 31) * 8;
    if (m >= rows) return;
    float v[8] = {};
    if (c0 < k) {
        float up[8];
        const T* gate = gate_up + (size_t)m * 2 * k + (group ? (size_t)(c0 / group) * 2 * group + c0 % group : (size_t)c0);
        load_neighbours(v, gate);
        load_neighbours(up, gate + (group ? group : k));
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_float(from_float<T>(gated_value<sizeof(T) == 2>(v[i], up[i], act, limit)));
    }
    quantise_neighbours(v, values, scales, rows, k, m, c0, c0 < k);
}
// The same of a norm: stream += the sum of delta's planes (where there are some), and the rows are stream / rms(stream) * weight, rounded to T first as the norm by itself leaves
// them.  A block a row, eight columns a thread and chunk, which stay in registers between the sum and the write.  Bound by memory where rows are many: 4096 rows of 4096
// (a bfloat16 plane) 37 us, 5.0 TB/s, where the norm and the rows to 8 bits take 50 in two launches; 8 rows 3.2 and 4.7.
constexpr int NORM_CHUNKS = 2, NORM_MOST = NORM_CHUNKS * 1024 * 8;
template <typename T, typename TD>
__global__ void __launch_bounds__(1024) norm_rows_kernel(float* stream, const TD* delta, int planes, size_t plane_stride, const float* weight, float eps, uint8_t* values, float* scales,
                                                         int rows, int k) {
    __shared__ float scratch[32];
    pdl_launch_dependents();
    pdl_wait();
    const int m = blockIdx.x;
    float x[NORM_CHUNKS][8], sum = 0.f;
#pragma unroll
    for (int c = 0; c < NORM_CHUNKS; ++c) {
        const int c0 = (c * blockDim.x + threadIdx.x) * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[c][i] = 0.f;
        if (c0 >= k) continue;
        float* row = stream + (size_t)m * k + c0;
        load_neighbours(x[c], row);
        if (planes) {
            float d[8], more[8];
            load_neighbours(d, delta + (size_t)m * k + c0);
            for (int plane = 1; plane < planes; ++plane) {
                load_neighbours(more, delta + plane * plane_stride + (size_t)m * k + c0);
#pragma unroll
                for (int i = 0; i < 8; ++i) d[i] += more[i];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) x[c][i] += d[i];
            *reinterpret_cast<float4*>(row) = make_float4(x[c][0], x[c][1], x[c][2], x[c][3]);
            *reinterpret_cast<float4*>(row + 4) = make_float4(x[c][4], x[c][5], x[c][6], x[c][7]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = fmaf(x[c][i], x[c][i], sum);
    }
    const float factor = rsqrtf(block_sum(sum, scratch) / (float)k + eps);
#pragma unroll
    for (int c = 0; c < NORM_CHUNKS; ++c) {
        const int c0 = (c * blockDim.x + threadIdx.x) * 8;
        if (c * (int)blockDim.x * 8 >= k) break;            // the same for the block
        float w[8] = {};
        if (c0 < k) load_neighbours(w, weight + c0);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[c][i] = to_float(from_float<T>(x[c][i] * factor * w[i]));
        quantise_neighbours(x[c], values, scales, rows, k, m, c0, c0 < k);
    }
}
// The same for columns that are no multiple of 16 or rows off 16 bytes: a warp a row and 128 columns.
template <typename T>
__global__ void __launch_bounds__(256) quantise_rows_kernel(const T* x, uint8_t* values, float* scales, int rows, int k, int groups, int wide) {
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const long long unit = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (unit >= (long long)rows * groups) return;
    const int m = (int)(unit / groups), g = (int)(unit % groups), c0 = g * GROUP + lane * 4;
    float v[4], scale;
    load4(v, x + (size_t)m * k, c0, k, wide);
    const uint32_t four = quantise4(v, scale);
    if (lane == 0) scales[(size_t)g * rows + m] = scale;
    uint8_t* to = values + (size_t)m * k + c0;
    if (wide && c0 + 4 <= k) {
        *reinterpret_cast<uint32_t*>(to) = four;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (c0 + i < k) to[i] = (uint8_t)(four >> (8 * i));
    }
}

// A weight's block of 128 x 128, one scale for all of it, by a block of eight warps: a lane 16 neighbours of four rows, which stay in registers between the block's
// largest number and the write.  Bound by latency: 127 registers leave two blocks an SM, 24 % of its warps, and each waits for all of its reads before its first write (24576 x 4096 from
// bfloat16: 127 us, 2.4 TB/s; read twice and divided element by element 262).
__device__ __forceinline__ float block_scale(float largest, float* most) {
    largest = warp_max(largest);
    if ((threadIdx.x & 31) == 0) most[threadIdx.x >> 5] = largest;
    __syncthreads();
    return fmaxf(__fmul_rn(warp_max(most[threadIdx.x & 7]), PER_TOP), LEAST_SCALE);
}
template <typename T>
__global__ void __launch_bounds__(256) quantise_weight_wide_kernel(const T* w, uint8_t* values, float* scales, int n, int k) {
    __shared__ float most[8];
    pdl_launch_dependents();
    pdl_wait();
    const int row0 = blockIdx.y * GROUP + (threadIdx.x >> 3), c0 = blockIdx.x * GROUP + (threadIdx.x & 7) * 16;
    float v[4][16], largest = 0.f;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[r][i] = 0.f;
        if (row0 + 32 * r < n && c0 < k) load_neighbours(v[r], w + (size_t)(row0 + 32 * r) * k + c0);
#pragma unroll
        for (int i = 0; i < 16; ++i) largest = fmaxf(largest, fabsf(v[r][i]));
    }
    const float scale = block_scale(largest, most);
    const Divisor over{scale, __frcp_rn(scale), scale > 0x1p-60f && scale < 0x1p60f};
    if (threadIdx.x == 0) scales[(size_t)blockIdx.y * gridDim.x + blockIdx.x] = scale;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        if (row0 + 32 * r >= n || c0 >= k) continue;
        uint32_t out[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = pack4(over(v[r][4 * i]), over(v[r][4 * i + 1]), over(v[r][4 * i + 2]), over(v[r][4 * i + 3]));
        *reinterpret_cast<uint4*>(values + (size_t)(row0 + 32 * r) * k + c0) = make_uint4(out[0], out[1], out[2], out[3]);
    }
}
// The same for columns that are no multiple of 16, or addresses off 16 bytes.
template <typename T>
__global__ void __launch_bounds__(256) quantise_weight_kernel(const T* w, uint8_t* values, float* scales, int n, int k) {
    __shared__ float most[8];
    pdl_launch_dependents();
    pdl_wait();
    const int n0 = blockIdx.y * GROUP, k0 = blockIdx.x * GROUP, col = k0 + (threadIdx.x & 127);
    float largest = 0.f;
    for (int r = n0 + (threadIdx.x >> 7); r < min(n, n0 + GROUP); r += 2)
        if (col < k) largest = fmaxf(largest, fabsf(to_float(w[(size_t)r * k + col])));
    const float scale = block_scale(largest, most);
    if (threadIdx.x == 0) scales[(size_t)blockIdx.y * gridDim.x + blockIdx.x] = scale;
    for (int r = n0 + (threadIdx.x >> 7); r < min(n, n0 + GROUP); r += 2)
        if (col < k) values[(size_t)r * k + col] = (uint8_t)pack2(__fdiv_rn(to_float(w[(size_t)r * k + col]), scale), 0.f);
}

// ----------------------------------------------------------------------------- the product, any sizes
// For rows that do not begin where 16 bytes do, which no tensor map describes: 64 x 64 outputs a block, a group of K at a time through shared memory, the next one's words
// on their way meanwhile.  Eight warps of 16 x 32 outputs bring the numbers to halves (exact) for mma.sync; which element of K a place of a fragment is, is free as
// long as both operands agree, so a lane's four neighbouring bytes are its two pairs.  Bound by the way of a group's words, which a block has one of at a time (333 rows of
// 5120 x 8200: 260 us, 8 of 4096 x 4100 54, of 4096 x 4101, byte by byte, 109; on the FMA pipe 2,020 and 428).
constexpr int ANY = 64, ANY_ROW = GROUP + 16;               // bytes from a row to the next: eight rows' words are all the banks
constexpr int ANY_WORDS = ANY * GROUP / 4 / 256;            // words of an operand's group that a thread carries
// Four neighbours of a row from column `c` on; zeros behind its end.
__device__ __forceinline__ uint32_t four_of(const uint8_t* row, int c, int k, bool words) {
    if (words) return c < k ? *reinterpret_cast<const uint32_t*>(row + c) : 0u;
    uint32_t v = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (c + i < k) v |= (uint32_t)row[c + i] << (8 * i);
    return v;
}
template <typename T>
__global__ void __launch_bounds__(256) gemm_fp8_any_kernel(const uint8_t* x8, const float* x_scale, const uint8_t* w8, const float* w_scale, T* out, int rows, int n, int k, int groups,
                                                           int words) {
    __shared__ __align__(16) uint8_t xs[ANY * ANY_ROW], ws[ANY * ANY_ROW];
    pdl_launch_dependents();
    pdl_wait();
    const int m0 = blockIdx.y * ANY, n0 = blockIdx.x * ANY, warp = threadIdx.x >> 5, g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
    const int row0 = warp % 4 * 16 + g, col0 = warp / 4 * 32;                          // rows row0 and row0 + 8, columns col0 + 8 j + 2 t and the next
    uint32_t xw[ANY_WORDS], ww[ANY_WORDS];
    auto fetch = [&](int group) {
#pragma unroll
        for (int i = 0; i < ANY_WORDS; ++i) {
            const int at = threadIdx.x + 256 * i, r = at / (GROUP / 4), c = group * GROUP + at % (GROUP / 4) * 4;
            xw[i] = m0 + r < rows ? four_of(x8 + (size_t)(m0 + r) * k, c, k, words) : 0u;
            ww[i] = n0 + r < n ? four_of(w8 + (size_t)(n0 + r) * k, c, k, words) : 0u;
        }
    };
    float total[4][4] = {};
    fetch(0);
    for (int group = 0; group < groups; ++group) {
        __syncthreads();                                    // everybody has read the group before
#pragma unroll
        for (int i = 0; i < ANY_WORDS; ++i) {
            const int at = threadIdx.x + 256 * i, to = at / (GROUP / 4) * ANY_ROW + at % (GROUP / 4) * 4;
            *reinterpret_cast<uint32_t*>(xs + to) = xw[i];
            *reinterpret_cast<uint32_t*>(ws + to) = ww[i];
        }
        __syncthreads();
        if (group + 1 < groups) fetch(group + 1);
        float part[4][4] = {};
#pragma unroll
        for (int step = 0; step < GROUP / 16; ++step) {
            const uint32_t a = *reinterpret_cast<const uint32_t*>(xs + row0 * ANY_ROW + step * 16 + 4 * t), b = *reinterpret_cast<const uint32_t*>(xs + (row0 + 8) * ANY_ROW + step * 16 + 4 * t);
            const uint32_t a0 = halves(a), a1 = halves(b), a2 = halves(a >> 16), a3 = halves(b >> 16);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t w = *reinterpret_cast<const uint32_t*>(ws + (col0 + 8 * j + g) * ANY_ROW + step * 16 + 4 * t);
                asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                             : "+f"(part[j][0]), "+f"(part[j][1]), "+f"(part[j][2]), "+f"(part[j][3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(halves(w)), "r"(halves(w >> 16)));
            }
        }
        const float* scales = x_scale + (size_t)group * rows;
        const float s0 = m0 + row0 < rows ? scales[m0 + row0] : 0.f, s1 = m0 + row0 + 8 < rows ? scales[m0 + row0 + 8] : 0.f;
        const float by = w_scale[(size_t)(n0 / GROUP) * groups + group];               // a block's columns are of one scale block
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) total[j][i] = fmaf(part[j][i], (i < 2 ? s0 : s1) * by, total[j][i]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int m = m0 + row0 + 8 * (i >> 1), c = n0 + col0 + 8 * j + 2 * t + (i & 1);
            if (m < rows && c < n) out[(size_t)m * n + c] = from_float<T>(total[j][i]);
        }
}

// ----------------------------------------------------------------------------- the product on tcgen05
// Both operands are K-major tiles of 128-byte rows (one group of K), four tcgen05.mma of 32 elements a group.  The scales belong to the sums of a group: these
// go to one of two accumulators in tensor memory, and while the next group's are formed in the other, the epilogue's threads read them and add them, times both
// scales, to sums in their registers.
constexpr int BM = 128;                                     // the instruction's M
constexpr uint32_t A_BYTES = BM * GROUP;

// A whole warp goes through the same instructions, so that descriptors stay in the registers that a warp has in common, and one lane's products are carried out:
// issued by a lane that runs alone, a product takes about 100 cycles to leave and a commit 180, more than the tensor cores need for it.
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t elected;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(elected));
    return elected;
}
__device__ __forceinline__ void umma_fp8(uint32_t tmem_d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate, uint32_t one) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(tmem_d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(one) : "memory");
}
// Arrives at the barrier once the products issued so far are complete.
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
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, int* status, int code) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, status, code)); }
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
    const void* x; int x_wide;                              // FUSED: the rows as they are, and whether they begin where four elements do
    const float* x_scale; const float* w_scale; void* out;
    int rows, n, k, groups;
    int groups_per_split;
    int first_tile, end_tile;                               // many rows: the tiles of this launch
    int wide;                                               // rows of the output begin at boundaries of 32 bytes (2) or of four numbers (1)
    int* status;
};

// Few rows.  The weight's rows are the instruction's M (a tile is one row of scale blocks), BX rows of x its N; a cluster's blocks take a range of K each and add
// their sums through distributed shared memory in the order of their ranks.  Warp 0 copies, warp 1 issues, the others add up, a weight row and CW rows of x a
// thread.  Four accumulators: from the last product of a group to the slot's next one (a commit, two waits, the read) it takes about 1,000 cycles, and a group's
// products 300.  Bound by the weight's way from memory and, where it is small, by the latencies of a launch, a ring and a join (8 rows of 4096 x 12288: 13.4 us, 3.8 TB/s; of
// 51200 x 5120 49, 5.3 TB/s; one row of 1024 x 2048 4.1).  The weight asked into the L2 cache ahead of the wait for the kernels before only costs (14.2, 50.5 us).
// XT: the type of rows that the summing warps bring to 8 bits themselves, straight into shared memory, ahead of their sums (few of them, in up to FUSED_GROUPS groups a
// block: saves the launch); uint8_t: rows in 8 bits already.
constexpr int CHUNK = 16;                                   // groups whose scales are in shared memory at a time, twice
constexpr int FEW_SLOTS = 4, FUSED_GROUPS = 2 * CHUNK;
template <int BX, typename XT> struct Few {
    static constexpr bool FUSED = sizeof(XT) > 1;
    static constexpr int SUM_WARPS = BX >= 64 ? 8 : 4, CW = BX * 4 / SUM_WARPS, THREADS = 64 + 32 * SUM_WARPS;
    static constexpr uint32_t X_BYTES = BX * GROUP, STAGE_BYTES = A_BYTES + (FUSED ? 0 : X_BYTES), SCALE_BYTES = 2 * CHUNK * BX * 4;
    // ring, FUSED: the rows in 8 bits, scales, barriers, the address in tensor memory
    static size_t smem(int stages, int groups) {
        return (size_t)stages * STAGE_BYTES + (FUSED ? groups * X_BYTES : 0) + SCALE_BYTES + 8 * (2 * stages + 2 * FEW_SLOTS + (FUSED ? groups : 0)) + 16 + 1024;
    }
};

template <typename TO> __device__ __forceinline__ void store4(TO* at, const float (&y)[4], int there, bool wide) {
    if (wide && there >= 4) {
        if constexpr (sizeof(TO) == 2) {
            const __nv_bfloat162 a = __floats2bfloat162_rn(y[0], y[1]), b = __floats2bfloat162_rn(y[2], y[3]);
            *reinterpret_cast<uint2*>(at) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
        } else {
            *reinterpret_cast<float4*>(at) = make_float4(y[0], y[1], y[2], y[3]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < there) at[i] = from_float<TO>(y[i]);
    }
}

template <int BX, typename XT, typename TO>
__global__ void __launch_bounds__(Few<BX, XT>::THREADS) gemm_fp8_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                                                                            const GemmParams p, int stages) {
    using F = Few<BX, XT>;
    constexpr bool FUSED = F::FUSED;
    constexpr uint32_t STAGE_BYTES = F::STAGE_BYTES, TMEM_COLS = FEW_SLOTS * BX, IDESC = FP8_IDESC<BX>;
    constexpr int CW = F::CW, SUM_THREADS = 32 * F::SUM_WARPS;
    extern __shared__ uint8_t smem_raw[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = blockIdx.x, splits = gridDim.x, w0 = blockIdx.y * BM, x0 = blockIdx.z * BX;
    const int g_begin = split * p.groups_per_split, count = min(p.groups, g_begin + p.groups_per_split) - g_begin;      // >= 1: the host cuts so
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t* smem = smem_raw + (base - raw);
    const uint32_t rows_at = stages * STAGE_BYTES, scales_at = rows_at + (FUSED ? p.groups_per_split * F::X_BYTES : 0), bars = base + scales_at + F::SCALE_BYTES;
    const uint32_t full0 = bars, empty0 = bars + 8 * stages, acc_full = empty0 + 8 * stages, acc_empty = acc_full + 8 * FEW_SLOTS, x_full = acc_empty + 8 * FEW_SLOTS;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + (x_full + (FUSED ? 8 * p.groups_per_split : 0) - base));
    float* scales = reinterpret_cast<float*>(smem + scales_at);                             // [2][CHUNK][BX]
    int* status = p.status;
    if (threadIdx.x == 0) {
        prefetch_tensor_map(&map_w);
        if (!FUSED) prefetch_tensor_map(&map_x);
        for (int s = 0; s < stages; ++s) { mbar_init(full0 + 8 * s, 1); mbar_init(empty0 + 8 * s, 1); }
        for (int s = 0; s < FEW_SLOTS; ++s) { mbar_init(acc_full + 8 * s, 1); mbar_init(acc_empty + 8 * s, F::SUM_WARPS); }
        if (FUSED)
            for (int i = 0; i < count; ++i) mbar_init(x_full + 8 * i, p.rows);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    // The address in tensor memory, for the issuing and the summing warps.  Columns are taken once the kernels before this one are done (their blocks never wait for
    // columns that this one holds), and dependents are let in once this block has its own.
    auto columns = [&]() {
        asm volatile("bar.sync 2, %0;" ::"n"(SUM_THREADS + 32) : "memory");
        tc_fence_after();
        return *(volatile uint32_t*)tmem_slot;
    };

    if (warp == 0) {
        if (lane == 0) {
            pdl_wait();
            for (int i = 0; i < count; ++i) {
                const int s = i % stages;
                if (i >= stages && !mbar_wait(empty0 + 8 * s, (uint32_t)(i / stages - 1) & 1u, status, 1)) break;
                mbar_expect_tx(full0 + 8 * s, STAGE_BYTES);
                const uint32_t dst = base + s * STAGE_BYTES;
                tma_load_2d(dst, &map_w, full0 + 8 * s, (g_begin + i) * GROUP, w0);
                if (!FUSED) tma_load_2d(dst + A_BYTES, &map_x, full0 + 8 * s, (g_begin + i) * GROUP, x0);
            }
        }
    } else if (warp == 1) {
        pdl_wait();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        tc_fence_before();
        const uint32_t tmem_base = columns();
        pdl_launch_dependents();
        const uint64_t a_desc0 = operand_desc(base), b_desc0 = operand_desc(base + (FUSED ? rows_at : A_BYTES));
        const uint32_t one = elect_one();
        int s = 0;
        uint32_t phase = 0;
        for (int i = 0; i < count; ++i) {
            const int b = i % FEW_SLOTS;
            if (i >= FEW_SLOTS && !wait_warp(acc_empty + 8 * b, (uint32_t)(i / FEW_SLOTS - 1) & 1u, status, 2)) break;
            if (FUSED && !wait_warp(x_full + 8 * i, 0, status, 2)) break;
            if (!wait_warp(full0 + 8 * s, phase, status, 2)) break;
            tc_fence_after();
            const uint64_t a_desc = a_desc0 + (uint64_t)(s * (STAGE_BYTES >> 4)), b_desc = b_desc0 + (uint64_t)(FUSED ? i * (F::X_BYTES >> 4) : s * (STAGE_BYTES >> 4));
#pragma unroll
            for (int k = 0; k < GROUP / 32; ++k) umma_fp8(tmem_base + b * BX, a_desc + 2 * k, b_desc + 2 * k, IDESC, k > 0 ? 1u : 0u, one);
            commit_one(acc_full + 8 * b, one);
            commit_one(empty0 + 8 * s, one);
            if (++s == stages) { s = 0; phase ^= 1u; }
        }
    } else {
        const int quarter = warp & 3, part = (warp - 2) >> 2, row = quarter * 32 + lane, thread = threadIdx.x - 64;
        constexpr int PER = CHUNK * BX / SUM_THREADS;       // scales of a chunk that a thread fetches
        pdl_wait();                                         // the rows come from the kernel before; the output may still be read by one
        const uint32_t tmem_base = columns();
        const float* w_scale = p.w_scale + (size_t)blockIdx.y * p.groups + g_begin;
        float fetched[PER];
        auto fetch = [&](int i0) {
            const float* x_scale = p.x_scale + (size_t)g_begin * p.rows + x0;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int e = thread + j * SUM_THREADS, i = i0 + e / BX, c = e % BX;
                fetched[j] = i < count && x0 + c < p.rows ? x_scale[(size_t)i * p.rows + c] * w_scale[i] : 0.f;
            }
        };
        if constexpr (FUSED) {
            // units of a group and row, four at a time in flight; as the swizzle of 128 bytes has them: 16-byte pieces of a row, their number xor the row's
            const XT* x = (const XT*)p.x;
            const int units = count * p.rows;
            for (int u0 = warp - 2; u0 < units; u0 += 4 * F::SUM_WARPS) {
                float v[4][4], by[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int u = u0 + j * F::SUM_WARPS, i = u / p.rows, m = u % p.rows;
                    if (u < units) {
                        load4(v[j], x + (size_t)m * p.k, (g_begin + i) * GROUP + lane * 4, p.k, p.x_wide);
                        by[j] = w_scale[i];
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int u = u0 + j * F::SUM_WARPS, i = u / p.rows, m = u % p.rows;
                    if (u >= units) break;
                    float scale;
                    const uint32_t four = quantise4(v[j], scale);
                    *reinterpret_cast<uint32_t*>(smem + rows_at + i * F::X_BYTES + m * GROUP + (((lane >> 2) ^ (m & 7)) << 4) + ((lane & 3) << 2)) = four;
                    if (lane == 0) scales[i * BX + m] = scale * by[j];
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");       // the products read it
                    __syncwarp();
                    if (lane == 0) mbar_arrive(x_full + 8 * i);
                }
            }
        } else {
            fetch(0);
        }
        uint64_t acc[CW / 2];
#pragma unroll
        for (int c = 0; c < CW / 2; ++c) acc[c] = 0ull;
        bool ok = true;                                     // a wait that gave up ends the work, not the way through the barriers
        if (FUSED) asm volatile("bar.sync 1, %0;" ::"n"(SUM_THREADS) : "memory");           // every scale is there
        for (int i = 0; i < count; ++i) {
            const int b = i % FEW_SLOTS;
            float* chunk = scales + ((i / CHUNK) & 1) * (CHUNK * BX);
            if (!FUSED && i % CHUNK == 0) {
#pragma unroll
                for (int j = 0; j < PER; ++j) chunk[thread + j * SUM_THREADS] = fetched[j];
                if (i + CHUNK < count) fetch(i + CHUNK);
                asm volatile("bar.sync 1, %0;" ::"n"(SUM_THREADS) : "memory");
            }
            ok = ok && mbar_wait(acc_full + 8 * b, (uint32_t)(i / FEW_SLOTS) & 1u, status, 3);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) continue;
            tc_fence_after();
            const uint32_t at = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(b * BX + part * CW);
            uint32_t v[CW / 16][16];
#pragma unroll
            for (int c = 0; c < CW / 16; ++c) tmem_load16_start(at + 16 * c, v[c]);
            const float* by = chunk + (i % CHUNK) * BX + part * CW;
            tmem_wait_ld();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_empty + 8 * b);
#pragma unroll
            for (int c = 0; c < CW; c += 4) {
                const float4 f = *reinterpret_cast<const float4*>(by + c);
                acc[c / 2] = fma2(pair_u32(v[c / 16][c % 16], v[c / 16][c % 16 + 1]), pair_f32(f.x, f.y), acc[c / 2]);
                acc[c / 2 + 1] = fma2(pair_u32(v[c / 16][c % 16 + 2], v[c / 16][c % 16 + 3]), pair_f32(f.z, f.w), acc[c / 2 + 1]);
            }
        }
        if (splits == 1) {
            if (w0 + row < p.n) {
#pragma unroll
                for (int c = 0; c < CW; ++c) {
                    const float2 y = unpair(acc[c / 2]);
                    const int m = x0 + part * CW + c;
                    if (m < p.rows) ((TO*)p.out)[(size_t)m * p.n + w0 + row] = from_float<TO>((c & 1) ? y.y : y.x);
                }
            }
        } else {
            float* park = reinterpret_cast<float*>(smem);   // [BX][BM] over the ring: every product that read it is complete
            // (after a wait that gave up, copies may still land there; the result is invalid then)
#pragma unroll
            for (int c = 0; c < CW; ++c) {
                const float2 y = unpair(acc[c / 2]);
                park[(part * CW + c) * BM + row] = (c & 1) ? y.y : y.x;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (*(volatile int*)status != 0) {                      // a wait gave up: let copies in flight land before the block leaves
        const unsigned long long t0 = global_timer();
        while (global_timer() - t0 < 2000000ull) __nanosleep(1000);
    }
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(*(volatile uint32_t*)tmem_slot), "r"(TMEM_COLS) : "memory");
    if (splits > 1) {
        cluster_sync_all();
        // the block of rank r finishes columns r, r + splits, ..., four weight rows a thread: the ranks' sums one after the other
        for (int i = threadIdx.x;; i += F::THREADS) {
            const int c = (i >> 5) * splits + split, row = (i & 31) * 4;
            if (c >= BX || x0 + c >= p.rows) break;
            float v[8][4];
#pragma unroll
            for (int r = 0; r < 8; ++r)
                if (r < splits)
                    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[r][0]), "=f"(v[r][1]), "=f"(v[r][2]), "=f"(v[r][3])
                                 : "r"(map_to_cta(base + (uint32_t)(c * BM + row) * 4, r)) : "memory");
            float sum[4] = {};
#pragma unroll
            for (int r = 0; r < 8; ++r)
#pragma unroll
                for (int j = 0; j < 4; ++j) sum[j] += r < splits ? v[r][j] : 0.f;
            if (w0 + row < p.n) store4((TO*)p.out + (size_t)(x0 + c) * p.n + w0 + row, sum, p.n - w0 - row, p.wide != 0);
        }
        cluster_sync_all();                                 // nobody leaves while its sums are read
    }
}

// Many rows.  128 rows of x are the instruction's M, 256 weight rows its N; eight warps add up, a row of x and 128 weight rows (of one scale block) a thread.  One
// block an SM walks tiles.  384 threads: warp 0 copies, warp 1 issues, warps 4 to 11 add up and store, with most of the registers: 56 + 224 + 224 = 3 * 168 (without
// the exchange ten warps have 168 each, of which the sums spill some: 4096 rows of 24576 x 4096 450 us in the place of 417).  SPLIT: a cluster a tile, whose blocks take
// a range of K each and add their sums through distributed shared memory, as for few rows.
//
// Bound by the operands' way from the L2 cache: a group of a tile is 48 KB for 520 cycles of products and takes 0.57 us, 12.5 TB/s to all SMs (4096 rows of 51200 x 5120:
// 1,150 us, 1.87 PFLOP/s).  With fewer blocks it takes 0.42 us, the way round of one of the two accumulators: products, commit, eight reads of 16 columns, release.  Tiles of
// 256 x 256 by pairs of blocks (a third less to fetch) were tried only while the sums still spilled: 2,048 rows 210 us, these tiles then 220, more rows slower.  Reads of 32 columns spill.
constexpr int BN = 256, PARK_ROW = BN + 4;                  // floats from a row of parked sums to the next: 16 bytes of eight neighbouring rows are all the banks
constexpr int MANY_THREADS = 384, MANY_STAGES = 4, MANY_SLOTS = 512 / BN, MANY_CW = BN / 2;
constexpr uint32_t MANY_STAGE_BYTES = A_BYTES + BN * GROUP;
constexpr uint32_t MANY_TURN = MANY_STAGES * MANY_STAGE_BYTES + 8 * (2 * MANY_STAGES + 2 * MANY_SLOTS) + 16;         // 32 rows of 32 columns of each of the eight warps
constexpr int TURN_ROW = 33, TURN_WARP = 32 * TURN_ROW;
constexpr size_t MANY_SMEM = MANY_TURN + 8 * TURN_WARP * 4 + 1024;
static_assert(MANY_SMEM <= 227 * 1024, "shared memory of a block");
constexpr int RASTER = 8;

__device__ __forceinline__ void tile_of(int t, int w_tiles, int x_tiles, int& w, int& x) {     // groups of RASTER weight tiles, in a group rows of tiles
    const int per_group = RASTER * x_tiles, group = t / per_group, r = t % per_group, first = group * RASTER, width = min(RASTER, w_tiles - first);
    w = first + r % width;
    x = r / width;
}

template <bool SPLIT, typename TO>
__global__ void __launch_bounds__(MANY_THREADS, 1) gemm_fp8_many_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const GemmParams p) {
    constexpr int STAGES = MANY_STAGES, SLOTS = MANY_SLOTS, CW = MANY_CW;
    constexpr uint32_t IDESC = FP8_IDESC<BN>, TMEM_COLS = 512, STAGE_BYTES = MANY_STAGE_BYTES;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t* smem = smem_raw + (base - raw);
    const uint32_t bars = base + STAGES * STAGE_BYTES;
    const uint32_t full0 = bars, empty0 = bars + 8 * STAGES, acc_full = empty0 + 8 * STAGES, acc_empty = acc_full + 8 * SLOTS;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + (acc_empty + 8 * SLOTS - base));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int w_tiles = (p.n + BN - 1) / BN, x_tiles = (p.rows + BM - 1) / BM, tiles = p.end_tile;
    const int splits = SPLIT ? gridDim.x : 1, split = SPLIT ? blockIdx.x : 0, first = p.first_tile + (SPLIT ? blockIdx.y : blockIdx.x), step = SPLIT ? gridDim.y : gridDim.x;
    const int g_begin = split * p.groups_per_split, count = min(p.groups, g_begin + p.groups_per_split) - g_begin;
    int* status = p.status;
    if (threadIdx.x == 0) {
        prefetch_tensor_map(&map_w);
        prefetch_tensor_map(&map_x);
        for (int s = 0; s < STAGES; ++s) { mbar_init(full0 + 8 * s, 1); mbar_init(empty0 + 8 * s, 1); }
        for (int s = 0; s < SLOTS; ++s) { mbar_init(acc_full + 8 * s, 1); mbar_init(acc_empty + 8 * s, 8); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_wait();                                             // ahead of the columns: see the kernel for few rows
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    pdl_launch_dependents();
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 0) {
            if (lane == 0) {
                int s = 0;
                uint32_t phase = 1;
                bool ok = true;
                for (int tile = first; tile < tiles && ok; tile += step) {
                    int w, x;
                    tile_of(tile, w_tiles, x_tiles, w, x);
                    for (int g = 0; g < count; ++g) {
                        ok = wait(empty0 + 8 * s, phase, status, 1);
                        if (!ok) break;
                        mbar_expect_tx(full0 + 8 * s, STAGE_BYTES);
                        const uint32_t dst = base + s * STAGE_BYTES;
                        tma_load_2d(dst, &map_x, full0 + 8 * s, (g_begin + g) * GROUP, x * BM);
                        tma_load_2d(dst + A_BYTES, &map_w, full0 + 8 * s, (g_begin + g) * GROUP, w * BN);
                        if (++s == STAGES) { s = 0; phase ^= 1u; }
                    }
                }
            }
        } else if (warp == 1) {
            const uint64_t a_desc0 = operand_desc(base), b_desc0 = operand_desc(base + A_BYTES);
            const uint32_t one = elect_one();
            int s = 0, b = 0;
            uint32_t phase = 0, acc_phase = 1;
            bool ok = true;
            for (int tile = first; tile < tiles && ok; tile += step)
                for (int g = 0; g < count; ++g) {
                    ok = __all_sync(0xffffffffu, wait(full0 + 8 * s, phase, status, 2)) && __all_sync(0xffffffffu, wait(acc_empty + 8 * b, acc_phase, status, 2));
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t at = (uint64_t)(s * (STAGE_BYTES >> 4));
#pragma unroll
                    for (int k = 0; k < GROUP / 32; ++k) umma_fp8(tmem_base + b * BN, a_desc0 + at + 2 * k, b_desc0 + at + 2 * k, IDESC, k > 0 ? 1u : 0u, one);
                    commit_one(acc_full + 8 * b, one);
                    commit_one(empty0 + 8 * s, one);
                    if (++s == STAGES) { s = 0; phase ^= 1u; }
                    if (++b == SLOTS) { b = 0; acc_phase ^= 1u; }
                }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        const int quarter = warp & 3, part = (warp - 4) >> 2, row = quarter * 32 + lane;
        const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(part * CW);
        int b = 0;
        uint32_t acc_phase = 0;
        bool ok = true;
        for (int tile = first; tile < tiles && ok; tile += step) {
            int w, x;
            tile_of(tile, w_tiles, x_tiles, w, x);
            const int m = x * BM + row, n0 = w * BN + part * CW;
            const float* x_scale = p.x_scale + (size_t)g_begin * p.rows + min(m, p.rows - 1);
            const float* w_scale = p.w_scale + (size_t)min(n0 / GROUP, (p.n - 1) / GROUP) * p.groups + g_begin;
            uint64_t acc[CW / 2];
#pragma unroll
            for (int c = 0; c < CW / 2; ++c) acc[c] = 0ull;
            // scales four groups at a time, the next four on their way: a group is shorter than their way from the L2 cache
            float by[4], next[4];
            auto fetch = [&](int g0) {
#pragma unroll
                for (int i = 0; i < 4; ++i) next[i] = x_scale[(size_t)min(g0 + i, count - 1) * p.rows] * w_scale[min(g0 + i, count - 1)];
            };
            fetch(0);
            for (int g = 0; g < count; ++g) {
                if ((g & 3) == 0) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) by[i] = next[i];
                    if (g + 4 < count) fetch(g + 4);
                }
                const float now = (g & 2) ? (g & 1) ? by[3] : by[2] : (g & 1) ? by[1] : by[0];
                ok = __all_sync(0xffffffffu, wait(acc_full + 8 * b, acc_phase, status, 3));
                if (!ok) break;
                tc_fence_after();
                const uint32_t at = lane_addr + (uint32_t)(b * BN);
                const uint64_t by2 = pair_f32(now, now);
                uint32_t v[2][16];
                tmem_load16_start(at, v[0]);
#pragma unroll
                for (int i = 0; i < CW / 16; ++i) {
                    tmem_wait_ld();
                    if (i + 1 < CW / 16) {
                        tmem_load16_start(at + 16 * (i + 1), v[(i + 1) & 1]);
                    } else {                                // everything is read: the slot may take other sums
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(acc_empty + 8 * b);
                    }
#pragma unroll
                    for (int c = 0; c < 8; ++c) acc[8 * i + c] = fma2(pair_u32(v[i & 1][2 * c], v[i & 1][2 * c + 1]), by2, acc[8 * i + c]);
                }
                if (++b == SLOTS) { b = 0; acc_phase ^= 1u; }
            }
            if (SPLIT) {
                float* park = reinterpret_cast<float*>(smem) + row * PARK_ROW + part * CW;      // over the ring: every product that read it is complete
#pragma unroll
                for (int c = 0; c < CW / 2; c += 2) {
                    const float2 lo = unpair(acc[c]), hi = unpair(acc[c + 1]);
                    *reinterpret_cast<float4*>(park + 2 * c) = make_float4(lo.x, lo.y, hi.x, hi.y);
                }
            } else if (!ok) {
            } else if (p.wide != 2 || n0 + CW > p.n) {
                // rows that do not begin where 32 bytes do, and the last columns: through shared memory, so that a warp writes 32 neighbours of a row at a time
                // (2795 rows of 2568 x 8576: 85 us, each lane its own row 154)
                float* turn = reinterpret_cast<float*>(smem + MANY_TURN) + (warp - 4) * TURN_WARP;
                const int rows = min(32, p.rows - (m - lane));
#pragma unroll
                for (int c0 = 0; c0 < CW; c0 += 32) {
#pragma unroll
                    for (int c = 0; c < 16; ++c) {
                        const float2 y = unpair(acc[c0 / 2 + c]);
                        turn[lane * TURN_ROW + 2 * c] = y.x;
                        turn[lane * TURN_ROW + 2 * c + 1] = y.y;
                    }
                    __syncwarp();
                    const int n = n0 + c0 + lane;
                    TO* to = (TO*)p.out + (size_t)(m - lane) * p.n + n;
                    if (n < p.n)
#pragma unroll 4
                        for (int r = 0; r < rows; ++r) to[(size_t)r * p.n] = from_float<TO>(turn[r * TURN_ROW + lane]);
                    __syncwarp();
                }
            } else if (m < p.rows) {
                TO* dst = (TO*)p.out + (size_t)m * p.n + n0;
                constexpr int PER = 32 / sizeof(TO);       // numbers in 32 bytes
#pragma unroll
                for (int c = 0; c < CW; c += PER) {
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
    if (SPLIT) {
        cluster_sync_all();
        // the block of rank r finishes rows r, r + splits, ..., a warp a row, four neighbouring numbers a lane at a time
        int w, x;
        tile_of(first, w_tiles, x_tiles, w, x);
        for (int i = warp - 4; i >= 0 && i * splits + split < BM; i += 8) {
            const int r = i * splits + split, m = x * BM + r;
            if (m >= p.rows) break;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int c = half * 128 + lane * 4;
                float v[8][4];
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    if (q < splits)
                        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[q][0]), "=f"(v[q][1]), "=f"(v[q][2]), "=f"(v[q][3])
                                     : "r"(map_to_cta(base + (uint32_t)(r * PARK_ROW + c) * 4, q)) : "memory");
                float sum[4] = {};
#pragma unroll
                for (int q = 0; q < 8; ++q)
#pragma unroll
                    for (int j = 0; j < 4; ++j) sum[j] += q < splits ? v[q][j] : 0.f;
                if (w * BN + c < p.n) store4((TO*)p.out + (size_t)m * p.n + w * BN + c, sum, p.n - w * BN - c, p.wide != 0);
            }
        }
        cluster_sync_all();                                 // nobody leaves while its sums are read
    }
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

template <int BX, typename XT, typename TO>
int launch_few(const void* x8, const void* w8, GemmParams p, int splits, cudaStream_t stream) {
    using F = Few<BX, XT>;
    CUtensorMap map_w, map_x;
    int rc = byte_map(&map_w, w8, p.n, p.k, BM);
    if (rc) return rc;
    if (F::FUSED) map_x = map_w;                            // not used
    else rc = byte_map(&map_x, x8, p.rows, p.k, BX);
    if (rc) return rc;
    p.groups_per_split = (p.groups + splits - 1) / splits;
    splits = (p.groups + p.groups_per_split - 1) / p.groups_per_split;
    QT_REQUIRE(splits >= 1 && splits <= 8 && (!F::FUSED || (p.groups_per_split <= FUSED_GROUPS && p.rows <= BX)), "gemm_fp8: %d ranges of %d groups", splits, p.groups_per_split);
    int stages = std::min(4, p.groups_per_split);
    const int park = splits > 1 ? (int)((BX * BM * 4 + F::STAGE_BYTES - 1) / F::STAGE_BYTES) : 1;
    stages = std::max(std::max(stages, park), 2);
    const cudaError_t raised = raise_shared<gemm_fp8_few_kernel<BX, XT, TO>>(227 * 1024);
    if (raised != cudaSuccess) QT_FAIL(QT_ERR_LAUNCH, "gemm_fp8: cannot raise shared memory: %s", cudaGetErrorString(raised));
    launch_kernel_cluster(gemm_fp8_few_kernel<BX, XT, TO>, dim3(splits, (p.n + BM - 1) / BM, (p.rows + BX - 1) / BX), dim3(F::THREADS), F::smem(stages, p.groups_per_split), stream,
                          splits, map_w, map_x, p, stages);
    QT_CHECK_LAUNCH("gemm_fp8 few");
    return QT_OK;
}

template <typename TO> int launch_many(const void* x8, const void* w8, GemmParams p, int splits, int last, cudaStream_t stream) {
    CUtensorMap map_w, map_x;
    int rc = byte_map(&map_w, w8, p.n, p.k, BN);
    if (rc) return rc;
    rc = byte_map(&map_x, x8, p.rows, p.k, BM);
    if (rc) return rc;
    cudaError_t raised = raise_shared<gemm_fp8_many_kernel<false, TO>>(227 * 1024);
    if (raised == cudaSuccess) raised = raise_shared<gemm_fp8_many_kernel<true, TO>>(227 * 1024);
    if (raised != cudaSuccess) QT_FAIL(QT_ERR_LAUNCH, "gemm_fp8: cannot raise shared memory: %s", cudaGetErrorString(raised));
    const long long tiles = (long long)((p.n + BN - 1) / BN) * ((p.rows + BM - 1) / BM);
    QT_REQUIRE(tiles <= 0x7fffffff / RASTER, "gemm_fp8: %d x %d outputs are too many", p.rows, p.n);
    auto cut = [&p](int ranges) {                           // the ranges that are not empty
        p.groups_per_split = (p.groups + ranges - 1) / ranges;
        return (p.groups + p.groups_per_split - 1) / p.groups_per_split;
    };
    auto launch_split = [&](int ranges, long long count) {
        launch_kernel_cluster(gemm_fp8_many_kernel<true, TO>, dim3(ranges, (unsigned)count), dim3(MANY_THREADS), MANY_SMEM, stream, ranges, map_w, map_x, p);
    };
    p.first_tile = 0;
    p.end_tile = (int)tiles;
    if (splits > 1) splits = cut(splits);
    if (splits > 1) {
        QT_REQUIRE(splits <= 8 && tiles <= 65535, "gemm_fp8: %d ranges of K for %lld tiles", splits, tiles);
        launch_split(splits, tiles);
    } else {
        const int sms = sm_count(), rest = (int)(tiles % sms), ranges = tiles > sms && rest ? last : 1;
        QT_REQUIRE(last >= 1 && last <= 8, "gemm_fp8: %d ranges of K for the last round", last);
        p.groups_per_split = p.groups;
        if (ranges > 1) p.end_tile = (int)tiles - rest;
        launch_kernel(gemm_fp8_many_kernel<false, TO>, dim3((unsigned)std::min<long long>(p.end_tile, sms)), dim3(MANY_THREADS), MANY_SMEM, stream, map_w, map_x, p);
        if (ranges > 1) {
            QT_CHECK_LAUNCH("gemm_fp8 many");
            p.first_tile = p.end_tile;
            p.end_tile = (int)tiles;
            launch_split(cut(ranges), rest);
        }
    }
    QT_CHECK_LAUNCH("gemm_fp8 many");
    return QT_OK;
}

int quantise_rows(const void* x, int dtype, void* values, float* scales, int rows, int k, cudaStream_t stream) {
    const int groups = (k + GROUP - 1) / GROUP;
    const long long blocks = ((long long)rows * groups + 7) / 8;
    if (k % 16 == 0 && (((uintptr_t)x | (uintptr_t)values) & 15) == 0 && rows <= 65535 * 8) {
        return QT_DISPATCH_DTYPE(dtype, "quantise_rows", {
            launch_kernel(quantise_rows_wide_kernel<T>, dim3((k + 511) / 512, (rows + 7) / 8), dim3(256), 0, stream, (const T*)x, (uint8_t*)values, scales, rows, k);
            QT_CHECK_LAUNCH("quantise_rows");
            return QT_OK;
        });
    }
    QT_REQUIRE(blocks <= 0x7fffffff, "quantise_rows: %d x %d is too large", rows, k);
    const int wide = k % 4 == 0 && (((uintptr_t)x & 15) | ((uintptr_t)values & 3)) == 0;
    return QT_DISPATCH_DTYPE(dtype, "quantise_rows", {
        launch_kernel(quantise_rows_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, stream, (const T*)x, (uint8_t*)values, scales, rows, k, groups, wide);
        QT_CHECK_LAUNCH("quantise_rows");
        return QT_OK;
    });
}

template <typename XT, typename TO> int launch_fused(const GemmParams& p, const void* w8, int splits, cudaStream_t stream) {
    return launch_few<16, XT, TO>(nullptr, w8, p, splits, stream);
}

}  // namespace

// The arguments of qt_gemm_fp8 as one structure: rows in 8 bits (x8, x_scale), which are made from x first where it is given.
struct Fp8Call {
    const void* x; void* x8; float* x_scale; const void* w8; const float* w_scale; void* out; int* status; void* stream;
    int x_dtype, out_dtype, rows, n, k, form, splits, fused, last, unused;
};
static_assert(sizeof(Fp8Call) == 8 * 8 + 10 * 4, "8 addresses and 10 numbers of 32 bits, without gaps");

// x [rows, k] -> values [rows, k] e4m3, scales [ceil(k / 128), rows].
extern "C" int qt_quantise_rows(const void* x, int dtype, void* values, float* scales, int rows, int k, void* stream) {
    QT_REQUIRE(rows >= 0 && k > 0, "quantise_rows: bad sizes %d x %d", rows, k);
    return rows == 0 ? QT_OK : quantise_rows(x, dtype, values, scales, rows, k, (cudaStream_t)stream);
}

// gate_up [rows, 2 k] -> act(gate) * up as values [rows, k] e4m3, scales [ceil(k / 128), rows].  `group`: 0, or how many numbers of gate and of up alternate.
extern "C" int qt_gated_rows(const void* gate_up, int dtype, void* values, float* scales, int rows, int k, int group, int act, float limit, void* stream) {
    QT_REQUIRE(rows >= 0 && k > 0 && k % 16 == 0 && rows <= 65535 * 8, "gated_rows: %d x %d (columns in steps of 16)", rows, k);
    QT_REQUIRE(group >= 0 && group % 16 == 0 && (group == 0 || k % group == 0) && ((act >= 0 && act < QT_ACT_COUNT) || act == QT_ACT_CAPPED), "gated_rows: groups of %d of %d, activation %d", group, k, act);
    QT_REQUIRE((((uintptr_t)gate_up | (uintptr_t)values) & 15) == 0, "gated_rows: operands must be 16-byte aligned");
    if (rows == 0) return QT_OK;
    return QT_DISPATCH_DTYPE(dtype, "gated_rows", {
        launch_kernel(gated_rows_kernel<T>, dim3((k + 255) / 256, (rows + 7) / 8), dim3(256), 0, (cudaStream_t)stream, (const T*)gate_up, (uint8_t*)values, scales, rows, k, group, act,
                      limit);
        QT_CHECK_LAUNCH("gated_rows");
        return QT_OK;
    });
}

// stream [rows, k] += delta [planes, rows, k] (planes 0: none); stream / rms(stream) * weight, rounded to `dtype`, as values [rows, k] e4m3, scales [ceil(k / 128), rows].
extern "C" int qt_norm_rows(float* stream_rows, const void* delta, int delta_dtype, int planes, long long plane_stride, const float* weight, float eps, int dtype, void* values,
                            float* scales, int rows, int k, void* stream) {
    QT_REQUIRE(rows >= 0 && k > 0 && k % 16 == 0 && k <= NORM_MOST && planes >= 0, "norm_rows: %d x %d (columns in steps of 16 up to %d)", rows, k, NORM_MOST);
    QT_REQUIRE((((uintptr_t)stream_rows | (uintptr_t)delta | (uintptr_t)weight | (uintptr_t)values) & 15) == 0 && (planes < 2 || plane_stride % 8 == 0), "norm_rows: operands must be 16-byte aligned");
    QT_REQUIRE((dtype == QT_F32 || dtype == QT_BF16) && (delta_dtype == QT_F32 || delta_dtype == QT_BF16), "norm_rows: unknown element types %d, %d", dtype, delta_dtype);
    if (rows == 0) return QT_OK;
    // two chunks where rows are many: smaller blocks, more of them an SM (4096 rows of 4096 / 5120: 37 / 47 us, in one chunk 41 / 70)
    const int chunks = std::max((k / 8 + 1023) / 1024, rows > 4 * sm_count() && k >= 2048 ? 2 : 1), threads = ((k / 8 + chunks - 1) / chunks + 31) / 32 * 32;
    auto go = [&](auto kernel, auto* planes_at) {
        launch_kernel(kernel, dim3((unsigned)rows), dim3(threads), 0, (cudaStream_t)stream, stream_rows, planes_at, planes, (size_t)plane_stride, weight, eps, (uint8_t*)values, scales, rows, k);
    };
    if (dtype == QT_BF16 && delta_dtype == QT_BF16) go(norm_rows_kernel<__nv_bfloat16, __nv_bfloat16>, (const __nv_bfloat16*)delta);
    else if (dtype == QT_BF16) go(norm_rows_kernel<__nv_bfloat16, float>, (const float*)delta);
    else if (delta_dtype == QT_BF16) go(norm_rows_kernel<float, __nv_bfloat16>, (const __nv_bfloat16*)delta);
    else go(norm_rows_kernel<float, float>, (const float*)delta);
    QT_CHECK_LAUNCH("norm_rows");
    return QT_OK;
}

// w [n, k] -> values [n, k] e4m3, scales [ceil(n / 128), ceil(k / 128)].
extern "C" int qt_quantise_weight(const void* w, int dtype, void* values, float* scales, int n, int k, void* stream) {
    QT_REQUIRE(n > 0 && k > 0 && (n + GROUP - 1) / GROUP <= 65535, "quantise_weight: bad sizes %d x %d", n, k);
    const bool wide = k % 16 == 0 && (((uintptr_t)w | (uintptr_t)values) & 15) == 0;
    const dim3 grid((k + GROUP - 1) / GROUP, (n + GROUP - 1) / GROUP);
    return QT_DISPATCH_DTYPE(dtype, "quantise_weight", {
        if (wide) launch_kernel(quantise_weight_wide_kernel<T>, grid, dim3(256), 0, (cudaStream_t)stream, (const T*)w, (uint8_t*)values, scales, n, k);
        else launch_kernel(quantise_weight_kernel<T>, grid, dim3(256), 0, (cudaStream_t)stream, (const T*)w, (uint8_t*)values, scales, n, k);
        QT_CHECK_LAUNCH("quantise_weight");
        return QT_OK;
    });
}

// x [rows, k] or null, x8 [rows, k], x_scale [groups, rows], w8 [n, k], w_scale [ceil(n / 128), groups], out [rows, n].  `form`: 0 any sizes; 16, 32, 64: few rows in
// tiles of so many, 256: many rows, with `splits` ranges of K, or, in one range, `last` of them for the tiles of a last round that leaves most SMs idle.  `fused` (form 16, at most 16 rows and 32 groups a range): x is brought to 8 bits on the way, and x8
// and x_scale stay as they are.
extern "C" int qt_gemm_fp8(const Fp8Call* call) {
    const Fp8Call& c = *call;
    QT_REQUIRE(c.rows >= 0 && c.n > 0 && c.k > 0 && (c.rows + 63) / 64 <= 65535 && (c.n + BM - 1) / BM <= 65535, "gemm_fp8: bad sizes M=%d N=%d K=%d", c.rows, c.n, c.k);
    if (c.rows == 0) return QT_OK;
    QT_REQUIRE(c.status != nullptr && (c.x || !c.fused), "gemm_fp8: a status word is required");
    const int size = c.out_dtype == QT_F32 ? 4 : 2;
    cudaStream_t s = (cudaStream_t)c.stream;
    const GemmParams p{c.x, c.k % 4 == 0 && (uintptr_t)c.x % 16 == 0, c.x_scale, c.w_scale, c.out, c.rows, c.n, c.k, (c.k + GROUP - 1) / GROUP, 0, 0, 0,
                       (uintptr_t)c.out % 32 == 0 && (size_t)c.n * size % 32 == 0 ? 2 : (uintptr_t)c.out % 16 == 0 && c.n % 4 == 0 ? 1 : 0, c.status};
    const bool aligned = c.k % 16 == 0 && (((uintptr_t)c.x8 | (uintptr_t)c.w8) & 15) == 0;
    const int form = aligned ? c.form : 0;
    if (c.fused && form == 16) {
        if (c.x_dtype == QT_F32 && c.out_dtype == QT_F32) return launch_fused<float, float>(p, c.w8, c.splits, s);
        if (c.x_dtype == QT_F32 && c.out_dtype == QT_BF16) return launch_fused<float, __nv_bfloat16>(p, c.w8, c.splits, s);
        if (c.x_dtype == QT_BF16 && c.out_dtype == QT_F32) return launch_fused<__nv_bfloat16, float>(p, c.w8, c.splits, s);
        if (c.x_dtype == QT_BF16 && c.out_dtype == QT_BF16) return launch_fused<__nv_bfloat16, __nv_bfloat16>(p, c.w8, c.splits, s);
        QT_FAIL(QT_ERR_ARG, "gemm_fp8: unknown element types %d, %d", c.x_dtype, c.out_dtype);
    }
    if (c.x) {
        const int rc = quantise_rows(c.x, c.x_dtype, c.x8, c.x_scale, c.rows, c.k, s);
        if (rc) return rc;
    }
    return QT_DISPATCH_DTYPE(c.out_dtype, "gemm_fp8", {
        if (form == 16) return launch_few<16, uint8_t, T>(c.x8, c.w8, p, c.splits, s);
        if (form == 32) return launch_few<32, uint8_t, T>(c.x8, c.w8, p, c.splits, s);
        if (form == 64) return launch_few<64, uint8_t, T>(c.x8, c.w8, p, c.splits, s);
        if (form == 256) return launch_many<T>(c.x8, c.w8, p, c.splits, c.last, s);
        launch_kernel(gemm_fp8_any_kernel<T>, dim3((c.n + 63) / 64, (c.rows + 63) / 64), dim3(256), 0, s, (const uint8_t*)c.x8, c.x_scale, (const uint8_t*)c.w8, c.w_scale, (T*)c.out,
                      c.rows, c.n, c.k, p.groups, c.k % 4 == 0 && (((uintptr_t)c.x8 | (uintptr_t)c.w8) & 3) == 0);
        QT_CHECK_LAUNCH("gemm_fp8");
        return QT_OK;
    });
}

QT_DEFINE_LAST_ERROR(gemm_fp8)
