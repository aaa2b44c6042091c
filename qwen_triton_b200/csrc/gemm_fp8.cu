// y = x W^T for a weight of 8-bit numbers with a scale for each block of 128 x 128, and what makes rows and weights such numbers.
//
//   s_x[g, m] = max(amax_{k in g} |x[m, k]| / 448, 2^-100),  x8[m, k] = e4m3(x[m, k] / s_x[g, m])        g: 128 columns
//   y[m, n]   = sum_g s_x[g, m] s_w[n / 128, g] sum_{k in g} x8[m, k] w8[n, k]
//
// Sums are held in 32 bits; y is rounded once.
#include "fp8.cuh"

using namespace qt;
using namespace qt_fp8;

namespace {

constexpr float LEAST_SCALE = 0x1p-100f;

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
    const float scale = fmaxf(__fdiv_rn(largest, TOP), LEAST_SCALE);
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
    const float scale = fmaxf(__fdiv_rn(largest, TOP), LEAST_SCALE);
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

// x8 [rows, k], x_scale [groups, rows], w8 [n, k], w_scale [ceil(n / 128), groups], out [rows, n].
extern "C" int qt_gemm_fp8(const void* x8, const float* x_scale, const void* w8, const float* w_scale, void* out, int dtype, int rows, int n, int k, int* status,
                           void* stream) {
    QT_REQUIRE(rows >= 0 && n > 0 && k > 0 && (rows + 63) / 64 <= 65535, "gemm_fp8: bad sizes M=%d N=%d K=%d", rows, n, k);
    QT_REQUIRE(status != nullptr, "gemm_fp8: a status word is required");
    if (rows == 0) return QT_OK;
    return QT_DISPATCH_DTYPE(dtype, "gemm_fp8", {
        launch_kernel(gemm_fp8_any_kernel<T>, dim3((n + 63) / 64, (rows + 63) / 64), dim3(256), 0, (cudaStream_t)stream, (const uint8_t*)x8, x_scale, (const uint8_t*)w8,
                      w_scale, (T*)out, rows, n, k, (k + GROUP - 1) / GROUP);
        QT_CHECK_LAUNCH("gemm_fp8");
        return QT_OK;
    });
}

QT_DEFINE_LAST_ERROR(gemm_fp8)
