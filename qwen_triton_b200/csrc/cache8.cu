// The heads of a projection into a cache held in 8 bits: norm and rotation of queries and keys, and the write of keys and values into pages
// [pages, kv_heads, 64, d] of e4m3 numbers with a scale for each page and head.
//
// The scale of a page and head is 2^e, e the smallest between -40 and 40 with amax <= 448 * 2^e over the finite numbers held there.  Powers of two
// lose nothing against other scales (the numbers have exponents of their own) and let a page's earlier tokens be held under a larger scale without a
// second rounding, but for numbers that become smaller than 2^-6 of it.  A call that writes a page's first place starts the page anew; otherwise e only
// grows.  Whatever lies behind the last token written stays as it was.  Infinities are held as NaN.
#include "fp8.cuh"

using namespace qt;
using namespace qt_fp8;

namespace {

constexpr int PAGE = 64;
constexpr int THREADS = 256;

struct WriteParams {
    const void* qkv; int n_splits; size_t split_stride;
    void* q_out;
    uint8_t* k; uint8_t* v; float* k_scale; float* v_scale;
    const int* seq_start; const int* seq_past; const int* block_table; int max_blocks, n_pages;
    const float* q_weight; const float* k_weight; float eps;
    const float* cos_sin; int rotary_dim, max_pos, interleaved;
    int nq, nkv, d;
};

// A row's factor of the norm: 1 over its root mean square.
template <typename TI>
__device__ __forceinline__ float row_factor(const WriteParams& p, size_t at, int lane) {
    const TI* x = (const TI*)p.qkv + at;
    float sum = 0.f;
    for (int i = lane; i < p.d; i += 32) {
        const float v = load_sum(x, (size_t)i, p.n_splits, p.split_stride);
        sum = fmaf(v, v, sum);
    }
    return rsqrtf(warp_sum(sum) / (float)p.d + p.eps);
}

// Element i of a row, normed and rotated.
template <typename TI>
__device__ __forceinline__ float treated(const WriteParams& p, size_t at, int i, float factor, const float* weight, const float* angles) {
    const TI* x = (const TI*)p.qkv + at;
    auto element = [&](int j) {
        const float v = load_sum(x, (size_t)j, p.n_splits, p.split_stride);
        return weight ? v * factor * weight[j] : v;
    };
    const float own = element(i);
    if (angles == nullptr || i >= p.rotary_dim) return own;
    const int half = p.rotary_dim / 2;
    const int pair = p.interleaved ? i >> 1 : i % half;
    const bool first = p.interleaved ? (i & 1) == 0 : i < half;
    const float other = element(p.interleaved ? i ^ 1 : first ? i + half : i - half);
    const float c = angles[pair], s = angles[half + pair];
    return first ? own * c - other * s : own * c + other * s;
}

// grid: (2 nkv + nq heads, pages that a sequence's tokens touch, sequences); a warp a token.
template <typename TI, typename TO>
__global__ void __launch_bounds__(THREADS) qkv_write_cache8_kernel(const WriteParams p) {
    extern __shared__ float rows[];                        // [64][d] of keys or values
    __shared__ float most[THREADS / 32];
    pdl_launch_dependents();
    pdl_wait();
    const int seq = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int start = p.seq_start[seq], count = p.seq_start[seq + 1] - start, past = p.seq_past[seq];
    if (count <= 0) return;
    const int page_at = past / PAGE + blockIdx.y;
    const int low = max(past, page_at * PAGE), high = min(past + count, (page_at + 1) * PAGE);
    if (low >= high) return;
    const int head = blockIdx.x, width = (p.nq + 2 * p.nkv) * p.d;
    const bool query = head >= 2 * p.nkv, value = !query && head >= p.nkv;
    const int column = query ? (head - 2 * p.nkv) * p.d : (p.nq + head) * p.d;         // values lie behind the keys
    const float* weight = query ? p.q_weight : value ? nullptr : p.k_weight;
    if (!query && page_at >= p.max_blocks) return;
    float largest = 0.f;
    for (int pos = low + warp; pos < high; pos += THREADS / 32) {
        const int token = start + pos - past;
        const size_t at = (size_t)token * width + column;
        const float factor = weight ? row_factor<TI>(p, at, lane) : 1.f;
        const float* angles = value || p.cos_sin == nullptr ? nullptr : p.cos_sin + (size_t)min(pos, p.max_pos - 1) * p.rotary_dim;
        for (int i = lane; i < p.d; i += 32) {
            const float y = treated<TI>(p, at, i, factor, weight, angles);
            if (query) {
                ((TO*)p.q_out)[((size_t)token * p.nq + head - 2 * p.nkv) * p.d + i] = from_float<TO>(y);
            } else {
                const float held = nan_if_infinite(y);
                rows[(pos - page_at * PAGE) * p.d + i] = held;
                largest = fmaxf(largest, fabsf(held));     // of the finite ones: fmaxf passes over NaN
            }
        }
    }
    if (query) return;
    largest = warp_max(largest);
    if (lane == 0) most[warp] = largest;
    __syncthreads();
    largest = warp_max(most[lane & (THREADS / 32 - 1)]);
    const int kvh = value ? head - p.nkv : head;
    const int page = min(max(p.block_table[(size_t)seq * p.max_blocks + page_at], 0), p.n_pages - 1);
    float* scales = (value ? p.v_scale : p.k_scale) + (size_t)page * p.nkv + kvh;
    uint8_t* block = (value ? p.v : p.k) + ((size_t)page * p.nkv + kvh) * PAGE * p.d;
    const int first = low - page_at * PAGE, last = high - page_at * PAGE;
    const float was = first ? *scales : 0.f;
    const int power = first ? max(power_over(was), power_for(largest)) : power_for(largest);
    const float scale = power_of_two(power), inverse = power_of_two(-power);
    __syncthreads();                                       // everybody has read the scale
    if (threadIdx.x == 0) *scales = scale;
    if (first && scale != was) {                           // what the page holds, under the larger scale
        const float smaller = was * inverse;
        uint32_t* words = (uint32_t*)block;
        for (int i = threadIdx.x; i < first * p.d / 4; i += THREADS) {
            const float2 a = floats(words[i]), b = floats(words[i] >> 16);
            words[i] = pack4(a.x * smaller, a.y * smaller, b.x * smaller, b.y * smaller);
        }
    }
    uint32_t* words = (uint32_t*)(block + (size_t)first * p.d);
    const float* from = rows + first * p.d;
    for (int i = threadIdx.x; i < (last - first) * p.d / 4; i += THREADS) {
        const float4 y = *reinterpret_cast<const float4*>(from + 4 * i);
        words[i] = pack4(y.x * inverse, y.y * inverse, y.z * inverse, y.w * inverse);
    }
}

}  // namespace

extern "C" int qt_qkv_write_cache8(const void* qkv, int in_dtype, int n_splits, long long split_stride, void* q_out, int out_dtype, void* k, void* v, float* k_scale,
                                   float* v_scale, const int* seq_start, const int* seq_past, int n_seqs, int max_q_len, const int* block_table, int max_blocks, int n_pages,
                                   const float* q_weight, const float* k_weight, float eps, const float* cos_sin, int rotary_dim, int max_pos, int interleaved, int nq,
                                   int nkv, int d, void* stream) {
    if (n_seqs == 0 || max_q_len == 0) return QT_OK;
    QT_REQUIRE(n_seqs > 0 && n_seqs <= 65535 && max_q_len > 0 && nq > 0 && nkv > 0 && n_pages > 0 && max_blocks > 0 && n_splits >= 1, "qkv_write_cache8: bad sizes");
    QT_REQUIRE(d > 0 && d <= 256 && d % 16 == 0, "qkv_write_cache8: head_dim=%d is not a multiple of 16 up to 256", d);
    QT_REQUIRE(rotary_dim >= 0 && rotary_dim <= d && rotary_dim % 2 == 0 && (rotary_dim == 0 || (cos_sin && max_pos > 0)), "qkv_write_cache8: rotary_dim=%d of %d", rotary_dim, d);
    const int pages = (max_q_len - 1 + PAGE - 1) / PAGE + 1;
    QT_REQUIRE(pages <= 65535, "qkv_write_cache8: %d tokens of a sequence are too many", max_q_len);
    WriteParams p{qkv, n_splits, (size_t)split_stride, q_out, (uint8_t*)k, (uint8_t*)v, k_scale, v_scale, seq_start, seq_past, block_table, max_blocks, n_pages, q_weight,
                  k_weight, eps, rotary_dim ? cos_sin : nullptr, rotary_dim, max_pos, interleaved, nq, nkv, d};
    const dim3 grid(2 * nkv + nq, pages, n_seqs);
    const size_t smem = (size_t)PAGE * d * 4;
#define QT_WRITE(TI, TO)                                                                                                                                     \
    do {                                                                                                                                                     \
        const cudaError_t raised = raise_shared<qkv_write_cache8_kernel<TI, TO>>(PAGE * 256 * 4);                                                             \
        if (raised != cudaSuccess) QT_FAIL(QT_ERR_LAUNCH, "qkv_write_cache8: cannot raise shared memory: %s", cudaGetErrorString(raised));                    \
        launch_kernel(qkv_write_cache8_kernel<TI, TO>, grid, dim3(THREADS), smem, (cudaStream_t)stream, p);                                                   \
        QT_CHECK_LAUNCH("qkv_write_cache8");                                                                                                                  \
        return QT_OK;                                                                                                                                         \
    } while (0)
    if (in_dtype == QT_F32 && out_dtype == QT_F32) QT_WRITE(float, float);
    if (in_dtype == QT_F32 && out_dtype == QT_BF16) QT_WRITE(float, __nv_bfloat16);
    if (in_dtype == QT_BF16 && out_dtype == QT_BF16) QT_WRITE(__nv_bfloat16, __nv_bfloat16);
    if (in_dtype == QT_BF16 && out_dtype == QT_F32) QT_WRITE(__nv_bfloat16, float);
#undef QT_WRITE
    QT_FAIL(QT_ERR_ARG, "qkv_write_cache8: unknown element types %d, %d", in_dtype, out_dtype);
}

QT_DEFINE_LAST_ERROR(cache8)
