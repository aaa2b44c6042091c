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

constexpr int PAGE = 64, THREADS = 256, WARPS = THREADS / 32;

struct WriteParams {
    const void* qkv; int n_splits; size_t split_stride;
    int wide;                                              // eight elements of the projection begin where 16 bytes do
    void* q_out;
    uint8_t* k; uint8_t* v; float* k_scale; float* v_scale;
    const int* seq_start; const int* seq_past; const int* block_table; int n_seqs, max_blocks, n_pages;
    const float* q_weight; const float* k_weight; float eps;
    const float* cos_sin; int rotary_dim, max_pos, interleaved;
    int nq, nkv, d;
};

__device__ __forceinline__ void load4(float* v, const float* at) {
    const float4 f = *reinterpret_cast<const float4*>(at);
    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
}
__device__ __forceinline__ void store4(float* at, const float* v) { *reinterpret_cast<float4*>(at) = make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ void store4(__nv_bfloat16* at, const float* v) {
    const __nv_bfloat162 lo = __floats2bfloat162_rn(v[0], v[1]), hi = __floats2bfloat162_rn(v[2], v[3]);
    *reinterpret_cast<uint2*>(at) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
}

// The eight elements of a lane of a row, four from `e0` and four from `e1` on: of halves that turn against each other it has both, so that a rotation needs no
// exchange and half as many angles as with eight neighbours (prompts of 3,600 tokens of 32 + 8 + 8 heads of 128: 31 us, with neighbours 36).
struct Place { int e0, e1; bool there; };
template <int L> __device__ __forceinline__ Place place_of(const WriteParams& p) {
    const int lane = threadIdx.x & (L - 1), half = p.interleaved ? 0 : p.rotary_dim / 2;
    Place r;
    r.e0 = lane < half / 4 ? 4 * lane : 8 * lane;          // 2 half + 8 (lane - half / 4)
    r.e1 = r.e0 + (lane < half / 4 ? half : 4);
    r.there = lane < p.d / 8;                              // the others have none
    return r;
}
// A lane's elements of the projection, asked for ahead of their use; zeros where it has none.
template <typename TI> struct Asked {
    uint2 words[sizeof(TI)];                               // 4 elements are sizeof(TI) / 2 of them
    __device__ __forceinline__ void ask(const WriteParams& p, size_t at, const Place& place, bool there) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(TI); ++i) words[i] = make_uint2(0u, 0u);
        if (!there) return;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const TI* from = (const TI*)p.qkv + at + (h ? place.e1 : place.e0);
            if (p.wide) {
                if constexpr (sizeof(TI) == 2) {
                    words[h] = *reinterpret_cast<const uint2*>(from);
                } else {
                    const uint4 w = *reinterpret_cast<const uint4*>(from);
                    words[2 * h] = make_uint2(w.x, w.y);
                    words[2 * h + 1] = make_uint2(w.z, w.w);
                }
            } else {
                TI some[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) some[i] = from[i];
                memcpy(&words[h * sizeof(TI) / 2], some, sizeof(some));
            }
        }
    }
    __device__ __forceinline__ void give(float (&x)[8]) const {
        TI some[8];
        memcpy(some, words, sizeof(words));
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_float(some[i]);
    }
};

struct Head { bool query, value; int index; size_t column; };
__device__ __forceinline__ Head head_of(const WriteParams& p, int h) {     // keys, values, queries
    Head r;
    r.query = h >= 2 * p.nkv;
    r.value = !r.query && h >= p.nkv;
    r.index = r.query ? h - 2 * p.nkv : r.value ? h - p.nkv : h;
    r.column = (size_t)(r.query ? r.index : p.nq + h) * p.d;               // values lie behind the keys
    return r;
}
// The lane's part of a head's norm weight; false for a head that has none.
__device__ __forceinline__ bool weight_of(float (&w)[8], const WriteParams& p, const Head& head, const Place& place) {
    const float* weight = head.query ? p.q_weight : head.value ? nullptr : p.k_weight;
    if (!weight) return false;
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = 0.f;
    if (place.there) {
        load4(w, weight + place.e0);
        load4(w + 4, weight + place.e1);
    }
    return true;
}
// A row of L lanes: the sums of its planes, normed where there is a weight, rotated where there are angles.
// Every lane of the warp calls, rows of a warp may be treated differently, and the exchanges are all lanes' together; `there` says whether this lane has elements.
template <int L, typename TI>
__device__ __forceinline__ void treat_row(float (&x)[8], const Asked<TI>& asked, const WriteParams& p, size_t at, const Place& place, int position, const float (&weight)[8], bool normed,
                                          bool rotate, bool there) {
    const int half = p.rotary_dim / 2;
    const float* angles = p.cos_sin + (size_t)min(position, p.max_pos - 1) * p.rotary_dim;
    const bool turns = there && rotate && !p.interleaved && place.e0 < half;
    float c[4], s[4];
    if (turns) {                                           // on their way while the norm's sum is formed
        load4(c, angles + place.e0);
        load4(s, angles + half + place.e0);
    }
    asked.give(x);
    if (there)
        for (int plane = 1; plane < p.n_splits; ++plane) {
            Asked<TI> more;
            float y[8];
            more.ask(p, at + plane * p.split_stride, place, true);
            more.give(y);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] += y[i];
        }
    if (p.q_weight || p.k_weight) {                        // the same for all lanes, as what follows it
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = fmaf(x[i], x[i], sum);
#pragma unroll
        for (int off = L / 2; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        const float factor = rsqrtf(sum / (float)p.d + p.eps);
        if (normed) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = x[i] * factor * weight[i];
        }
    }
    if (turns) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a = x[i], b = x[i + 4];
            x[i] = a * c[i] - b * s[i];
            x[i + 4] = b * c[i] + a * s[i];
        }
    } else if (p.interleaved && there && rotate) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const int e = place.e0 + i;                    // eight neighbours
            if (e < p.rotary_dim) {
                const float c = angles[e / 2], s = angles[half + e / 2], a = x[i], b = x[i + 1];
                x[i] = a * c - b * s;
                x[i + 1] = b * c + a * s;
            }
        }
    }
}
// Infinities as NaN, and the largest finite size: fmaxf passes over NaN.
__device__ __forceinline__ float hold(float (&x)[8]) {
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        x[i] = nan_if_infinite(x[i]);
        most = fmaxf(most, fabsf(x[i]));
    }
    return most;
}
__device__ __forceinline__ void write8(uint8_t* row, const Place& place, const float (&x)[8], float by) {
    *reinterpret_cast<uint32_t*>(row + place.e0) = pack4(x[0] * by, x[1] * by, x[2] * by, x[3] * by);
    *reinterpret_cast<uint32_t*>(row + place.e1) = pack4(x[4] * by, x[5] * by, x[6] * by, x[7] * by);
}
// Eight held numbers under a larger scale.
__device__ __forceinline__ uint2 smaller8(uint2 w, float by) {
    const float2 a = floats(w.x), b = floats(w.x >> 16), c = floats(w.y), d = floats(w.y >> 16);
    return make_uint2(pack4(a.x * by, a.y * by, b.x * by, b.y * by), pack4(c.x * by, c.y * by, d.x * by, d.y * by));
}
// grid: (2 nkv + nq heads, pages that a sequence's tokens touch, sequences).  A row of L lanes a token; what is to be held stays in registers between
// the page's largest number and the write.  Bound by latency and instructions (15 an element): all rows' elements are asked for first, and four blocks an SM
// hide more of it than three (3,600 tokens of 32 + 8 + 8 heads of 128 in bfloat16: 28.5 us, 2.9 TB/s, with three blocks 30.2; asked for row by row 43).  Four blocks leave 64 registers a
// thread: heads of 65 to 128 spill 56 bytes of them at most, heads of 129 to 256, whose rows are whole warps', 1.1 to 1.2 KB, which they pay for (heads of 256: 88 us for twice the
// bytes of 33, in float32 125).
template <int L, typename TI, typename TO>
__global__ void __launch_bounds__(THREADS, 4) write_pages_kernel(const WriteParams p) {
    constexpr int ROWS = THREADS / L, ITERS = (PAGE + ROWS - 1) / ROWS;
    __shared__ float most[WARPS];
    pdl_launch_dependents();
    pdl_wait();
    const int seq = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Place place = place_of<L>(p);
    const int start = p.seq_start[seq], count = p.seq_start[seq + 1] - start, past = p.seq_past[seq];
    const int page_at = past / PAGE + blockIdx.y, low = max(past, page_at * PAGE), high = min(past + count, (page_at + 1) * PAGE);
    if (low >= high) return;
    const Head head = head_of(p, blockIdx.x);
    if (!head.query && page_at >= p.max_blocks) return;
    float weight[8];
    const bool normed = weight_of(weight, p, head, place);
    const size_t width = (size_t)(p.nq + 2 * p.nkv) * p.d;
    float x[ITERS][8], largest = 0.f;
    Asked<TI> asked[ITERS];
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
        const int pos = low + i * ROWS + threadIdx.x / L;
        asked[i].ask(p, (start + min(pos, high - 1) - past) * width + head.column, place, pos < high && place.there);
    }
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
        const int pos = low + i * ROWS + threadIdx.x / L;
        if (low + i * ROWS >= high) break;                 // the same for the block
        const bool there = pos < high && place.there;
        const int token = start + min(pos, high - 1) - past;
        treat_row<L>(x[i], asked[i], p, token * width + head.column, place, pos, weight, normed, !head.value, there);
        if (head.query) {
            TO* to = (TO*)p.q_out + ((size_t)token * p.nq + head.index) * p.d;
            if (there) { store4(to + place.e0, x[i]); store4(to + place.e1, x[i] + 4); }
        } else {
            largest = fmaxf(largest, hold(x[i]));          // lanes without elements hold zeros
        }
    }
    if (head.query) return;
    largest = warp_max(largest);
    if (lane == 0) most[warp] = largest;
    __syncthreads();
    largest = warp_max(most[lane & (WARPS - 1)]);
    const int page = min(max(p.block_table[(size_t)seq * p.max_blocks + page_at], 0), p.n_pages - 1);
    float* scales = (head.value ? p.v_scale : p.k_scale) + (size_t)page * p.nkv + head.index;
    uint8_t* block = (head.value ? p.v : p.k) + ((size_t)page * p.nkv + head.index) * PAGE * p.d;
    const int first = low - page_at * PAGE;
    const float was = first ? *scales : 0.f;
    const int power = first ? max(power_over(was), power_for(largest)) : power_for(largest);
    const float scale = power_of_two(power), inverse = power_of_two(-power);
    __syncthreads();                                       // everybody has read the scale
    if (threadIdx.x == 0) *scales = scale;
    if (first && scale != was) {                           // what the page holds, under the larger scale
        uint2* words = reinterpret_cast<uint2*>(block);
        for (int i = threadIdx.x; i < first * p.d / 8; i += THREADS) words[i] = smaller8(words[i], was * inverse);
    }
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
        const int pos = low + i * ROWS + threadIdx.x / L;
        if (pos < high && place.there) write8(block + (size_t)(pos - page_at * PAGE) * p.d, place, x[i], inverse);
    }
}

// One token a sequence at most: a row of L lanes a (sequence, head).  Bound by one launch's latency where no scale grows (64 sequences of 32 + 8 + 8 heads of 128: 3.1 us).  Where one does,
// its lanes bring the page's earlier rows under it one after the other, 0.6 us a row, and the launch takes as long as its longest page: 18 us more with 32 earlier rows, 37 with 63,
// for one sequence as for 64.
template <int L, typename TI, typename TO>
__global__ void __launch_bounds__(THREADS) write_tokens_kernel(const WriteParams p) {
    pdl_launch_dependents();
    pdl_wait();
    const int heads = p.nq + 2 * p.nkv, e = (threadIdx.x & (L - 1)) * 8;
    const Place place = place_of<L>(p);
    const long long row = (long long)blockIdx.x * (THREADS / L) + threadIdx.x / L;
    const int seq = (int)min(row / heads, (long long)p.n_seqs - 1);
    const Head head = head_of(p, (int)(row % heads));
    const int token = p.seq_start[seq], pos = p.seq_past[seq], page_at = pos / PAGE;
    const bool live = row < (long long)p.n_seqs * heads && p.seq_start[seq + 1] > token && (head.query || page_at < p.max_blocks), there = live && e < p.d;
    float x[8], weight[8];
    const bool normed = weight_of(weight, p, head, place);
    Asked<TI> asked;
    asked.ask(p, (size_t)token * heads * p.d + head.column, place, there);
    treat_row<L>(x, asked, p, (size_t)token * heads * p.d + head.column, place, pos, weight, normed, !head.value, there);
    if (head.query && there) {
        TO* to = (TO*)p.q_out + ((size_t)token * p.nq + head.index) * p.d;
        store4(to + place.e0, x);
        store4(to + place.e1, x + 4);
    }
    float largest = head.query ? 0.f : hold(x);
#pragma unroll
    for (int off = L / 2; off > 0; off >>= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, off));
    const int page = live && !head.query ? min(max(p.block_table[(size_t)seq * p.max_blocks + page_at], 0), p.n_pages - 1) : 0;
    float* scales = (head.value ? p.v_scale : p.k_scale) + (size_t)page * p.nkv + head.index;
    uint8_t* block = (head.value ? p.v : p.k) + ((size_t)page * p.nkv + head.index) * PAGE * p.d;
    const int first = pos % PAGE;
    const bool writes = live && !head.query;
    const float was = writes && first ? *scales : 0.f;
    __syncwarp();                                          // every lane of the row has read the scale
    if (!writes || e >= p.d) return;
    const int power = first ? max(power_over(was), power_for(largest)) : power_for(largest);
    const float scale = power_of_two(power), inverse = power_of_two(-power);
    if (e == 0) *scales = scale;
    if (first && scale != was)                             // what the page holds, under the larger scale
        for (int i = 0; i < first; ++i) {
            uint2* words = reinterpret_cast<uint2*>(block + (size_t)i * p.d + e);
            *words = smaller8(*words, was * inverse);
        }
    write8(block + (size_t)first * p.d, place, x, inverse);
}

template <int L, typename TI, typename TO> int launch(const WriteParams& p, int max_q_len, cudaStream_t stream) {
    const int heads = p.nq + 2 * p.nkv;
    if (max_q_len == 1) {
        const long long blocks = ((long long)p.n_seqs * heads + THREADS / L - 1) / (THREADS / L);
        QT_REQUIRE(blocks <= 0x7fffffff, "qkv_write_cache8: %d sequences of %d heads", p.n_seqs, heads);
        launch_kernel(write_tokens_kernel<L, TI, TO>, dim3((unsigned)blocks), dim3(THREADS), 0, stream, p);
    } else {
        const int pages = (max_q_len - 1 + PAGE - 1) / PAGE + 1;
        QT_REQUIRE(pages <= 65535 && p.n_seqs <= 65535, "qkv_write_cache8: %d sequences of up to %d tokens", p.n_seqs, max_q_len);
        launch_kernel(write_pages_kernel<L, TI, TO>, dim3(heads, pages, p.n_seqs), dim3(THREADS), 0, stream, p);
    }
    QT_CHECK_LAUNCH("qkv_write_cache8");
    return QT_OK;
}
template <typename TI, typename TO> int launch_size(const WriteParams& p, int max_q_len, cudaStream_t stream) {
    if (p.d <= 32) return launch<4, TI, TO>(p, max_q_len, stream);
    if (p.d <= 64) return launch<8, TI, TO>(p, max_q_len, stream);
    if (p.d <= 128) return launch<16, TI, TO>(p, max_q_len, stream);
    return launch<32, TI, TO>(p, max_q_len, stream);
}

}  // namespace

// The arguments of the call below as one structure.
struct WriteCall {
    const void* qkv;
    long long split_stride;
    void *q_out, *k, *v;
    float *k_scale, *v_scale;
    const int *seq_start, *seq_past, *block_table;
    const float *q_weight, *k_weight, *cos_sin;
    void* stream;
    double eps;
    int in_dtype, out_dtype, n_splits, n_seqs, max_q_len, max_blocks, n_pages, rotary_dim, max_pos, interleaved, nq, nkv, d, unused;
};
static_assert(sizeof(WriteCall) == 15 * 8 + 14 * 4, "15 numbers of 64 bits and 14 of 32, without gaps");

extern "C" int qt_qkv_write_cache8(const WriteCall* call) {
    const WriteCall& c = *call;
    const int n_seqs = c.n_seqs, max_q_len = c.max_q_len, nq = c.nq, nkv = c.nkv, d = c.d, rotary_dim = c.rotary_dim;
    if (n_seqs == 0 || max_q_len == 0) return QT_OK;
    QT_REQUIRE(n_seqs > 0 && max_q_len > 0 && nq > 0 && nkv > 0 && c.n_pages > 0 && c.max_blocks > 0 && c.n_splits >= 1, "qkv_write_cache8: bad sizes");
    QT_REQUIRE(d > 0 && d <= 256 && d % 16 == 0, "qkv_write_cache8: head_dim=%d is not a multiple of 16 up to 256", d);
    QT_REQUIRE(rotary_dim >= 0 && rotary_dim <= d && rotary_dim % (c.interleaved ? 2 : 16) == 0 && (rotary_dim == 0 || (c.cos_sin && c.max_pos > 0)),
               "qkv_write_cache8: rotary_dim=%d of %d (of pairs that are not neighbours a multiple of 16)", rotary_dim, d);
    QT_REQUIRE((((uintptr_t)c.q_out | (uintptr_t)c.k | (uintptr_t)c.v | (uintptr_t)c.q_weight | (uintptr_t)c.k_weight | (uintptr_t)c.cos_sin) & 15) == 0,
               "qkv_write_cache8: operands must be 16-byte aligned");
    const int size = c.in_dtype == QT_F32 ? 4 : 2;
    const WriteParams p{c.qkv, c.n_splits, (size_t)c.split_stride, (uintptr_t)c.qkv % 16 == 0 && c.split_stride * size % 16 == 0, c.q_out, (uint8_t*)c.k, (uint8_t*)c.v, c.k_scale,
                        c.v_scale, c.seq_start, c.seq_past, c.block_table, n_seqs, c.max_blocks, c.n_pages, c.q_weight, c.k_weight, (float)c.eps, rotary_dim ? c.cos_sin : nullptr,
                        rotary_dim, c.max_pos, c.interleaved, nq, nkv, d};
    cudaStream_t s = (cudaStream_t)c.stream;
    if (c.in_dtype == QT_F32 && c.out_dtype == QT_F32) return launch_size<float, float>(p, max_q_len, s);
    if (c.in_dtype == QT_F32 && c.out_dtype == QT_BF16) return launch_size<float, __nv_bfloat16>(p, max_q_len, s);
    if (c.in_dtype == QT_BF16 && c.out_dtype == QT_BF16) return launch_size<__nv_bfloat16, __nv_bfloat16>(p, max_q_len, s);
    if (c.in_dtype == QT_BF16 && c.out_dtype == QT_F32) return launch_size<__nv_bfloat16, float>(p, max_q_len, s);
    QT_FAIL(QT_ERR_ARG, "qkv_write_cache8: unknown element types %d, %d", c.in_dtype, c.out_dtype);
}

QT_DEFINE_LAST_ERROR(cache8)
