// Attention over a cache held in 8 bits: pages [pages, kv_heads, 64, d] of e4m3 numbers with a scale for each page and head (cache8.cu writes them).
//
//   out_i = sum_j softmax_j(scale q_i . k_j) v_j,     k_j = s_k[page of j] k8_j,     v_j = s_v[page of j] v8_j
//
// A block takes eight rows (query token, head of a kv head's group) and a range of pages; each of its warps walks pages of its own, 32 keys at a time, straight
// from memory into the registers of mma.sync: which keys and elements a lane's share of a fragment is, is free as long as both operands agree, so a lane
// loads 16 neighbouring bytes.  S^T = K q^T and O^T += V^T P^T have keys and values as the operand with 16 rows and the eight query rows as the other.
//
// Every e4m3 number is a half.  Queries are brought to halves with a power of two for each row (its largest element lies in [2^14, 2^15), so no digit
// of it is lost but below 2^-38 of that); FLOAT queries are two halves, and so is P then.  A weight is p_j s_v[j] relative to the largest such: the running
// maximum is that of the score plus log2 s_v, so that halves hold the weights whatever scales the pages have; the sum of the p_j takes the scale back out.
#include "fp8.cuh"

#include <math.h>

using namespace qt;
using namespace qt_fp8;

namespace {

constexpr int PAGE = 64;
constexpr int WARPS = 4;
constexpr int ROWS = 8;                                    // query rows of a block
constexpr float LOG2E = 1.4426950408889634f;
constexpr float RESCALE_STEP = 8.f;                        // a row's maximum moves when the true one is more than 2^8 above it

struct Params {
    const void* q; void* out;
    const uint8_t* k; const uint8_t* v; const float* k_scale; const float* v_scale;
    const int* block_table; int max_blocks, n_pages;
    const int* seq_start; const int* seq_past;             // prompts
    const int* seq_len;                                    // one query a sequence
    int nq, nkv, d;
    float scale;
    int ranges, range_pages;                               // a block walks range_pages pages of its sequence
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
template <int D, typename T>
__global__ void __launch_bounds__(32 * WARPS) attention_cache8_kernel(const Params p) {
    constexpr bool FLOAT = sizeof(T) == 4;
    constexpr int CHUNKS = D / 64, STEPS = D / 16;         // 64 elements of a key among four lanes; 16 an instruction
    constexpr int SUBS = D > 128 ? 1 : 2;                  // 16 keys each, at a time
    constexpr int KEYS = 16 * SUBS, PER_PAGE = PAGE / KEYS;
    constexpr int VBYTES = D / 8;                          // of a value row, a lane's neighbouring elements
    constexpr int VPIECE = VBYTES < 16 ? VBYTES : 16, VPIECES = VBYTES / VPIECE;
    extern __shared__ float shared[];                      // [WARPS][ROWS][D], then [WARPS][ROWS][2]
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int seq = blockIdx.z, kvh = blockIdx.y % p.nkv, group = p.nq / p.nkv;
    const int tile = p.seq_start ? blockIdx.x : blockIdx.y / p.nkv, range = p.seq_start ? 0 : blockIdx.x;
    pdl_wait();
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
    if (row0 >= rows) return;
    const int last_row = min(row0 + ROWS, rows) - 1;
    const int end = min(past + last_row / group + 1, capacity);          // keys that any row sees
    const int page_begin = range * p.range_pages, pages = (end + PAGE - 1) / PAGE;
    const int page_end = range == p.ranges - 1 ? pages : min(pages, page_begin + p.range_pages);        // the last range takes what is left
    if (page_begin >= page_end && range > 0) return;       // the join knows from the length

    // queries: row g of the block, elements 64 c + 16 t + 4 j .. + 3 for instruction 4 c + j
    uint32_t qh[STEPS][2], ql[FLOAT ? STEPS : 1][2];
    float factor;
    {
        const int row = row0 + g;
        const bool there = row <= last_row;
        const T* q = (const T*)p.q + ((size_t)(token0 + row / group) * p.nq + kvh * group + row % group) * p.d;
        float x[STEPS][4], most = 0.f;
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at = (s >> 2) * 64 + 16 * t + 4 * (s & 3);
                x[s][i] = there && at < p.d ? to_float(q[at + i]) : 0.f;
                most = fmaxf(most, fabsf(x[s][i]));
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

    const int* table = p.block_table + (size_t)seq * p.max_blocks;
    auto page_number = [&](int at) { return at < page_end ? min(max(table[at], 0), p.n_pages - 1) : 0; };
    float acc[STEPS][4] = {};
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    uint32_t kw[SUBS][2][STEPS], vw[SUBS][4][VBYTES / 4];
    auto load_keys = [&](int page, int key) {              // 16 u + g and + 8, from place `key` of the page
        const uint8_t* at = p.k + (((size_t)page * p.nkv + kvh) * PAGE + key) * p.d;
#pragma unroll
        for (int u = 0; u < SUBS; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int c = 0; c < CHUNKS; ++c) {
                    const int byte = 64 * c + 16 * t;
                    if (byte < p.d) load_words<4>(&kw[u][h][4 * c], at + (size_t)(16 * u + 8 * h + g) * p.d + byte);
                    else
#pragma unroll
                        for (int j = 0; j < 4; ++j) kw[u][h][4 * c + j] = 0;
                }
    };
    auto load_values = [&](int page, int key, int there) {  // keys 16 u + 2 t, + 1, + 8, + 9; those behind the last are zero
        const uint8_t* at = p.v + (((size_t)page * p.nkv + kvh) * PAGE + key) * p.d;
#pragma unroll
        for (int u = 0; u < SUBS; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 16 * u + 2 * t + (i & 1) + 8 * (i >> 1);
#pragma unroll
                for (int c = 0; c < VPIECES; ++c) {
                    const int byte = g * VBYTES + c * VPIECE;
                    uint32_t* w = &vw[u][i][c * VPIECE / 4];
                    if (byte < p.d && r < there) load_words<VPIECE / 4>(w, at + (size_t)r * p.d + byte);
                    else
#pragma unroll
                        for (int j = 0; j < VPIECE / 4; ++j) w[j] = 0;
                }
            }
    };

    int page_at = page_begin + warp;
    int page = page_number(page_at), next_page = page_number(page_at + WARPS);
    if (page_at < page_end) load_keys(page, 0);
    for (; page_at < page_end; page_at += WARPS) {
        const float ks = p.k_scale[(size_t)page * p.nkv + kvh], vs = p.v_scale[(size_t)page * p.nkv + kvh];
        const int after_next = page_number(page_at + 2 * WARPS);
        const float f0 = factor0 * ks, f1 = factor1 * ks, lift = log2f(vs), out_of = 1.f / vs;
#pragma unroll
        for (int part = 0; part < PER_PAGE; ++part) {
            const int key0 = page_at * PAGE + part * KEYS;
            load_values(page, part * KEYS, end - key0);
            float s[SUBS][4];
#pragma unroll
            for (int u = 0; u < SUBS; ++u) {
                float c[4] = {};
#pragma unroll
                for (int i = 0; i < STEPS; ++i) {
                    const uint32_t a = kw[u][0][i], b = kw[u][1][i];
                    const uint32_t a0 = halves(a), a1 = halves(b), a2 = halves(a >> 16), a3 = halves(b >> 16);
                    mma(c, a0, a1, a2, a3, qh[i][0], qh[i][1]);
                    if (FLOAT) mma(c, a0, a1, a2, a3, ql[FLOAT ? i : 0][0], ql[FLOAT ? i : 0][1]);
                }
                s[u][0] = fmaf(c[0], f0, lift); s[u][1] = fmaf(c[1], f1, lift);
                s[u][2] = fmaf(c[2], f0, lift); s[u][3] = fmaf(c[3], f1, lift);
            }
            if (part + 1 < PER_PAGE) load_keys(page, (part + 1) * KEYS);
            else if (page_at + WARPS < page_end) load_keys(next_page, 0);
            if (key0 + KEYS > least || last_row < row0 + ROWS - 1) {
#pragma unroll
                for (int u = 0; u < SUBS; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (key0 + 16 * u + g + 8 * (i >> 1) >= ((i & 1) ? limit1 : limit0)) s[u][i] = -INFINITY;
            }
            float top0 = -INFINITY, top1 = -INFINITY;
#pragma unroll
            for (int u = 0; u < SUBS; ++u) {
                top0 = fmaxf(top0, fmaxf(s[u][0], s[u][2]));
                top1 = fmaxf(top1, fmaxf(s[u][1], s[u][3]));
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
                for (int i = 0; i < STEPS; ++i) { acc[i][0] *= a0; acc[i][1] *= a1; acc[i][2] *= a0; acc[i][3] *= a1; }
                m0 = n0; m1 = n1;
            }
            const float u0 = m0 == -INFINITY ? 0.f : m0, u1 = m1 == -INFINITY ? 0.f : m1;
#pragma unroll
            for (int u = 0; u < SUBS; ++u) {
                const float w0 = fast_exp2(s[u][0] - u0), w1 = fast_exp2(s[u][1] - u1), w2 = fast_exp2(s[u][2] - u0), w3 = fast_exp2(s[u][3] - u1);
                l0 = fmaf(w0 + w2, out_of, l0);
                l1 = fmaf(w1 + w3, out_of, l1);
                const uint32_t h0 = pack_half(w0, w1), h1 = pack_half(w2, w3);
                const uint32_t b0 = transposed(h0), b1 = transposed(h1);
                uint32_t r0 = 0, r1 = 0;
                if (FLOAT) {
                    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&h0)), y = __half22float2(*reinterpret_cast<const __half2*>(&h1));
                    r0 = transposed(pack_half(w0 - x.x, w1 - x.y));
                    r1 = transposed(pack_half(w2 - y.x, w3 - y.y));
                }
#pragma unroll
                for (int w = 0; w < VBYTES / 4; ++w) {
                    // bytes of neighbouring keys side by side: an element's two keys are one half2
                    const uint32_t a01 = __byte_perm(vw[u][0][w], vw[u][1][w], 0x5140), a23 = __byte_perm(vw[u][0][w], vw[u][1][w], 0x7362);
                    const uint32_t b01 = __byte_perm(vw[u][2][w], vw[u][3][w], 0x5140), b23 = __byte_perm(vw[u][2][w], vw[u][3][w], 0x7362);
                    const uint32_t x0 = halves(a01), x1 = halves(a01 >> 16), x2 = halves(b01), x3 = halves(b01 >> 16);
                    const uint32_t y0 = halves(a23), y1 = halves(a23 >> 16), y2 = halves(b23), y3 = halves(b23 >> 16);
                    mma(acc[2 * w], x0, x1, x2, x3, b0, b1);
                    mma(acc[2 * w + 1], y0, y1, y2, y3, b0, b1);
                    if (FLOAT) {
                        mma(acc[2 * w], x0, x1, x2, x3, r0, r1);
                        mma(acc[2 * w + 1], y0, y1, y2, y3, r0, r1);
                    }
                }
            }
        }
        page = next_page;
        next_page = after_next;
    }
    // the warps' results, then the block's
#pragma unroll
    for (int off = 4; off < 32; off *= 2) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, off);
        l1 += __shfl_xor_sync(0xffffffffu, l1, off);
    }
    float* sums = shared + WARPS * ROWS * D;
    if (g == 0) {
        sums[(warp * ROWS + 2 * t) * 2] = m0; sums[(warp * ROWS + 2 * t) * 2 + 1] = l0;
        sums[(warp * ROWS + 2 * t + 1) * 2] = m1; sums[(warp * ROWS + 2 * t + 1) * 2 + 1] = l1;
    }
    float* own = shared + warp * ROWS * D + g * VBYTES;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {                      // elements 2 i and 2 i + 1 of the lane's
        *reinterpret_cast<float2*>(own + (2 * t) * D + 2 * i) = make_float2(acc[i][0], acc[i][2]);
        *reinterpret_cast<float2*>(own + (2 * t + 1) * D + 2 * i) = make_float2(acc[i][1], acc[i][3]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < ROWS * p.d; i += 32 * WARPS) {
        const int r = i / p.d, c = i % p.d, row = row0 + r;
        if (row > last_row) break;
        float m = -INFINITY, l = 0.f, a = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) m = fmaxf(m, sums[(w * ROWS + r) * 2]);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float mw = sums[(w * ROWS + r) * 2];
            const float by = mw == -INFINITY ? 0.f : fast_exp2(mw - m);
            // a warp without keys has nothing; one whose sums are NaN hands that on
            l = fmaf(sums[(w * ROWS + r) * 2 + 1], mw == -INFINITY ? 1.f : by, l);
            a = fmaf(shared[(w * ROWS + r) * D + c], mw == -INFINITY ? 1.f : by, a);
        }
        const int head = kvh * group + row % group;
        if (p.ranges == 1) {
            ((T*)p.out)[((size_t)(token0 + row / group) * p.nq + head) * p.d + c] = from_float<T>(l == 0.f ? 0.f : a / l);
        } else {
            const size_t part = ((size_t)seq * p.nq + head) * p.ranges + range;
            p.part_acc[part * p.d + c] = a;
            if (c == 0) { p.part_ml[part * 2] = m; p.part_ml[part * 2 + 1] = l; }
        }
    }
}

// The ranges of a (sequence, head): sum of l and acc, each at its distance from the largest maximum.
template <typename T>
__global__ void __launch_bounds__(128) join_cache8_kernel(const Params p) {
    pdl_launch_dependents();
    pdl_wait();
    const int head = blockIdx.x, seq = blockIdx.y;
    const int pages = (min(p.seq_len[seq], p.max_blocks * PAGE) + PAGE - 1) / PAGE;
    const int used = min(max(1, (pages + p.range_pages - 1) / p.range_pages), p.ranges);
    const size_t first = ((size_t)seq * p.nq + head) * p.ranges;
    const float* ml = p.part_ml + first * 2;
    float m = -INFINITY, l = 0.f;
    for (int r = 0; r < used; ++r) m = fmaxf(m, ml[2 * r]);
    for (int c = threadIdx.x; c < p.d; c += 128) {
        float a = 0.f;
        l = 0.f;
        for (int r = 0; r < used; ++r) {
            const float by = ml[2 * r] == -INFINITY ? 1.f : fast_exp2(ml[2 * r] - m);
            l = fmaf(ml[2 * r + 1], by, l);
            a = fmaf(p.part_acc[(first + r) * p.d + c], by, a);
        }
        ((T*)p.out)[((size_t)seq * p.nq + head) * p.d + c] = from_float<T>(l == 0.f ? 0.f : a / l);
    }
}

template <int D, typename T> int launch(const Params& p, dim3 grid, cudaStream_t stream) {
    constexpr size_t smem = (size_t)(WARPS * ROWS * D + WARPS * ROWS * 2) * 4;
    launch_kernel(attention_cache8_kernel<D, T>, grid, dim3(32 * WARPS), smem, stream, p);
    QT_CHECK_LAUNCH("attention_cache8");
    if (p.ranges > 1) {
        launch_kernel(join_cache8_kernel<T>, dim3(p.nq, grid.z), dim3(128), 0, stream, p);
        QT_CHECK_LAUNCH("attention_cache8 join");
    }
    return QT_OK;
}
template <typename T> int launch_size(const Params& p, dim3 grid, cudaStream_t stream) {
    if (p.d <= 64) return launch<64, T>(p, grid, stream);
    if (p.d <= 128) return launch<128, T>(p, grid, stream);
    return launch<256, T>(p, grid, stream);
}

int check(const char* name, int dtype, int nq, int nkv, int d, int max_blocks, int n_pages, const void* q, const void* k, const void* v, const void* out) {
    QT_REQUIRE(dtype == QT_F32 || dtype == QT_BF16, "%s: unknown element type %d", name, dtype);
    QT_REQUIRE(nq > 0 && nkv > 0 && nq % nkv == 0 && max_blocks > 0 && max_blocks <= 0x7fffffff / PAGE && n_pages > 0, "%s: bad sizes nq=%d nkv=%d", name, nq, nkv);
    QT_REQUIRE(d > 0 && d <= 256 && d % 16 == 0, "%s: head_dim=%d is not a multiple of 16 up to 256", name, d);
    QT_REQUIRE((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & 15) == 0, "%s: operands must be 16-byte aligned", name);
    return QT_OK;
}

}  // namespace

// One query a sequence: q and out [n_seqs, nq, d], seq_len [n_seqs] keys each (none: zeros).  With `ranges` > 1, part_acc holds n_seqs nq ranges d floats and part_ml
// n_seqs nq ranges 2.  A block walks range_pages pages of its
// sequence, the last range whatever is left.
extern "C" int qt_attention_decode_cache8(const void* q, int dtype, const void* k, const void* v, const float* k_scale, const float* v_scale, void* out, const int* block_table,
                                          int max_blocks, int n_pages, const int* seq_len, int n_seqs, int nq, int nkv, int d, float scale, int ranges, int range_pages,
                                          float* part_acc, float* part_ml, void* stream) {
    if (n_seqs == 0) return QT_OK;
    const int rc = check("attention_decode_cache8", dtype, nq, nkv, d, max_blocks, n_pages, q, k, v, out);
    if (rc) return rc;
    const int tiles = (nq / nkv + ROWS - 1) / ROWS;
    QT_REQUIRE(n_seqs > 0 && n_seqs <= 65535 && (long long)nkv * tiles <= 65535, "attention_decode_cache8: %d sequences of %d heads", n_seqs, nq);
    QT_REQUIRE(ranges >= 1 && range_pages >= 1 && (ranges == 1 || (part_acc && part_ml)), "attention_decode_cache8: %d ranges of %d pages", ranges, range_pages);
    Params p{q, out, (const uint8_t*)k, (const uint8_t*)v, k_scale, v_scale, block_table, max_blocks, n_pages, nullptr, nullptr, seq_len, nq, nkv, d, scale, ranges,
             range_pages, part_acc, part_ml};
    const dim3 grid(ranges, nkv * tiles, n_seqs);
    return dtype == QT_F32 ? launch_size<float>(p, grid, (cudaStream_t)stream) : launch_size<__nv_bfloat16>(p, grid, (cudaStream_t)stream);
}

// Packed queries [n_tokens, nq, d] of sequences whose keys, this call's own among them, are in the cache; causal.
extern "C" int qt_attention_prefill_cache8(const void* q, int dtype, const void* k, const void* v, const float* k_scale, const float* v_scale, void* out, const int* block_table,
                                           int max_blocks, int n_pages, const int* seq_start, const int* seq_past, int n_seqs, int max_q_len, int nq, int nkv, int d,
                                           float scale, void* stream) {
    if (n_seqs == 0 || max_q_len == 0) return QT_OK;
    const int rc = check("attention_prefill_cache8", dtype, nq, nkv, d, max_blocks, n_pages, q, k, v, out);
    if (rc) return rc;
    QT_REQUIRE(n_seqs > 0 && n_seqs <= 65535 && nkv <= 65535 && max_q_len > 0 && (long long)max_q_len * (nq / nkv) <= 0x7fffffff - ROWS,
               "attention_prefill_cache8: %d sequences of up to %d tokens", n_seqs, max_q_len);
    Params p{q, out, (const uint8_t*)k, (const uint8_t*)v, k_scale, v_scale, block_table, max_blocks, n_pages, seq_start, seq_past, nullptr, nq, nkv, d, scale, 1,
             0x7fffffff / PAGE, nullptr, nullptr};
    const dim3 grid((unsigned)((max_q_len * (nq / nkv) + ROWS - 1) / ROWS), nkv, n_seqs);
    return dtype == QT_F32 ? launch_size<float>(p, grid, (cudaStream_t)stream) : launch_size<__nv_bfloat16>(p, grid, (cudaStream_t)stream);
}

QT_DEFINE_LAST_ERROR(attention_cache8)
