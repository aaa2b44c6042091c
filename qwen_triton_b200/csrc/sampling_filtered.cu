// One token per row of float logits with parameters of the row's own: temperature T, top_k, top_p, min_p and a given uniform number u.
//
//   y_i = (x_i - max x) / T,  w_i = e^(y_i)
//   top_k   a token stays if fewer than k logits lie strictly above its own
//   top_p   of these, a token stays if the mass of those strictly above it is less than p times the mass of all of them
//   min_p   of these, a token stays if w_i >= min_p
//   token = the first id, in vocabulary order, at which the running mass of what stays exceeds u times the whole; its log-probability is
//           y - log(mass)
//
// So tokens that tie share their fate, and every filter is a threshold on the logit.  A mass is a sum of whole numbers, w in units of 2^-40
// of the largest: w has 24 bits, so a weight above 2^-16 loses nothing and a smaller one at most 2^-41, and no order of additions shows.
// T <= 0 takes the lowest id of the largest logit (log-probability 0).  NaN counts as -inf; a row without anything above -inf gives id 0 with
// log-probability -inf.
#include "common.cuh"

#include <math.h>

using namespace qt;

namespace {

constexpr int THREADS = 1024;
typedef unsigned long long u64;

// Floats as unsigned integers of the same order; the two zeros share a key, NaN is -inf.
__device__ __forceinline__ unsigned int ordered_key(float x) {
    if (isnan(x)) x = -INFINITY;
    unsigned int bits = __float_as_uint(x);
    if (bits == 0x80000000u) bits = 0u;
    return (bits & 0x80000000u) ? ~bits : (bits | 0x80000000u);
}

__device__ __forceinline__ float depth_of(float x, float mx, float t) { return (x == mx ? 0.f : (isnan(x) ? -INFINITY : x - mx)) / t; }
__device__ __forceinline__ u64 units_of(float w) { return (u64)__float2ll_rn(w * 1099511627776.f); }

__device__ u64 block_total(u64 v, u64* scratch) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    v = scratch[threadIdx.x & 31];
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    return v;
}

struct Rows {
    const float* logits; long long row_stride;
    const float* temperature; const int* top_k; const float* top_p; const float* min_p; const float* uniform;
    int* token; float* logprob;
    int vocab;
};

__global__ void __launch_bounds__(THREADS) sample_filtered_kernel(const Rows r) {
    pdl_launch_dependents();
    pdl_wait();
    __shared__ u64 scratch[32];
    __shared__ u64 warp_mass[32];
    __shared__ float best[32];
    const int at = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const float* row = r.logits + at * r.row_stride;
    const float t = r.temperature[at];
    float mx = -INFINITY;
    for (int i = threadIdx.x; i < r.vocab; i += THREADS) mx = fmaxf(mx, row[i]);
    mx = warp_max(mx);
    if (lane == 0) best[warp] = mx;
    __syncthreads();
    mx = warp_max(best[lane]);
    if (!(t > 0.f) || mx == -INFINITY) {
        unsigned int first = 0x7fffffffu;
        for (int i = threadIdx.x; i < r.vocab; i += THREADS)
            if (row[i] == mx) { first = i; break; }
        first = __reduce_min_sync(0xffffffffu, first);
        if (lane == 0) scratch[warp] = first;
        __syncthreads();
        if (threadIdx.x == 0) {
            u64 token = scratch[0];
            for (int w = 1; w < 32; ++w) token = scratch[w] < token ? scratch[w] : token;
            r.token[at] = mx == -INFINITY ? 0 : (int)token;
            if (r.logprob) r.logprob[at] = mx == -INFINITY ? -INFINITY : 0.f;
        }
        return;
    }
    unsigned int floor_key = 0;
    const int k = r.top_k[at];
    if (k > 0 && k < r.vocab) {                              // the lowest threshold above which fewer than k logits lie
        unsigned int low = 0, high = ordered_key(mx);
        while (low < high) {
            const unsigned int mid = low + (high - low) / 2;
            u64 n = 0;
            for (int i = threadIdx.x; i < r.vocab; i += THREADS) n += ordered_key(row[i]) > mid;
            if (block_total(n, scratch) < (u64)k) high = mid; else low = mid + 1;
        }
        floor_key = low;
    }
    auto mass_above = [&](unsigned int key, bool with) {
        u64 m = 0;
        for (int i = threadIdx.x; i < r.vocab; i += THREADS) {
            const float x = row[i];
            const unsigned int mine = ordered_key(x);
            if (mine > key || (with && mine == key)) m += units_of(expf(depth_of(x, mx, t)));
        }
        return block_total(m, scratch);
    };
    const float p = r.top_p[at];
    if (p < 1.f) {                                           // the lowest threshold above which less than p of the mass lies
        const double target = (double)p * (double)mass_above(floor_key, true);
        unsigned int low = floor_key, high = ordered_key(mx);
        while (low < high) {
            const unsigned int mid = low + (high - low) / 2;
            if ((double)mass_above(mid, false) < target) high = mid; else low = mid + 1;
        }
        floor_key = low;
    }
    const float least = fminf(r.min_p[at], 1.f);
    const int chunk = ((r.vocab + 31) / 32 + 31) & ~31;      // ids a warp, in vocabulary order
    const int begin = min(r.vocab, warp * chunk), end = min(r.vocab, begin + chunk);
    auto mass_at = [&](int i) -> u64 {
        if (i >= end) return 0;
        const float x = row[i];
        if (ordered_key(x) < floor_key) return 0;
        const float w = expf(depth_of(x, mx, t));
        return w < least ? 0 : units_of(w);
    };
    u64 mine = 0;
    for (int i = begin + lane; i < end; i += 32) mine += mass_at(i);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, off);
    if (lane == 0) warp_mass[warp] = mine;
    __syncthreads();
    u64 total = 0, before = 0;
    for (int w = 0; w < 32; ++w) { if (w == warp) before = total; total += warp_mass[w]; }
    const double wanted = floor((double)r.uniform[at] * (double)total);
    u64 target = wanted > 0. ? (u64)wanted : 0;
    if (target >= total) target = total - 1;                 // a number of 1 and more: the last token that stays
    if (before <= target && target < before + warp_mass[warp]) {
        u64 running = before;
        for (int i0 = begin; i0 < end; i0 += 32) {
            const u64 m = mass_at(i0 + lane);
            u64 prefix = m;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const u64 other = __shfl_up_sync(0xffffffffu, prefix, off);
                if (lane >= off) prefix += other;
            }
            const unsigned int beyond = __ballot_sync(0xffffffffu, running + prefix > target);
            if (beyond) {
                const int token = i0 + __ffs(beyond) - 1;
                if (lane == 0) {
                    r.token[at] = token;
                    if (r.logprob) r.logprob[at] = depth_of(row[token], mx, t) - logf((float)total * (1.f / 1099511627776.f));
                }
                return;
            }
            running += __shfl_sync(0xffffffffu, prefix, 31);
        }
    }
}

}  // namespace

// logits [rows, vocab] float with rows `row_stride` elements apart; temperature, top_p, min_p, uniform float [rows], top_k int [rows]; token int [rows],
// logprob float [rows] or null.
extern "C" int qt_sample_filtered(const float* logits, long long row_stride, const float* temperature, const int* top_k, const float* top_p,
                                  const float* min_p, const float* uniform, int* token, float* logprob, int rows, int vocab, void* stream) {
    QT_REQUIRE(rows >= 0 && vocab > 0 && (rows <= 1 || row_stride >= vocab), "sample_filtered: bad sizes rows=%d vocab=%d stride=%lld", rows, vocab, row_stride);
    if (rows == 0) return QT_OK;
    const Rows r{logits, row_stride, temperature, top_k, top_p, min_p, uniform, token, logprob, vocab};
    launch_kernel(sample_filtered_kernel, dim3(rows), dim3(THREADS), 0, (cudaStream_t)stream, r);
    QT_CHECK_LAUNCH("sample_filtered");
    return QT_OK;
}

QT_DEFINE_LAST_ERROR(sampling_filtered)
