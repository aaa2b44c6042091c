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
// of the largest: w has 24 bits, so a weight above 2^-16 loses nothing and a smaller one at most 2^-41, and no order of additions shows.  A row of 2^24 equal
// logits would sum to 2^64, which 64 bits do not hold: a call of more than 2^23 is refused.
// T <= 0 takes the lowest id of the largest logit (log-probability 0).  NaN counts as -inf; a row without anything above -inf gives id 0 with
// log-probability -inf.
//
// A row is shared by a cluster of up to eight blocks.  What survives the filters is a small head of the row as a rule, and is found in one pass over the row:
//
//   * every thread notes the largest logit of each few of its turns.  These go into 256 bins by their distance below the row's largest; where the bins' running
//     count reaches top_k (or their mass p times the row's mass) lies a bound that at least so many tokens reach, and seldom many more;
//   * only where a noted logit lies above the bound (min_p gives one by itself) the tokens behind it are read again, and those above the bound go to the first
//     block in vocabulary order; that block sorts their keys, finds the thresholds on the running count and mass, and draws.
//
// Only the row's mass for top_p without top_k takes an exponential a token, an approximate one, in the same pass.  Where the threshold lies within that mass's error
// the mass is formed again, in units.  A row whose head does not fit the list finds its thresholds by bins of all of its tokens, each 256 times narrower than the one
// before, until the bin of the threshold has few tokens, which are sorted (three times; a bin that is still longer than the list is bisected).  Such a row, and one
// without filters, draws over all blocks.  For these passes a block keeps its ids in shared memory where they fit, and reads them again otherwise.
//
// The first pass goes at the memory's rate where every row is read at once, by few blocks a row if rows are many; passes with exponentials want many blocks a row.  So rows
// that need those are then marked and left to a second launch.
//
// Measured behind a cold cache: one row of 151,936 14.5 us, 64 rows 31 to 59, 256 rows (156 MB, 24 us of copying) 113 to 139, by what the rows ask for; with every row on
// eight blocks that kept it in shared memory (37 rows at a time) 15.8, 49 to 78 and 131 to 170.  A row of 256 is read in 30 us; the rest is the head: what it runs is
// short and serial (bins 5 us, tokens read again 4 to 17, sort and draw 8 to 12), so that its instructions' way into the SM counts, and loops stay loops.
#include "common.cuh"

#include <math.h>

using namespace qt;

namespace {

constexpr int THREADS = 512;
constexpr int WARPS = THREADS / 32;
constexpr int MAX_BLOCKS = 8;
constexpr int BINS = 256;
constexpr int LIST = 2048;             // tokens that the first block takes; a block of b hands over LIST / b at most
constexpr float BINS_PER_NAT = 8.f;
constexpr int TURNS = 5;               // turns whose loads are in flight together in the first pass; a noted logit is the largest of so many, or of a multiple
constexpr int WAITING = 32 * (TURNS + 1);
constexpr int FEW = 256;               // keys that are sorted rather than sent through narrower bins
constexpr int MARK = -1, TAKEN = -2;   // in place of a token: the row is left to the second launch; a cluster of that launch has it
constexpr int MAX_NOTES = 16;          // noted logits of a thread
constexpr int MAX_VOCAB = 1 << 23;     // whose masses fit 64 bits, whatever the row
constexpr double LOG2E = 1.4426950408889634;
typedef unsigned long long u64;

struct Rows {
    const float* logits; long long row_stride;
    const float* temperature; const int* top_k; const float* top_p; const float* min_p; const float* uniform;
    int* token; float* logprob;
    int rows, vocab, blocks, turns, span;      // blocks a row; turns of a warp over its ids, 128 a turn; turns a noted logit
    int cached;                        // whether a block keeps its ids in shared memory for further passes
    int mark;                          // whether rows that need more passes get MARK for a token
    double mass_error;
};

// How far, relative to it, a row's mass from the first pass may lie from the sum of units that decides.
//
//   first pass   2^-22 of each exponential; 2^-24 for each of seven additions of floats; a thread's sum is scaled once more for each time its largest logit grew,
//                TURNS turns at a time, and once at the end, 2^-22 of an expf each (of all floats from -87 to 0, 2.6 2^-24 at most)
//   units        2^-22 of an expf, and half a unit, 2^-41, of every token
//   exponents    in both, a difference and a quotient or product are rounded, 2^-24 of the exponent each; steps on a thread's way to the largest logit add up to
//                the token's distance y from it.  On the average that the weights give, y is their entropy less the logarithm of their sum, at most ln(vocabulary)
inline double mass_error(int vocab, int turns) {
    return (4. + (turns + TURNS - 1) / TURNS + log((double)vocab) + vocab / 524288.) / 4194304.;
}

// Floats as unsigned integers of the same order (no NaN comes here); the two zeros share a key.
__device__ __forceinline__ unsigned int ordered_key(float x) {
    unsigned int bits = __float_as_uint(x);
    if (bits == 0x80000000u) bits = 0u;
    return (bits & 0x80000000u) ? ~bits : (bits | 0x80000000u);
}
__device__ __forceinline__ float of_key(unsigned int key) { return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key); }

// The number of a key, -inf for that of no number.
__device__ __forceinline__ float least_of(unsigned int key) { return key == 0 ? -INFINITY : of_key(key); }
__device__ __forceinline__ float below(float x, float mx) { return x == mx ? 0.f : x - mx; }      // two equal infinities too

// e^((x - mx) / t) without a branch, so that several can be under way.  The quotient is that of a division, by Markstein's method (a product with the rounded
// reciprocal, and a correction by the exact remainder): t and the numerator are scaled to t in [1, 2), and what is 200 t below the largest weighs nothing.
struct Weigh {
    float mx, scale, t, inverse, lowest;
    __device__ __forceinline__ Weigh(float mx, float temperature) : mx(mx) {
        const int exponent = (int)(__float_as_uint(temperature) >> 23) - 127;
        scale = __uint_as_float((unsigned int)(127 - min(max(exponent, -127), 126)) << 23);
        t = temperature * scale;
        inverse = 1.f / t;
        lowest = -200.f * t;
    }
    __device__ __forceinline__ float operator()(float x) const {
        const float d = fmaxf(below(x, mx) * scale, lowest), q = d * inverse;
        return expf(fmaf(fmaf(-q, t, d), inverse, q));
    }
};
// w in units of 2^-40, rounded to nearest even: the whole units of 2^-20, then what is left, each by adding a number whose last place is one.
__device__ __forceinline__ u64 units_of(float w) {
    const float high = w * 1048576.f, sum = high + 8388608.f;
    const float low = (high - (sum - 8388608.f)) * 1048576.f + 12582912.f;
    return ((u64)(__float_as_uint(sum) - 0x4b000000u) << 20) + (long long)(int)(__float_as_uint(low) - 0x4b400000u);
}

__device__ __forceinline__ u64 warp_total(u64 v) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    return v;
}
__device__ __forceinline__ u64 warp_prefix(u64 v, int lane) {                                     // inclusive
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const u64 other = __shfl_up_sync(0xffffffffu, v, off);
        if (lane >= off) v += other;
    }
    return v;
}

__device__ __forceinline__ void remote_store(const unsigned int* local, uint32_t rank, unsigned int value) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"((uint32_t)__cvta_generic_to_shared(local)), "r"(rank));
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(remote), "r"(value) : "memory");
}
__device__ __forceinline__ unsigned int remote_add(const unsigned int* local, uint32_t rank) {
    uint32_t remote;
    unsigned int before;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"((uint32_t)__cvta_generic_to_shared(local)), "r"(rank));
    asm volatile("atom.shared::cluster.add.u32 %0, [%1], 1;" : "=r"(before) : "r"(remote) : "memory");
    return before;
}
__device__ __forceinline__ void remote_store(const u64* local, uint32_t rank, u64 value) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"((uint32_t)__cvta_generic_to_shared(local)), "r"(rank));
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(remote), "l"(value) : "memory");
}
__device__ __forceinline__ unsigned int remote_load(const unsigned int* local, uint32_t rank) {
    uint32_t remote;
    unsigned int value;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"((uint32_t)__cvta_generic_to_shared(local)), "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(value) : "r"(remote) : "memory");
    return value;
}

struct Shared {
    u64 slots[2][MAX_BLOCKS][2];                 // two numbers of every block, by turns
    u64 scratch[WARPS][2];
    u64 per_warp[WARPS];
    unsigned int bins[2][3][BINS];               // count, mass low, mass high, by turns
    unsigned int bin_found, bin_tokens, taken;
    u64 above, all;
};

// The sum of the warps' numbers (their last lane's) in front of this one; all: of all of them.
__device__ __noinline__ u64 warps_before(u64 mine, u64* per_warp, int warp, int lane, u64& all) {
    __syncthreads();
    if (lane == 31) per_warp[warp] = mine;
    __syncthreads();
    u64 base = 0;
    all = 0;
#pragma unroll 4
    for (int w = 0; w < WARPS; ++w) { const u64 n = per_warp[w]; if (w < warp) base += n; all += n; }
    return base;
}
// n <= LIST keys, largest first (bitonic, the next power of two filled up with zeros).
__device__ __noinline__ void sort_down(unsigned int* keys, int n) {
    int size = 32;
    while (size < n) size *= 2;
    for (int i = n + threadIdx.x; i < size; i += THREADS) keys[i] = 0;
    for (int k = 2; k <= size; k *= 2)
        for (int j = k / 2; j > 0; j /= 2) {
            __syncthreads();
            for (int i = threadIdx.x; i < size / 2; i += THREADS) {
                const int a = 2 * i - (i & (j - 1)), b = a + j;                  // the pair of this step
                const unsigned int x = keys[a], y = keys[b];
                if ((a & k) == 0 ? x < y : x > y) { keys[a] = y; keys[b] = x; }
            }
        }
    __syncthreads();
}

// Of n sorted keys, the last of at least floor_key in front of which less than `wanted` lies (their number or their mass, `above` included; `share` of what all of
// them have where it is positive); the first if there is none.  Beside it in bit 32, whether a key, or the list's end, begins within `error` of that; error < 0: whether
// the list ends in front of it.
// One copy of this and of the sort: a block waits for instructions that it runs once.
__device__ __noinline__ u64 cut(const unsigned int* keys, u64* before, u64* per_warp, int n, bool by_mass, unsigned int floor_key, u64 above, double wanted, double share,
                                double error, Weigh weigh) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    u64 total = above;
#pragma unroll 1
    for (int j = 0; j < n; j += THREADS) {
        const int i = j + threadIdx.x;
        const u64 own = i >= n || keys[i] < floor_key ? 0 : by_mass ? units_of(weigh(of_key(keys[i]))) : 1, upto = warp_prefix(own, lane);
        u64 all;
        const u64 base = warps_before(upto, per_warp, warp, lane, all);
        if (i < n) before[i] = total + base + upto - own;
        total += all;
    }
    if (share > 0.) wanted = share * (double)total;
    bool doubt = error < 0. ? (double)total < wanted : fabs((double)total - wanted) <= error;
    int last = 0;
    for (int i = threadIdx.x; i < n; i += THREADS) {
        const double lies = (double)before[i];
        if (keys[i] >= floor_key && lies < wanted) last = i;
        doubt |= i > 0 && fabs(lies - wanted) <= error;
    }
    last = __reduce_max_sync(0xffffffffu, last);
    doubt = __syncthreads_or(doubt);
    if (lane == 0) per_warp[warp] = last;
    __syncthreads();
    return (u64)doubt << 32 | keys[__reduce_max_sync(0xffffffffu, lane < WARPS ? (int)per_warp[lane] : 0)];
}

__device__ __forceinline__ u64 target_of(u64 total, float uniform) {
    const double wanted = floor((double)uniform * (double)total);
    const u64 target = wanted > 0. ? (u64)wanted : 0;
    return target < total ? target : total - 1;               // a number of 1 and more: the last token that stays
}
__device__ __forceinline__ void give_answer(const Rows& r, int at, int token, float depth, u64 total) {
    r.token[at] = token;
    if (r.logprob) r.logprob[at] = depth - logf((float)total * (1.f / 1099511627776.f));
}
// Adds a token to its bin of [count, mass low, mass high][BINS].
__device__ __forceinline__ void add_to_bins(unsigned int (*bins)[BINS], int bin, bool by_mass, u64 m, bool count = true) {
    if (count) atomicAdd(&bins[0][bin], 1u);
    if (!by_mass) return;
    const unsigned int low = (unsigned int)m, before = atomicAdd(&bins[1][bin], low);
    const unsigned int high = (unsigned int)(m >> 32) + (before > 0xffffffffu - low ? 1u : 0u);
    if (high) atomicAdd(&bins[2][bin], high);
}

// Above 1e30 the weights of finite logits are alike; NaN stays.
__device__ __forceinline__ float temperature_of(const Rows& r, int at) { const float t = r.temperature[at]; return t > 1e30f ? 1e30f : t; }

struct Filters {
    int k;
    float p, least;
    bool by_count, by_mass, by_weight;
    __device__ __forceinline__ Filters(const Rows& r, int at) : k(r.top_k[at]), p(r.top_p[at]) {
        const float m = r.min_p[at];
        least = m > 0.f ? fminf(m, 1.f) : 0.f;
        by_count = k > 0 && k < r.vocab, by_mass = p < 1.f, by_weight = least > 0.f;
    }
};

struct Row {
    const Rows& r;
    Shared& sh;
    const float* row;
    float4* kept;                                // this block's ids, where they are kept
    float* notes;                                // [note][thread]; null: not wanted
    unsigned int* waiting;                       // [WAITING] of a warp: quads to be read again, in vocabulary order
    unsigned int* keys;                          // [LIST], the first block's, to be sorted
    u64* before;                                 // [LIST], the first block's: what lies before each
    int rank, blocks, warp, lane, shift, quads, turn;
    float mx, t;

    // ids in fours from the 16-byte boundary at or before the row's start on; a place outside the row is -inf
    __device__ __forceinline__ int quad_at(int i) const { return ((rank * WARPS + warp) * r.turns + i) * 32 + lane; }
    __device__ __forceinline__ float4 load(int i) const { return load_quad(quad_at(i)); }
    __device__ __forceinline__ float4 load_quad(int q) const {
        const int id = 4 * q - shift;
        float4 v = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        if (q < quads) {
            if (id >= 0 && id + 4 <= r.vocab) {
                v = *reinterpret_cast<const float4*>(row + id);
            } else {
                if (id >= 0 && id < r.vocab) v.x = row[id];
                if (id + 1 >= 0 && id + 1 < r.vocab) v.y = row[id + 1];
                if (id + 2 >= 0 && id + 2 < r.vocab) v.z = row[id + 2];
                if (id + 3 >= 0 && id + 3 < r.vocab) v.w = row[id + 3];
            }
        }
        return v;
    }
    static __device__ __forceinline__ float without_nan(float x) { return fmaxf(x, -INFINITY); }
    static __device__ __forceinline__ float4 without_nan(float4 v) { return make_float4(without_nan(v.x), without_nan(v.y), without_nan(v.z), without_nan(v.w)); }
    // quad number q of this block, whichever thread has read it
    __device__ __forceinline__ float4 any_quad(int q) const { return r.cached ? kept[q] : without_nan(load_quad(rank * WARPS * r.turns * 32 + q)); }
    struct Four { float x[4]; };
    // Another pass over this thread's logits.  The loop stays a loop: with an exponential and a division for every number, a pass that is unrolled is tens of
    // kilobytes of instructions that run once or twice, and a block waits for those.
    template <typename F> __device__ __forceinline__ void each(F f) const {
#pragma unroll 1
        for (int i = 0; i < r.turns; ++i) {
            const float4 v = any_quad((warp * r.turns + i) * 32 + lane);
            f({v.x, v.y, v.z, v.w});
        }
    }

    // The first pass: notes the largest logit of each `span` turns and returns this thread's.  With SUM, sum becomes the mass of this thread's logits in units of
    // that of its largest: one exponential a token against the largest so far, and the sum scaled where that grows.
    template <bool SUM> __device__ __forceinline__ float fetch(double& sum) const {
        float best = -INFINITY;
        sum = 0.;
        const float per_nat = (float)(LOG2E / t), rest = (float)(LOG2E / t - per_nat), lowest = -200.f * t;       // e^-200: nothing
        for (int note = 0, i0 = 0; i0 < r.turns; ++note) {
            float top = -INFINITY;
            for (const int end = min(i0 + r.span, r.turns); i0 < end; i0 += TURNS) {
                float4 v[TURNS];
#pragma unroll
                for (int j = 0; j < TURNS; ++j) v[j] = i0 + j < end ? load(i0 + j) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                float most = -INFINITY;
#pragma unroll
                for (int j = 0; j < TURNS; ++j) most = fmaxf(most, fmaxf(fmaxf(v[j].x, v[j].y), fmaxf(v[j].z, v[j].w)));
                top = fmaxf(top, most);
                if (r.cached) {
#pragma unroll
                    for (int j = 0; j < TURNS; ++j) if (i0 + j < end) kept[(warp * r.turns + i0 + j) * 32 + lane] = without_nan(v[j]);
                }
                if (SUM) {
                    if (most > best) { sum = best > -INFINITY ? sum * expf((best - most) / t) : 0.; best = most; }
                    if (best > -INFINITY) {
                        auto of = [&](float x) {
                            const float d = fmaxf(x - best, lowest);          // NaN too
                            float e;
                            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fmaf(d, per_nat, d * rest)));
                            return e;
                        };
                        float part = 0.f;
#pragma unroll
                        for (int j = 0; j < TURNS; ++j) part += (of(v[j].x) + of(v[j].y)) + (of(v[j].z) + of(v[j].w));
                        sum += part;
                    }
                }
            }
            best = fmaxf(best, top);
            if (notes) notes[note * THREADS + threadIdx.x] = top;
        }
        return best;
    }
    // Calls f(quad of the block, logits) for the quads behind this warp's notes that `hit` takes, in vocabulary order, up to 32 of them in a call (lanes
    // without one: logits of -inf); ends where f returns false.
    template <typename H, typename F> __device__ __forceinline__ void again(H hit, F f) const {
        int have = 0;
        auto take = [&](int from, int n) {
            const int q = lane < n ? (int)waiting[from + lane] : 0;
            return f(q, lane < n ? any_quad(q) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY));
        };
        for (int note = 0; note * r.span < r.turns; ++note) {
            const unsigned int lanes = __ballot_sync(0xffffffffu, hit(notes[note * THREADS + threadIdx.x]));
            if (lanes == 0) continue;
            const int all = __popc(lanes), end = min((note + 1) * r.span, r.turns);
            const bool mine = lanes >> lane & 1;
            for (int i = note * r.span; i < end; i += TURNS) {
                int to = have + __popc(lanes & ((1u << lane) - 1));
#pragma unroll
                for (int j = 0; j < TURNS; ++j, to += all) if (mine && i + j < end) waiting[to] = (unsigned int)(warp * r.turns + i + j) * 32 + lane;
                have += all * min(TURNS, end - i);
                __syncwarp();
                int from = 0;
                for (; have - from >= 32; from += 32) if (!take(from, 32)) return;
                if (from == 0) continue;
                const unsigned int rest = from + lane < have ? waiting[from + lane] : 0;
                __syncwarp();
                have -= from;
                if (lane < have) waiting[lane] = rest;
                __syncwarp();
            }
        }
        if (have > 0) take(0, have);
    }

    __device__ __forceinline__ void barrier() const { if (blocks > 1) cluster_barrier(); else __syncthreads(); }
    // Every block's two numbers (all of its first threads have them), seen by all: sh.slots[returned][block].
    __device__ __forceinline__ int exchange(u64 a, u64 b) {
        const int at = turn;
        turn ^= 1;
        if (threadIdx.x < blocks) {
            if (blocks > 1) { remote_store(&sh.slots[at][rank][0], threadIdx.x, a); remote_store(&sh.slots[at][rank][1], threadIdx.x, b); }
            else { sh.slots[at][0][0] = a; sh.slots[at][0][1] = b; }
        }
        barrier();
        return at;
    }
    // Sums over the row of what every thread brings.
    __device__ __forceinline__ u64 row_total(u64 v) {
        v = warp_total(v);
        __syncthreads();
        if (lane == 0) sh.scratch[warp][0] = v;
        __syncthreads();
        v = warp_total(lane < WARPS ? sh.scratch[lane][0] : 0);
        const int at = exchange(v, 0);
        u64 all = 0;
        for (int k = 0; k < blocks; ++k) all += sh.slots[at][k][0];
        return all;
    }
    // The least and the largest.
    __device__ __forceinline__ void row_ends(unsigned int& least, unsigned int& most) {
        least = __reduce_min_sync(0xffffffffu, least);
        most = __reduce_max_sync(0xffffffffu, most);
        __syncthreads();
        if (lane == 0) { sh.scratch[warp][0] = least; sh.scratch[warp][1] = most; }
        __syncthreads();
        least = __reduce_min_sync(0xffffffffu, lane < WARPS ? (unsigned int)sh.scratch[lane][0] : 0xffffffffu);
        most = __reduce_max_sync(0xffffffffu, lane < WARPS ? (unsigned int)sh.scratch[lane][1] : 0u);
        const int at = exchange(least, most);
        for (int k = 0; k < blocks; ++k) {
            least = min(least, (unsigned int)sh.slots[at][k][0]);
            most = max(most, (unsigned int)sh.slots[at][k][1]);
        }
    }

    __device__ __forceinline__ float depth(float x) const { return below(x, mx) / t; }
    __device__ __forceinline__ Weigh weigh() const { return Weigh(mx, t); }

    __device__ __forceinline__ void clear_bins(int at) const {
        for (int i = threadIdx.x; i < 3 * BINS; i += THREADS) (&sh.bins[at][0][0])[i] = 0;
    }
    // After a barrier behind the last addition: the first bin at which the running number over all blocks, started from `above`, reaches `wanted`, or `share` of
    // all of them where share > 0 (wanted: that).  above: the number in front of it; sh.bin_tokens: its tokens.  BINS where none does.
    __device__ __forceinline__ int find_bin(int at, bool by_mass, double& wanted, double share, u64& above) {
        __syncthreads();
        if (threadIdx.x == 0) { sh.bin_found = BINS; sh.above = above; }
        u64 n = 0, upto = 0;
        unsigned int tokens = 0;
        if (threadIdx.x < BINS) {                             // a thread a bin, all blocks' loads in flight together
            unsigned int count[MAX_BLOCKS], low[MAX_BLOCKS], high[MAX_BLOCKS];
            auto load = [&](int what, int k) { return blocks > 1 ? remote_load(&sh.bins[at][what][threadIdx.x], k) : sh.bins[at][what][threadIdx.x]; };
#pragma unroll
            for (int k = 0; k < MAX_BLOCKS; ++k) {
                count[k] = k < blocks ? load(0, k) : 0;
                low[k] = k < blocks && by_mass ? load(1, k) : 0;
                high[k] = k < blocks && by_mass ? load(2, k) : 0;
            }
#pragma unroll
            for (int k = 0; k < MAX_BLOCKS; ++k) { tokens += count[k]; n += ((u64)high[k] << 32) + low[k]; }
            if (!by_mass) n = tokens;
            upto = warp_prefix(n, lane);
            if (lane == 31) sh.per_warp[warp] = upto;
        }
        __syncthreads();
        if (threadIdx.x < BINS) {
            u64 all = 0;
#pragma unroll
            for (int i = 0; i < BINS / 32; ++i) { if (i < warp) upto += sh.per_warp[i]; all += sh.per_warp[i]; }
            if (share > 0.) wanted = share * (double)all;
            upto += above;
            if ((double)upto >= wanted && (threadIdx.x == 0 || (double)(upto - n) < wanted)) { sh.bin_found = threadIdx.x; sh.above = upto - n; sh.bin_tokens = tokens; }
            if (threadIdx.x == 0) sh.all = all;
        }
        __syncthreads();
        if (share > 0.) wanted = share * (double)sh.all;
        above = sh.above;
        return sh.bin_found;
    }

    // The lowest threshold above which (strictly) less than `wanted` of the tokens with a key of at least floor_key lies: their number, or their mass, of which
    // `share` is wanted where it is positive.
    __device__ unsigned int threshold(bool by_mass, double wanted, double share, unsigned int floor_key) {
        u64 above = 0;
        int prefix = 0, level = 0, tokens = 0;
        float scale = BINS_PER_NAT / t;
        const float floor_x = least_of(floor_key);
        const Weigh weight = weigh();
        auto index_of = [&](float x) {
            const float at = -below(x, mx) * scale;
            const int index = at < 1073741824.f ? (int)at : 1073741824;
            return level == 0 ? min(index, BINS - 1) : index;
        };
        for (;; ++level, scale *= 256.f) {                    // a power of two: a place is that of the level before and eight bits more
            clear_bins(level & 1);
            __syncthreads();
            each([&](const Four& v) {
                int index[4];
                bool in[4];
                u64 m[4] = {};
                for (int e = 0; e < 4; ++e) {
                    index[e] = index_of(v.x[e]);
                    in[e] = v.x[e] >= floor_x && (level == 0 || index[e] >> 8 == prefix);
                }
                if (by_mass && __any_sync(0xffffffffu, in[0] || in[1] || in[2] || in[3]))
                    for (int e = 0; e < 4; ++e) m[e] = units_of(weight(v.x[e]));
                for (int e = 0; e < 4; ++e) if (in[e]) add_to_bins(sh.bins[level & 1], index[e] & (BINS - 1), by_mass, m[e], !by_mass || level > 0);
            });
            barrier();
            const int bin = find_bin(level & 1, by_mass, wanted, level == 0 ? share : 0., above);
            if (bin == BINS) { barrier(); return floor_key; } // all of them are less than is wanted
            prefix = (prefix << 8) + bin;
            // the last bin of the first level has no lower end
            tokens = by_mass && level == 0 ? LIST + 1 : (int)sh.bin_tokens;        // masses alone at first: no row comes here for a few tokens
            if (tokens <= FEW || level == 2 || (level == 0 && bin == BINS - 1) || !(scale * 65536.f < INFINITY)) break;
        }
        auto inside = [&](float x) { return x >= floor_x && index_of(x) == prefix; };
        unsigned int found;
        if (tokens <= LIST) {                                 // the bin's keys to the first block, in any order: they are sorted there
            if (threadIdx.x == 0) sh.taken = 0;
            barrier();
            each([&](const Four& v) { for (int e = 0; e < 4; ++e) if (inside(v.x[e])) remote_store(keys + remote_add(&sh.taken, 0), 0, ordered_key(v.x[e])); });
            barrier();
            found = 0;
            if (rank == 0) {
                sort_down(keys, tokens);
                found = (unsigned int)cut(keys, before, sh.per_warp, tokens, by_mass, 0u, above, wanted, 0., 0., weigh());
            }
            const int slot = exchange(found, 0);
            found = (unsigned int)sh.slots[slot][0][0];
        } else {
            unsigned int low = 0xffffffffu, high = 0;
            each([&](const Four& v) {
                for (int e = 0; e < 4; ++e) if (inside(v.x[e])) { low = min(low, ordered_key(v.x[e])); high = max(high, ordered_key(v.x[e])); }
            });
            row_ends(low, high);
            while (low < high) {
                const unsigned int mid = low + (high - low) / 2;
                u64 n = 0;
                each([&](const Four& v) { for (int e = 0; e < 4; ++e) if (ordered_key(v.x[e]) > mid && inside(v.x[e])) n += by_mass ? units_of(weight(v.x[e])) : 1; });
                if ((double)(above + row_total(n)) < wanted) high = mid; else low = mid + 1;
            }
            found = low;
        }
        barrier();                                            // every block is done with the bins
        return max(found, floor_key);
    }

    // The answer of a row without a number above -inf.
    __device__ __forceinline__ void give_nothing(int at) const {
        if (rank != 0 || threadIdx.x != 0) return;
        r.token[at] = 0;
        if (r.logprob) r.logprob[at] = -INFINITY;
    }
    // Thresholds and token by passes over the whole row.
    __device__ __forceinline__ void by_passes(int at, const Filters& f) {
        unsigned int floor_key = 0;
        if (f.by_count) floor_key = threshold(false, (double)f.k, 0., 0u);
        if (f.by_mass) floor_key = f.p > 0.f ? threshold(true, 0., (double)f.p, floor_key) : ordered_key(mx);
        draw(at, floor_key, f.least);
        barrier();
    }

    // The row's mass in units.
    __device__ __forceinline__ u64 mass() {
        const Weigh weight = weigh();
        u64 mine = 0;
        each([&](const Four& v) { for (int e = 0; e < 4; ++e) mine += units_of(weight(v.x[e])); });
        return row_total(mine);
    }
    // Draws among the tokens with a key of at least floor_key and a weight of at least `least`, over all blocks.
    __device__ void draw(int at, unsigned int floor_key, float least) {
        const float floor_x = least_of(floor_key);
        const Weigh weight = weigh();
        auto stays = [&](float x) -> u64 {
            const float w = weight(x);
            const u64 m = units_of(w);
            return x >= floor_x && w >= least ? m : 0;
        };
        u64 mine = 0;
        each([&](const Four& v) { mine += (stays(v.x[0]) + stays(v.x[1])) + (stays(v.x[2]) + stays(v.x[3])); });
        mine = warp_total(mine);
        __syncthreads();
        if (lane == 0) sh.per_warp[warp] = mine;
        __syncthreads();
        u64 block = 0, before = 0;
        for (int w = 0; w < WARPS; ++w) { if (w == warp) before = block; block += sh.per_warp[w]; }
        const int slot = exchange(block, 0);
        u64 total = 0;
        for (int k = 0; k < blocks; ++k) { if (k == rank) before += total; total += sh.slots[slot][k][0]; }
        const u64 target = target_of(total, r.uniform[at]);
        // the warp in whose ids the target falls: its block looks at them again, four a thread
        if (lane == 0 && before <= target && target < before + mine) { sh.taken = warp; sh.above = before; }
        if (threadIdx.x == 0) sh.bin_found = before <= target && target < before + block;      // of warp 0, before is the block's
        __syncthreads();
        if (!sh.bin_found) return;
        u64 running = sh.above;
        const int quad0 = (rank * WARPS + (int)sh.taken) * r.turns * 32, all_quads = r.turns * 32;
        for (int q0 = 0; q0 < all_quads; q0 += THREADS) {
            const int q = q0 + threadIdx.x, id = 4 * (quad0 + q) - shift;
            const float4 v = q < all_quads ? any_quad((int)sh.taken * all_quads + q) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            const u64 m[4] = {stays(v.x), stays(v.y), stays(v.z), stays(v.w)};
            u64 sum = m[0] + m[1] + m[2] + m[3], all;
            const u64 own = sum, in_warp = warp_prefix(own, lane);
            sum = running + warps_before(in_warp, sh.per_warp, warp, lane, all) + in_warp - own;
            if (sum <= target && target < sum + own) {
                int e = 0;
                while (e < 3 && sum + m[e] <= target) sum += m[e++];
                give_answer(r, at, id + e, depth(e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w), total);
            }
            running += all;
        }
    }
};

// Shared memory of the first launch in front of what is kept: list and found, what waits, and the larger of places with notes and keys with what lies before them.
__host__ __device__ __forceinline__ size_t head_bytes(const Rows& r) {
    const size_t noting = LIST * sizeof(unsigned short) + (size_t)((r.turns + r.span - 1) / r.span) * THREADS * sizeof(float);
    const size_t sorting = LIST * (sizeof(unsigned int) + sizeof(u64));
    return 2 * LIST * sizeof(u64) + WARPS * WAITING * sizeof(unsigned int) + (noting > sorting ? noting : sorting);
}

// WHOLE: the list takes every row as it is, so that nothing is bound or summed beforehand.  A kernel of its own, since instructions that run once are waited for: 100
// rows of 503 tokens 14.1 us, by the kernel for all rows 16.1.
template <bool WHOLE> __global__ void __launch_bounds__(THREADS, 2) sample_filtered_kernel(const Rows r) {
    pdl_launch_dependents();
    if (r.blocks > 1) cluster_arrive_started();
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ Shared sh;
    u64* list = reinterpret_cast<u64*>(smem);                  // the first block's: tokens above the bound as (key, id), by block and in vocabulary order
    u64* found = list + LIST;                                  // this block's, as its warps find them, and their places among their warp's
    unsigned int* waiting = reinterpret_cast<unsigned int*>(found + LIST);
    unsigned short* place = reinterpret_cast<unsigned short*>(waiting + WARPS * WAITING);
    float* notes = reinterpret_cast<float*>(place + LIST);
    unsigned int* keys = reinterpret_cast<unsigned int*>(waiting + WARPS * WAITING);       // later, where places and notes were
    u64* before = reinterpret_cast<u64*>(keys + LIST);
    float4* kept = reinterpret_cast<float4*>(smem + head_bytes(r));
    const int blocks = r.blocks, rank = blockIdx.x % blocks, at = blockIdx.x / blocks, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_wait();
    const float* row = r.logits + at * r.row_stride;
    const int shift = (int)(((uintptr_t)row >> 2) & 3);
    Row w{r, sh, row, kept, notes, waiting + warp * WAITING, keys, before, rank, blocks, warp, lane, shift, (r.vocab + shift + 3) / 4, 0, -INFINITY, temperature_of(r, at)};
    w.clear_bins(0);
    const float t = w.t;
    const Filters f(r, at);
    const bool filtered = f.by_count || f.by_mass || f.by_weight;
    if (r.mark && !filtered && t > 0.f) {                      // the same for all blocks of the row
        if (rank == 0 && threadIdx.x == 0) r.token[at] = MARK;
        if (blocks > 1) cluster_wait_started();
        return;
    }
    const bool counting = f.by_count, summing = !WHOLE && f.by_mass && !f.by_count && t > 0.f;
    if (threadIdx.x == 0) sh.taken = 0;
    double sum;
    const float own_best = summing ? w.fetch<true>(sum) : w.fetch<false>(sum);
    if (blocks > 1) cluster_wait_started();
    {
        unsigned int low = 0, high = ordered_key(own_best);
        w.row_ends(low, high);
        w.mx = of_key(high);
    }
    const float mx = w.mx;
    if (!(t > 0.f) || mx == -INFINITY) {                       // the lowest id of the largest logit
        unsigned int first = 0xffffffffu, unused = 0;
        if (mx > -INFINITY)
            w.again([&](float x) { return x == mx; }, [&](int q, float4 v) {
                const unsigned int id = 4 * (rank * WARPS * r.turns * 32 + q) - shift;
                first = v.x == mx ? id : v.y == mx ? id + 1 : v.z == mx ? id + 2 : v.w == mx ? id + 3 : first;
                return !__any_sync(0xffffffffu, first != 0xffffffffu);
            });
        w.row_ends(first, unused);
        if (mx == -INFINITY) {
            w.give_nothing(at);
        } else if (rank == 0 && threadIdx.x == 0) {
            r.token[at] = (int)first;
            if (r.logprob) r.logprob[at] = 0.f;
        }
        w.barrier();
        return;
    }
    bool fits = filtered && mx < INFINITY && t > 1e-30f;
    float bound = -INFINITY;
    double row_mass = 0.;                                      // for top_p alone, in units
    if (fits && !WHOLE) {
        if (f.by_weight && !f.by_count) bound = mx + t * logf(f.least);
        if (f.by_count || f.by_mass) {
            const Weigh weight = w.weigh();
            for (int note = 0; note * r.span < r.turns; ++note) {
                const float x = notes[note * THREADS + threadIdx.x];
                if (x > -INFINITY) add_to_bins(sh.bins[0], min((int)(-w.depth(x) * BINS_PER_NAT), BINS - 1), !counting, counting ? 0 : units_of(weight(x)));
            }
            if (summing) {
                sum = own_best > -INFINITY ? sum * weight(own_best) : 0.;
#pragma unroll
                for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
                if (lane == 0) sh.scratch[warp][1] = (u64)__double_as_longlong(sum);
                __syncthreads();
                sum = 0.;
                for (int i = 0; i < WARPS; ++i) sum += __longlong_as_double((long long)sh.scratch[i][1]);
            }
            const int slot = w.exchange((u64)__double_as_longlong(sum), 0);
            for (int b = 0; b < blocks; ++b) row_mass += __longlong_as_double((long long)sh.slots[slot][b][0]);
            row_mass *= 1099511627776.;
            u64 above = 0;
            double wanted = counting ? (double)f.k : (double)f.p * row_mass;
            const int bin = w.find_bin(0, !counting, wanted, 0., above);
            // every token of the bins up to this one lies above the bound; the last bin has no end
            if (bin < BINS - 1) bound = fmaxf(bound, mx - t * (float)(bin + 1) * (1.f / BINS_PER_NAT));
        }
        // what the bound's and the bins' roundings are, and those of a weight at min_p, 4e-7 of it (at a high temperature many logits lie so near)
        bound -= 1e-5f * (fabsf(mx) + fabsf(mx - bound)) + 1e-6f * t;
    }
    if (fits) {
        auto above = [&](float x) { return x > -INFINITY && !(x < bound); };
        // a long list takes one block longer than the second launch does
        const int room = (r.mark ? LIST / 2 : LIST) / blocks;
        int in_warp = 0;
        w.again(above, [&](int q, float4 v) {
            const int own = above(v.x) + above(v.y) + above(v.z) + above(v.w);
            int upto = own;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int other = __shfl_up_sync(0xffffffffu, upto, off);
                if (lane >= off) upto += other;
            }
            const int all = __shfl_sync(0xffffffffu, upto, 31);
            int slot = 0;
            if (lane == 0) slot = (int)atomicAdd(&sh.taken, (unsigned int)all);
            slot = __shfl_sync(0xffffffffu, slot, 0);
            if (slot + all > room) return false;               // the list has no room for this row: sh.taken says so
            slot += upto - own;
            int of_warp = in_warp + upto - own;
            in_warp += all;
            auto put = [&](float x, int e) {
                if (!above(x)) return;
                found[slot] = ((u64)ordered_key(x) << 32) | (unsigned int)(4 * (rank * WARPS * r.turns * 32 + q) - shift + e);
                place[slot++] = (unsigned short)of_warp++;
            };
            put(v.x, 0); put(v.y, 1); put(v.z, 2); put(v.w, 3);
            return true;
        });
        __syncthreads();
        if (lane == 0) sh.per_warp[warp] = in_warp;
        __syncthreads();
        const int mine = (int)sh.taken;
        if (mine <= room)
            for (int i = threadIdx.x; i < mine; i += THREADS) {
                const int of = (((int)(unsigned int)found[i] + shift) / 4) / (r.turns * 32) - rank * WARPS;
                int to = rank * room + place[i];
                for (int b = 0; b < of; ++b) to += (int)sh.per_warp[b];
                if (blocks > 1) remote_store(list + to, 0, found[i]); else list[to] = found[i];
            }
        const int slot = w.exchange(mine, 0);
        for (int b = 0; b < blocks; ++b) fits = fits && (int)sh.slots[slot][b][0] <= room;
        if (fits && rank > 0) {
            if (!summing || sh.slots[w.exchange(0, 0)][0][0]) return;
            if (!r.mark) {
                w.mass();
                if (sh.slots[w.exchange(0, 0)][0][0]) return;
            }
        } else if (fits) {
            // the first block alone: places j THREADS + thread of the list a thread
            int count = 0;
            for (int b = 0; b < blocks; ++b) count += (int)sh.slots[slot][b][0];
#pragma unroll 1
            for (int to = threadIdx.x; to < count; to += THREADS) {
                int i = to, b = 0;
                while (i >= (int)sh.slots[slot][b][0]) i -= (int)sh.slots[slot][b++][0];
                const u64 entry = list[b * room + i];
                found[to] = entry;                             // what was there is in the list
                keys[to] = (unsigned int)(entry >> 32);
            }
            unsigned int floor_key = 0;
            if (f.by_count || f.by_mass) sort_down(keys, count);
            if (f.by_count && f.k <= count) floor_key = keys[f.k - 1];
            if (f.by_mass) {
                // the likeliest token stays whatever p is
                const double wanted = (double)f.p * row_mass;
                const u64 last = f.p > 0.f ? cut(keys, before, sh.per_warp, count, true, floor_key, 0, wanted, summing ? 0. : (double)f.p, wanted * r.mass_error, w.weigh()) : keys[0];
                floor_key = max(floor_key, (unsigned int)last);
                if (summing) {
                    fits = last >> 32 == 0;
                    w.exchange(fits, 0);
                    // in doubt, which the row's mass in units settles where the list reaches so far (64 rows of 151,936, one or more in doubt: 48 to 60 us, 60 to 119 by
                    // bins of all tokens)
                    if (!fits && !r.mark) {
                        const u64 settled = cut(keys, before, sh.per_warp, count, true, 0u, 0, (double)f.p * (double)w.mass(), 0., -1., w.weigh());
                        floor_key = (unsigned int)settled;
                        fits = settled >> 32 == 0;
                        w.exchange(fits, 0);
                    }
                }
            }
            if (fits) {
                u64 total = 0;
                const Weigh weigh = w.weigh();
#pragma unroll 1
                for (int j = 0; j < count; j += THREADS) {
                    const int i = j + threadIdx.x;
                    u64 own = 0, all;
                    if (i < count && (unsigned int)(found[i] >> 32) >= floor_key) {
                        const float weight = weigh(of_key((unsigned int)(found[i] >> 32)));
                        own = weight < f.least ? 0 : units_of(weight);
                    }
                    const u64 upto = warp_prefix(own, lane), base = warps_before(upto, sh.per_warp, warp, lane, all);
                    if (i < count) before[i] = total + base + upto - own;
                    total += all;
                }
                __syncthreads();
                const u64 target = target_of(total, r.uniform[at]);
#pragma unroll 1
                for (int i = threadIdx.x; i < count; i += THREADS)
                    if (before[i] <= target && target < (i + 1 < count ? before[i + 1] : total))
                        give_answer(r, at, (int)(unsigned int)found[i], w.depth(of_key((unsigned int)(found[i] >> 32))), total);
                return;
            }
        }
    }
    if (r.mark) {
        if (rank == 0 && threadIdx.x == 0) r.token[at] = MARK;
        return;
    }
    w.by_passes(at, f);
}

// The rows that the launch before has marked, each by the cluster that comes to it first; a block looks for them 512 rows at a time (4,096 rows of 20,000,
// every 97th marked: 259 us; a warp 32 at a time 306).
__global__ void __launch_bounds__(THREADS, 2) sample_marked_kernel(const Rows r) {
    pdl_launch_dependents();
    if (r.blocks > 1) cluster_arrive_started();
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ Shared sh;
    const int blocks = r.blocks, rank = blockIdx.x % blocks, cluster = blockIdx.x / blocks, clusters = gridDim.x / blocks, warp = threadIdx.x >> 5,
              lane = threadIdx.x & 31;
    if (blocks > 1) cluster_wait_started();
    pdl_wait();
    unsigned int* keys = reinterpret_cast<unsigned int*>(smem);
    u64* before = reinterpret_cast<u64*>(keys + LIST);
    float4* kept = reinterpret_cast<float4*>(before + LIST);
    const int start = (int)((long long)r.rows * cluster / clusters);
    int seen = 0;                                              // rows from start on that are known to be no longer there to take
    for (;;) {
        Row w{r, sh, nullptr, kept, nullptr, nullptr, keys, before, rank, blocks, warp, lane, 0, 0, 0, -INFINITY, 1.f};
        int taken = -1;
        if (rank == 0)
            while (taken < 0 && seen < r.rows) {
                const int i = seen + (int)threadIdx.x, at = i < r.rows - start ? start + i : start + i - r.rows;
                const bool marked = i < r.rows && *(volatile int*)(r.token + at) == MARK;
                if (threadIdx.x == 0) sh.bin_found = 0xffffffffu;
                __syncthreads();
                if (marked) atomicMin(&sh.bin_found, (unsigned int)i);
                __syncthreads();
                const unsigned int first = sh.bin_found;
                if (first == 0xffffffffu) { seen += THREADS; __syncthreads(); continue; }
                if (i == (int)first) sh.above = (u64)(unsigned int)(atomicCAS(r.token + at, MARK, TAKEN) == MARK ? at : -1);
                __syncthreads();
                taken = (int)(unsigned int)sh.above;
            }
        // from the first block to all
        const int at = (int)(unsigned int)sh.slots[w.exchange((u64)(unsigned int)taken, 0)][0][0];
        if (at < 0) break;
        w.row = r.logits + at * r.row_stride;
        w.shift = (int)(((uintptr_t)w.row >> 2) & 3);
        w.quads = (r.vocab + w.shift + 3) / 4;
        w.t = temperature_of(r, at);
        double unused;
        unsigned int low = 0, high = ordered_key(w.fetch<false>(unused));
        w.row_ends(low, high);
        w.mx = of_key(high);
        if (w.mx == -INFINITY) { w.give_nothing(at); w.barrier(); } else { w.by_passes(at, Filters(r, at)); }
    }
}

// How a call is cut.
struct Cut {
    int resident, most, blocks;        // blocks at a time; blocks a row at most, and as many as it takes
    bool mark;                         // whether rows that need more passes are left to a second launch
    Cut(int rows, int vocab) : resident(2 * sm_count()), most(1) {
        // down to 4,096 ids a block, and as many blocks a row as are resident at a time with two an SM
        while (most < MAX_BLOCKS && vocab / most > 8192) most *= 2;
        blocks = most;
        while (blocks > 1 && (long long)rows * blocks > resident) blocks /= 2;
        // 64 rows by four blocks each take 31 to 59 us where the rows that need more passes stay with them and 40 to 91 where these are left to the second launch; 256
        // rows by one block each take 113 to 139 with it and 244 without
        mark = blocks < most && blocks < 4;
    }
};

}  // namespace

// The launches that a call of qt_sample_filtered makes.
extern "C" int qt_sample_filtered_launches(int rows, int vocab) { return rows > 0 ? (Cut(rows, vocab).mark ? 2 : 1) : 0; }

// logits [rows, vocab] float with rows `row_stride` elements apart; temperature, top_p, min_p, uniform float [rows], top_k int [rows]; token int [rows],
// logprob float [rows] or null.
extern "C" int qt_sample_filtered(const float* logits, long long row_stride, const float* temperature, const int* top_k, const float* top_p,
                                  const float* min_p, const float* uniform, int* token, float* logprob, int rows, int vocab, void* stream) {
    QT_REQUIRE(rows >= 0 && vocab > 0 && (rows <= 1 || row_stride >= vocab), "sample_filtered: bad sizes rows=%d vocab=%d stride=%lld",
               rows, vocab, row_stride);
    QT_REQUIRE(vocab <= MAX_VOCAB, "sample_filtered: a vocabulary of %d tokens is beyond the %d whose masses fit 64 bits", vocab, MAX_VOCAB);
    if (rows == 0) return QT_OK;
    QT_REQUIRE(rows <= 0x7fffffff / MAX_BLOCKS, "sample_filtered: %d rows are more than one launch takes", rows);
    const Cut of(rows, vocab);
    const int resident = of.resident, most = of.most;
    auto rows_of = [&](int blocks) {
        const int quads = (vocab + 3 + 3) / 4, turns = (quads + blocks * THREADS - 1) / (blocks * THREADS);
        const int span = TURNS * ((turns + TURNS * MAX_NOTES - 1) / (TURNS * MAX_NOTES));
        return Rows{logits, row_stride, temperature, top_k, top_p, min_p, uniform, token, logprob, rows, vocab, blocks, turns, span, 0, 0, mass_error(vocab, turns)};
    };
    auto part_of = [&](const Rows& r) { return (size_t)r.turns * THREADS * sizeof(float4); };
    constexpr size_t ONE = 219 * 1024, TWO = 106 * 1024;        // of an SM's shared memory for one block and for each of two, the static part taken off
    const int blocks = of.blocks;
    Rows r = rows_of(blocks);
    r.mark = of.mark;
    size_t smem = head_bytes(r);
    r.cached = !r.mark && smem + part_of(r) <= ((long long)rows * blocks > sm_count() ? TWO : ONE);
    if (r.cached) smem += part_of(r);
    const bool whole = blocks == 1 && vocab <= LIST;
    cudaError_t raised = whole ? raise_shared<sample_filtered_kernel<true>>((int)smem) : raise_shared<sample_filtered_kernel<false>>((int)smem);
    if (raised != cudaSuccess) QT_FAIL(QT_ERR_LAUNCH, "sample_filtered: cannot raise shared memory: %s", cudaGetErrorString(raised));
    launch_kernel_cluster(whole ? sample_filtered_kernel<true> : sample_filtered_kernel<false>, dim3((unsigned)(rows * blocks)), dim3(THREADS), smem, (cudaStream_t)stream,
                          (unsigned)blocks, r);
    if (r.mark) {
        const int clusters = resident / most < rows ? resident / most : rows;
        Rows marked = rows_of(most);
        smem = LIST * (sizeof(unsigned int) + sizeof(u64));
        marked.cached = smem + part_of(marked) <= ONE;
        if (marked.cached) smem += part_of(marked);
        raised = raise_shared<sample_marked_kernel>((int)smem);
        if (raised != cudaSuccess) QT_FAIL(QT_ERR_LAUNCH, "sample_filtered: cannot raise shared memory: %s", cudaGetErrorString(raised));
        launch_kernel_cluster(sample_marked_kernel, dim3((unsigned)(clusters * most)), dim3(THREADS), smem, (cudaStream_t)stream, (unsigned)most, marked);
    }
    QT_CHECK_LAUNCH("sample_filtered");
    return QT_OK;
}

QT_DEFINE_LAST_ERROR(sampling_filtered)
