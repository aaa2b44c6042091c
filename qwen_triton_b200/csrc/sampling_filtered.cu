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
//
// A row is shared by a cluster of up to eight blocks, so many that all rows' blocks are resident at once, and comes from memory once as a rule.  What survives the
// filters is a small head of the row, mostly, and is found in that one pass:
//
//   * every thread keeps its four largest logits; the largest of each go into 256 bins by their distance below the row's.  Where the bins' running count
//     reaches top_k (or their mass p times the row's mass) lies a bound that at least so many tokens reach, and seldom many more; min_p gives one by itself;
//   * the tokens above the bound go to the first block in vocabulary order: those that the threads have kept, or, where some thread's fourth is above the
//     bound too, by a second look at the row.  That block sorts their keys, finds the thresholds on the running count and mass, and draws.
//
// Only the row's mass for top_p without top_k takes an exponential a token, an approximate one (its error, 2^-22, is that of a sum in float).  A row whose head
// does not fit the list finds its thresholds by bins of all of its tokens, each 256 times narrower than the one before, until what is in the bin of the threshold
// fits the list (three times; what is still alike then is bisected).  Such a row, and one without filters, draws over all blocks; where many rows leave few blocks
// to each, these rows are left to a second launch with eight blocks a row.
//
// Measured behind a cold cache: one row of 151,936 MEASURED_1, 64 rows MEASURED_64, 256 rows (156 MB) MEASURED_256.
#include "common.cuh"

#include <math.h>

using namespace qt;

namespace {

constexpr int THREADS = 512;
constexpr int WARPS = THREADS / 32;
constexpr int MAX_BLOCKS = 8;
constexpr int BINS = 256;
constexpr int LIST = 2048;             // tokens that the first block takes; a block of b hands over LIST / b at most
constexpr int PER_THREAD = LIST / THREADS;
constexpr int KEPT = 4;                // logits a thread keeps
constexpr int IN_FLIGHT = 5;           // loads of 16 bytes a thread
constexpr float BINS_PER_NAT = 8.f;
constexpr float LOG2E = 1.4426950408889634f;
constexpr int UNSETTLED = -1;          // the mark, in the place of a token
typedef unsigned long long u64;

struct Rows {
    const float* logits; long long row_stride;
    const float* temperature; const int* top_k; const float* top_p; const float* min_p; const float* uniform;
    int* token; float* logprob;
    int rows, vocab, blocks, turns;    // blocks a row; turns of a warp over its ids, 128 a turn
    int pass;                          // 0: every row from beginning to end; 1: rows that a list does not settle are marked; 2: the marked rows
};

// Floats as unsigned integers of the same order (no NaN comes here); the two zeros share a key.
__device__ __forceinline__ unsigned int ordered_key(float x) {
    unsigned int bits = __float_as_uint(x);
    if (bits == 0x80000000u) bits = 0u;
    return (bits & 0x80000000u) ? ~bits : (bits | 0x80000000u);
}
__device__ __forceinline__ float of_key(unsigned int key) { return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key); }

__device__ __forceinline__ float below(float x, float mx) { return x == mx ? 0.f : x - mx; }      // two equal infinities too
// w in units of 2^-40, rounded to nearest even: two 20-bit steps, each exact in float.
__device__ __forceinline__ u64 units_of(float w) {
    const float high = w * 1048576.f;
    const unsigned int whole = (unsigned int)high;
    return ((u64)whole << 20) + __float2uint_rn((high - (float)whole) * 1048576.f);
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
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

__device__ __forceinline__ void remote_store(const u64* local, uint32_t rank, u64 value) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"((uint32_t)__cvta_generic_to_shared(local)), "r"(rank));
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(remote), "l"(value) : "memory");
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
    u64 list[LIST];                              // the first block's: tokens above the bound as (key, id), by block, in vocabulary order
    unsigned int keys[LIST];                     // and keys to be sorted
};

// Inclusive prefix sums of PER_THREAD numbers a thread over the block; returns the whole.
__device__ __forceinline__ u64 block_prefix(u64 (&v)[PER_THREAD], u64* per_warp, int warp, int lane) {
#pragma unroll
    for (int j = 1; j < PER_THREAD; ++j) v[j] += v[j - 1];
    const u64 own = v[PER_THREAD - 1], upto = warp_prefix(own, lane);
    __syncthreads();
    if (lane == 31) per_warp[warp] = upto;
    __syncthreads();
    u64 base = upto - own, all = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) { if (w < warp) base += per_warp[w]; all += per_warp[w]; }
#pragma unroll
    for (int j = 0; j < PER_THREAD; ++j) v[j] += base;
    return all;
}

// n <= LIST keys, largest first (bitonic, the next power of two filled up with zeros).
__device__ void sort_down(unsigned int* keys, int n) {
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

struct Row {
    const Rows& r;
    Shared& sh;
    const float* row;
    int rank, blocks, warp, lane, shift, quads, turn;
    float mx, t;

    // ids in fours from the 16-byte boundary at or before the row's start on; a place outside the row is -inf
    __device__ __forceinline__ int quad_at(int i) const { return ((rank * WARPS + warp) * r.turns + i) * 32 + lane; }
    __device__ __forceinline__ float4 load(int i) const {
        const int q = quad_at(i), id = 4 * q - shift;
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
    static __device__ __forceinline__ float4 without_nan(float4 v) {
        v.x = isnan(v.x) ? -INFINITY : v.x; v.y = isnan(v.y) ? -INFINITY : v.y;
        v.z = isnan(v.z) ? -INFINITY : v.z; v.w = isnan(v.w) ? -INFINITY : v.w;
        return v;
    }
    // f(turn, four logits) for the turns of this warp, the loads of several in flight
    template <bool RAW = false, typename F> __device__ __forceinline__ void each_turn(F f) const {
        for (int i0 = 0; i0 < r.turns; i0 += IN_FLIGHT) {
            float4 v[IN_FLIGHT];
#pragma unroll
            for (int j = 0; j < IN_FLIGHT; ++j) v[j] = i0 + j < r.turns ? load(i0 + j) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
#pragma unroll
            for (int j = 0; j < IN_FLIGHT; ++j)
                if (i0 + j < r.turns) f(i0 + j, RAW ? v[j] : without_nan(v[j]));
        }
    }
    template <typename F> __device__ __forceinline__ void each(F f) const {
        each_turn([&](int, float4 v) { f(v.x); f(v.y); f(v.z); f(v.w); });
    }

    // The pass over the row: this thread's largest logits with their ids (the lowest of equal ones first) and, with MASS, its sum of 2^((x - best[0]) per_nat).
    template <bool MASS>
    __device__ __forceinline__ float stream(float (&best)[KEPT], int (&id)[KEPT], float per_nat) const {
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < KEPT; ++e) { best[e] = -INFINITY; id[e] = 0; }
        auto take = [&](float x, int at) {
            if (x > best[KEPT - 1]) {
                best[KEPT - 1] = x; id[KEPT - 1] = at;
#pragma unroll
                for (int e = KEPT - 1; e > 0; --e)
                    if (best[e] > best[e - 1]) {
                        const float b = best[e]; best[e] = best[e - 1]; best[e - 1] = b;
                        const int i = id[e]; id[e] = id[e - 1]; id[e - 1] = i;
                    }
            }
        };
        each_turn<!MASS>([&](int i, float4 c) {               // NaN is above nothing
            const int at = 4 * quad_at(i) - shift;
            const float before = best[0];
            if (fmaxf(fmaxf(c.x, c.y), fmaxf(c.z, c.w)) > best[KEPT - 1]) { take(c.x, at); take(c.y, at + 1); take(c.z, at + 2); take(c.w, at + 3); }
            if (MASS && best[0] > -INFINITY) {
                if (best[0] > before) sum *= ex2((before - best[0]) * per_nat);
                sum += (ex2((c.x - best[0]) * per_nat) + ex2((c.y - best[0]) * per_nat)) + (ex2((c.z - best[0]) * per_nat) + ex2((c.w - best[0]) * per_nat));
            }
        });
        return sum;
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
    __device__ __forceinline__ u64 mass(float x) const { return units_of(expf(depth(x))); }

    __device__ __forceinline__ void clear_bins(int at) const {
        for (int i = threadIdx.x; i < 3 * BINS; i += THREADS) (&sh.bins[at][0][0])[i] = 0;
    }
    __device__ __forceinline__ void add_to_bin(int at, int bin, bool by_mass, u64 m) const {
        atomicAdd(&sh.bins[at][0][bin], 1u);
        if (!by_mass) return;
        const unsigned int low = (unsigned int)m, before = atomicAdd(&sh.bins[at][1][bin], low);
        const unsigned int high = (unsigned int)(m >> 32) + (before > 0xffffffffu - low ? 1u : 0u);
        if (high) atomicAdd(&sh.bins[at][2][bin], high);
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
        int prefix = 0, level = 0;
        float scale = BINS_PER_NAT / t;
        auto index_of = [&](float x) {
            const float at = -below(x, mx) * scale;
            const int index = at < 1073741824.f ? (int)at : 1073741824;
            return level == 0 ? min(index, BINS - 1) : index;
        };
        for (;; ++level, scale *= 256.f) {                    // a power of two: a place is that of the level before and eight bits more
            clear_bins(level & 1);
            __syncthreads();
            each([&](float x) {
                if (ordered_key(x) < floor_key) return;
                const int index = index_of(x);
                if (level == 0 || index >> 8 == prefix) add_to_bin(level & 1, index & (BINS - 1), by_mass, by_mass ? mass(x) : 0);
            });
            barrier();
            const int bin = find_bin(level & 1, by_mass, wanted, level == 0 ? share : 0., above);
            if (bin == BINS) { barrier(); return floor_key; } // all of them are less than is wanted
            prefix = (prefix << 8) + bin;
            // the last bin of the first level has no lower end
            if (sh.bin_tokens <= LIST || level == 2 || (level == 0 && bin == BINS - 1) || !(scale * 65536.f < INFINITY)) break;
        }
        auto inside = [&](float x) { return ordered_key(x) >= floor_key && index_of(x) == prefix; };
        unsigned int found;
        if (sh.bin_tokens <= LIST) {                          // the bin's keys to the first block, in any order: they are sorted there
            if (threadIdx.x == 0) sh.taken = 0;
            const int tokens = sh.bin_tokens;
            barrier();
            each([&](float x) { if (inside(x)) remote_store(sh.keys + remote_add(&sh.taken, 0), 0, ordered_key(x)); });
            barrier();
            found = 0;
            if (rank == 0) {
                sort_down(sh.keys, tokens);
                u64 upto[PER_THREAD], own[PER_THREAD];
#pragma unroll
                for (int j = 0; j < PER_THREAD; ++j) {
                    const int i = threadIdx.x * PER_THREAD + j;
                    upto[j] = own[j] = i >= tokens ? 0 : by_mass ? mass(of_key(sh.keys[i])) : 1;
                }
                block_prefix(upto, sh.per_warp, warp, lane);
                found = sh.keys[last_below(upto, own, sh.keys, tokens, 0u, above, wanted)];
            }
            const int slot = exchange(found, 0);
            found = (unsigned int)sh.slots[slot][0][0];
        } else {
            unsigned int low = 0xffffffffu, high = 0;
            each([&](float x) { if (inside(x)) { low = min(low, ordered_key(x)); high = max(high, ordered_key(x)); } });
            row_ends(low, high);
            while (low < high) {
                const unsigned int mid = low + (high - low) / 2;
                u64 n = 0;
                each([&](float x) { if (ordered_key(x) > mid && inside(x)) n += by_mass ? mass(x) : 1; });
                if ((double)(above + row_total(n)) < wanted) high = mid; else low = mid + 1;
            }
            found = low;
        }
        barrier();                                            // every block is done with the bins
        return max(found, floor_key);
    }

    // Of sorted keys of at least floor_key, the last in front of which less than `wanted` lies, what lies above all of them included; the first if there is none.
    __device__ __forceinline__ int last_below(const u64 (&upto)[PER_THREAD], const u64 (&own)[PER_THREAD], const unsigned int* sorted, int n, unsigned int floor_key, u64 above,
                                              double wanted) const {
        int last = 0;
#pragma unroll
        for (int j = 0; j < PER_THREAD; ++j) {
            const int i = threadIdx.x * PER_THREAD + j;
            if (i < n && sorted[i] >= floor_key && (double)(above + upto[j] - own[j]) < wanted) last = i;
        }
        last = __reduce_max_sync(0xffffffffu, last);
        if (lane == 0) sh.scratch[warp][0] = last;
        __syncthreads();
        return __reduce_max_sync(0xffffffffu, lane < WARPS ? (int)sh.scratch[lane][0] : 0);
    }

    __device__ __forceinline__ u64 target_of(u64 total, float uniform) const {
        const double wanted = floor((double)uniform * (double)total);
        const u64 target = wanted > 0. ? (u64)wanted : 0;
        return target < total ? target : total - 1;           // a number of 1 and more: the last token that stays
    }
    __device__ __forceinline__ void answer(int at, int token, float x, u64 total) const {
        r.token[at] = token;
        if (r.logprob) r.logprob[at] = depth(x) - logf((float)total * (1.f / 1099511627776.f));
    }

    // Draws among the tokens with a key of at least floor_key and a weight of at least `least`, over all blocks.
    __device__ void draw(int at, unsigned int floor_key, float least) {
        auto stays = [&](float x) -> u64 {
            if (ordered_key(x) < floor_key) return 0;
            const float w = expf(depth(x));
            return w < least ? 0 : units_of(w);
        };
        u64 mine = 0;
        each([&](float x) { mine += stays(x); });
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
        if (!(before <= target && target < before + mine)) return;
        u64 running = before;
        bool found = false;
        each_turn([&](int i, float4 v) {
            if (found) return;
            const u64 m[4] = {stays(v.x), stays(v.y), stays(v.z), stays(v.w)};
            const u64 own = m[0] + m[1] + m[2] + m[3], upto = running + warp_prefix(own, lane);
            const unsigned int beyond = __ballot_sync(0xffffffffu, upto > target);
            if (beyond && lane == __ffs(beyond) - 1) {
                u64 sum = upto - own;
                int e = 0;
                while (e < 3 && sum + m[e] <= target) sum += m[e++];
                answer(at, 4 * quad_at(i) - shift + e, e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w, total);
            }
            found = beyond != 0;
            running = __shfl_sync(0xffffffffu, upto, 31);
        });
    }
};

// A row from beginning to end, by all blocks of a cluster.
__device__ __forceinline__ void sample_row(const Rows& r, Shared& sh, int at, int rank, bool& started) {
    u64* list = sh.list;
    unsigned int* keys = sh.keys;
    const int blocks = r.blocks, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const float* row = r.logits + at * r.row_stride;
    const int shift = (int)(((uintptr_t)row >> 2) & 3);
    const float t = r.temperature[at], p = r.top_p[at], m = r.min_p[at], per_nat = LOG2E / t;
    const int k = r.top_k[at];
    const bool by_count = k > 0 && k < r.vocab, by_mass = p < 1.f, counting = by_count;
    Row w{r, sh, row, rank, blocks, warp, lane, shift, (r.vocab + shift + 3) / 4, 0, -INFINITY, t};
    w.clear_bins(0);
    float best[KEPT], sum;
    int id[KEPT];
    if (by_mass && !by_count && t > 0.f && per_nat < INFINITY) sum = w.stream<true>(best, id, per_nat);
    else sum = w.stream<false>(best, id, per_nat);
    if (blocks > 1 && !started) cluster_wait_started();
    started = true;
    {
        unsigned int low = 0, high = ordered_key(best[0]);
        w.row_ends(low, high);
        w.mx = of_key(high);
    }
    const float mx = w.mx;
    if (!(t > 0.f) || mx == -INFINITY) {                       // the lowest id of the largest logit
        unsigned int first = best[0] == mx ? id[0] : 0xffffffffu, unused = 0;
        w.row_ends(first, unused);
        if (rank == 0 && threadIdx.x == 0) {
            r.token[at] = mx == -INFINITY ? 0 : (int)first;
            if (r.logprob) r.logprob[at] = mx == -INFINITY ? -INFINITY : 0.f;
        }
        w.barrier();
        return;
    }
    const float least = m > 0.f ? fminf(m, 1.f) : 0.f;
    const bool by_weight = least > 0.f;
    if (!by_count && !by_mass && !by_weight) {
        if (r.pass == 1) { if (rank == 0 && threadIdx.x == 0) r.token[at] = UNSETTLED; return; }
        w.draw(at, 0u, 0.f);
        w.barrier();
        return;
    }
    const bool whole = blocks == 1 && r.vocab <= LIST;         // the list takes the row as it is
    bool fits = r.pass < 2 && mx < INFINITY && per_nat < INFINITY && t < 1e30f;
    float bound = -INFINITY;
    double row_mass = 0.;                                      // for top_p alone, in units
    if (fits && !whole) {
        if (by_weight && !by_count) bound = mx + t * logf(least);
        if (by_count || by_mass) {
            if (best[0] > -INFINITY) w.add_to_bin(0, min((int)(-w.depth(best[0]) * BINS_PER_NAT), BINS - 1), !counting, counting ? 0 : w.mass(best[0]));
            if (!counting) {
                sum = warp_sum(best[0] > -INFINITY ? sum * ex2((best[0] - mx) * per_nat) : 0.f);
                if (lane == 0) sh.scratch[warp][1] = __float_as_uint(sum);
                __syncthreads();
                sum = warp_sum(lane < WARPS ? __uint_as_float((unsigned int)sh.scratch[lane][1]) : 0.f);
            }
            const int slot = w.exchange(__float_as_uint(sum), 0);
            for (int b = 0; b < blocks; ++b) row_mass += (double)__uint_as_float((unsigned int)sh.slots[slot][b][0]);
            row_mass *= 1099511627776.;
            u64 above = 0;
            double wanted = counting ? (double)k : (double)p * row_mass;
            const int bin = w.find_bin(0, !counting, wanted, 0., above);
            // every token of the bins up to this one lies above the bound; the last bin has no end
            if (bin < BINS - 1) bound = fmaxf(bound, mx - t * (float)(bin + 1) * (1.f / BINS_PER_NAT));
        }
        bound -= 1e-5f * (fabsf(mx) + fabsf(mx - bound));      // what the bound's and the bins' roundings are
    }
    if (fits) {
        auto above = [&](float x) { return x > -INFINITY && !(x < bound); };
        // a thread whose last kept logit is above the bound may have more of them: the whole block looks again
        const bool again = __syncthreads_or(above(best[KEPT - 1])) != 0;
        int n = 0;
        if (again) {
            w.each([&](float x) { n += above(x); });
        } else {
#pragma unroll
            for (int e = 0; e < KEPT; ++e) n += above(best[e]);
        }
        n = __reduce_add_sync(0xffffffffu, n);
        if (lane == 0) sh.per_warp[warp] = n;
        __syncthreads();
        int from = 0, mine = 0;
        for (int i = 0; i < WARPS; ++i) { if (i < warp) from += (int)sh.per_warp[i]; mine += (int)sh.per_warp[i]; }
        const int room = LIST / blocks;
        auto give = [&](int place, float x, int number) {
            const u64 entry = ((u64)ordered_key(x) << 32) | (unsigned int)number;
            if (blocks > 1) remote_store(list + rank * room + place, 0, entry); else list[place] = entry;
        };
        if (mine <= room && n > 0 && again) {
            w.each_turn([&](int i, float4 v) {
                const bool hit[4] = {above(v.x), above(v.y), above(v.z), above(v.w)};
                const int own = hit[0] + hit[1] + hit[2] + hit[3];
                if (!__any_sync(0xffffffffu, own)) return;
                const int upto = (int)warp_prefix(own, lane);
                int place = from + upto - own;
                const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (hit[e]) give(place++, x[e], 4 * w.quad_at(i) - shift + e);
                from += __shfl_sync(0xffffffffu, upto, 31);
            });
        } else if (mine <= room && n > 0) {                    // a token's place: how many of its warp's have lower ids
            int place[KEPT] = {};
#pragma unroll
            for (int e = 0; e < KEPT; ++e)
                for (unsigned int who = __ballot_sync(0xffffffffu, above(best[e])); who; who &= who - 1) {
                    const int other = __shfl_sync(0xffffffffu, id[e], __ffs(who) - 1);
#pragma unroll
                    for (int f = 0; f < KEPT; ++f) place[f] += other < id[f];
                }
#pragma unroll
            for (int e = 0; e < KEPT; ++e)
                if (above(best[e])) give(from + place[e], best[e], id[e]);
        }
        const int slot = w.exchange(mine, 0);
        for (int b = 0; b < blocks; ++b) fits = fits && (int)sh.slots[slot][b][0] <= room;
        if (fits) {
            if (rank > 0) return;
            // the first block alone: PER_THREAD neighbours of the list a thread
            int count = 0;
            for (int b = 0; b < blocks; ++b) count += (int)sh.slots[slot][b][0];
            u64 entry[PER_THREAD];
#pragma unroll
            for (int j = 0; j < PER_THREAD; ++j) {
                int i = threadIdx.x * PER_THREAD + j, b = 0;
                entry[j] = 0;
                if (i >= count) continue;
                const int to = i;
                while (i >= (int)sh.slots[slot][b][0]) i -= (int)sh.slots[slot][b++][0];
                entry[j] = list[b * room + i];
                keys[to] = (unsigned int)(entry[j] >> 32);
            }
            unsigned int floor_key = 0;
            if (by_count || by_mass) {
                sort_down(keys, count);
                if (by_count && k <= count) floor_key = keys[k - 1];
                if (by_mass) {
                    u64 upto[PER_THREAD], own[PER_THREAD];
#pragma unroll
                    for (int j = 0; j < PER_THREAD; ++j) {
                        const int i = threadIdx.x * PER_THREAD + j;
                        upto[j] = own[j] = i < count && keys[i] >= floor_key ? w.mass(of_key(keys[i])) : 0;
                    }
                    const u64 in_list = block_prefix(upto, sh.per_warp, warp, lane);
                    const double wanted = (double)p * (by_count || whole ? (double)in_list : row_mass);
                    const int last = w.last_below(upto, own, keys, count, floor_key, 0, wanted);      // the likeliest token stays whatever p is
                    floor_key = max(floor_key, keys[last]);
                }
            }
            u64 upto[PER_THREAD], own[PER_THREAD];
#pragma unroll
            for (int j = 0; j < PER_THREAD; ++j) {
                const unsigned int key = (unsigned int)(entry[j] >> 32);
                own[j] = 0;
                if (threadIdx.x * PER_THREAD + j < count && key >= floor_key) {
                    const float weight = expf(w.depth(of_key(key)));
                    own[j] = weight < least ? 0 : units_of(weight);
                }
                upto[j] = own[j];
            }
            const u64 total = block_prefix(upto, sh.per_warp, warp, lane);
            const u64 target = w.target_of(total, r.uniform[at]);
#pragma unroll
            for (int j = 0; j < PER_THREAD; ++j)
                if (upto[j] > target && upto[j] - own[j] <= target) w.answer(at, (int)(unsigned int)entry[j], of_key((unsigned int)(entry[j] >> 32)), total);
            return;
        }
    }
    if (r.pass == 1) { if (rank == 0 && threadIdx.x == 0) r.token[at] = UNSETTLED; return; }
    unsigned int floor_key = 0;
    if (by_count) floor_key = w.threshold(false, (double)k, 0., 0u);
    if (by_mass) floor_key = p > 0.f ? w.threshold(true, 0., (double)p, floor_key) : ordered_key(mx);
    w.draw(at, floor_key, least);
    w.barrier();
}

__global__ void __launch_bounds__(THREADS, 2) sample_filtered_kernel(const Rows r) {
    pdl_launch_dependents();
    if (r.blocks > 1) cluster_arrive_started();
    __shared__ Shared sh;
    const int rank = blockIdx.x % r.blocks, clusters = gridDim.x / r.blocks;
    bool started = false;                                      // every block of the cluster runs
    pdl_wait();
    if (r.pass < 2) {
        sample_row(r, sh, blockIdx.x / r.blocks, rank, started);
    } else {
        for (int at = blockIdx.x / r.blocks; at < r.rows; at += clusters)
            if (r.token[at] == UNSETTLED) sample_row(r, sh, at, rank, started);
        if (r.blocks > 1 && !started) cluster_wait_started();
    }
}

}  // namespace

// logits [rows, vocab] float with rows `row_stride` elements apart; temperature, top_p, min_p, uniform float [rows], top_k int [rows]; token int [rows],
// logprob float [rows] or null.
extern "C" int qt_sample_filtered(const float* logits, long long row_stride, const float* temperature, const int* top_k, const float* top_p,
                                  const float* min_p, const float* uniform, int* token, float* logprob, int rows, int vocab, void* stream) {
    QT_REQUIRE(rows >= 0 && vocab > 0 && vocab <= 0x3fffffff && (rows <= 1 || row_stride >= vocab), "sample_filtered: bad sizes rows=%d vocab=%d stride=%lld",
               rows, vocab, row_stride);
    if (rows == 0) return QT_OK;
    QT_REQUIRE(rows <= 0x7fffffff / MAX_BLOCKS, "sample_filtered: %d rows are more than one launch takes", rows);
    const long long sms = sm_count();
    int blocks = 1;                                            // as many a row as are all resident at once, two an SM, down to 4,096 ids a block
    while (blocks < MAX_BLOCKS && (long long)rows * blocks * 2 <= 2 * sms && vocab / blocks > 8192) blocks *= 2;
    auto launch = [&](int clusters, int per_row, int pass) {
        const int quads = (vocab + 3 + 3) / 4, turns = (quads + per_row * THREADS - 1) / (per_row * THREADS);
        const Rows r{logits, row_stride, temperature, top_k, top_p, min_p, uniform, token, logprob, rows, vocab, per_row, turns, pass};
        launch_kernel_cluster(sample_filtered_kernel, dim3((unsigned)clusters * per_row), dim3(THREADS), 0, (cudaStream_t)stream, (unsigned)per_row, r);
    };
    if (vocab / blocks <= 20480) {
        launch(rows, blocks, 0);
    } else {
        launch(rows, blocks, 1);
        launch((int)(2 * sms / MAX_BLOCKS), MAX_BLOCKS, 2);
    }
    QT_CHECK_LAUNCH("sample_filtered");
    return QT_OK;
}

QT_DEFINE_LAST_ERROR(sampling_filtered)
