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
// A row is shared by a cluster of up to eight blocks, each with a part of the ids in shared memory, so that it comes from memory once.  What survives the filters
// is a small head of the row as a rule, and is found without a look at the rest:
//
//   * the largest logit of every thread goes into 256 bins by its distance below the row's; where the bins' running count reaches top_k (or their
//     mass p times the row's mass) lies a bound that at least so many tokens reach, and seldom many more;
//   * the tokens above the bound go to the first block in vocabulary order (min_p gives a bound by itself); that block sorts their keys, finds the thresholds
//     on the running count and mass, and draws.
//
// Only the row's mass for top_p without top_k takes an exponential a token, an approximate one (its error, 2^-22, is that of a sum in float).  A row whose head
// does not fit the list finds its thresholds by bins of all of its tokens, each 256 times narrower than the one before, until what is in the bin of the threshold
// fits the list (three times; what is still alike then is bisected).  Such a row, and one without filters, draws over all blocks.
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
constexpr float BINS_PER_NAT = 8.f;
constexpr float LOG2E = 1.4426950408889634f;
typedef unsigned long long u64;

struct Rows {
    const float* logits; long long row_stride;
    const float* temperature; const int* top_k; const float* top_p; const float* min_p; const float* uniform;
    int* token; float* logprob;
    int vocab, blocks, turns, cached;  // blocks a row; turns of a warp over its ids, 128 a turn; whether they are kept in shared memory
};

// Floats as unsigned integers of the same order (no NaN comes here); the two zeros share a key.
__device__ __forceinline__ unsigned int ordered_key(float x) {
    unsigned int bits = __float_as_uint(x);
    if (bits == 0x80000000u) bits = 0u;
    return (bits & 0x80000000u) ? ~bits : (bits | 0x80000000u);
}
__device__ __forceinline__ float of_key(unsigned int key) { return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key); }

__device__ __forceinline__ float below(float x, float mx) { return x == mx ? 0.f : x - mx; }      // two equal infinities too
__device__ __forceinline__ float depth_of(float x, float mx, float t) { return below(x, mx) / t; }
__device__ __forceinline__ float weight_of(float x, float mx, float t) { return expf(below(x, mx) / t); }
// w in units of 2^-40, rounded to nearest even: two 20-bit steps, each exact in float.
__device__ __forceinline__ u64 units_of(float w) {
    const float high = w * 1048576.f;
    const unsigned int whole = (unsigned int)high;
    return ((u64)whole << 20) + __float2uint_rn((high - (float)whole) * 1048576.f);
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
// Inclusive prefix sums over the block of the numbers i = j THREADS + thread, of which there are n; returns the whole.
__device__ __forceinline__ u64 block_prefix(u64 (&v)[PER_THREAD], int n, u64* per_warp, int warp, int lane) {
    u64 base = 0;
#pragma unroll
    for (int j = 0; j < PER_THREAD; ++j) {
        if (j * THREADS >= n) break;
        const u64 upto = warp_prefix(v[j], lane);
        u64 all;
        const u64 before = warps_before(upto, per_warp, warp, lane, all);
        v[j] = base + before + upto;
        base += all;
    }
    return base;
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

// Of sorted keys of at least floor_key, the last in front of which less than `wanted` lies, what lies above all of them included; the first if there is none.
__device__ __forceinline__ int last_below(const u64 (&upto)[PER_THREAD], const u64 (&own)[PER_THREAD], const unsigned int* sorted, int n, unsigned int floor_key, u64 above,
                                          double wanted, u64* per_warp, int warp, int lane) {
    int last = 0;
#pragma unroll
    for (int j = 0; j < PER_THREAD; ++j) {
        const int i = j * THREADS + threadIdx.x;
        if (i < n && sorted[i] >= floor_key && (double)(above + upto[j] - own[j]) < wanted) last = i;
    }
    last = __reduce_max_sync(0xffffffffu, last);
    __syncthreads();
    if (lane == 0) per_warp[warp] = last;
    __syncthreads();
    return __reduce_max_sync(0xffffffffu, lane < WARPS ? (int)per_warp[lane] : 0);
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
__device__ __forceinline__ void add_to_bins(unsigned int (*bins)[BINS], int bin, bool by_mass, u64 m) {
    atomicAdd(&bins[0][bin], 1u);
    if (!by_mass) return;
    const unsigned int low = (unsigned int)m, before = atomicAdd(&bins[1][bin], low);
    const unsigned int high = (unsigned int)(m >> 32) + (before > 0xffffffffu - low ? 1u : 0u);
    if (high) atomicAdd(&bins[2][bin], high);
}

struct Row {
    const Rows& r;
    Shared& sh;
    const float* row;
    float4* kept;                                // this block's ids in shared memory
    unsigned int* keys;                          // the first block's: LIST of them, to be sorted
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
    static __device__ __forceinline__ float4 without_nan(float4 v) {
        v.x = isnan(v.x) ? -INFINITY : v.x; v.y = isnan(v.y) ? -INFINITY : v.y;
        v.z = isnan(v.z) ? -INFINITY : v.z; v.w = isnan(v.w) ? -INFINITY : v.w;
        return v;
    }
    // quad number q of this block, whichever thread has read it
    __device__ __forceinline__ float4 any_quad(int q) const { return r.cached ? kept[q] : without_nan(load_quad(rank * WARPS * r.turns * 32 + q)); }
    __device__ __forceinline__ float4 quad(int i) const { return r.cached ? kept[(warp * r.turns + i) * 32 + lane] : without_nan(load(i)); }
    // The loop stays a loop: with an exponential and a division for every number, a pass that is unrolled is tens of kilobytes of instructions that run once or
    // twice, and a block waits for those.
    template <typename F> __device__ __forceinline__ void each_turn(F f) const {
#pragma unroll 1
        for (int i = 0; i < r.turns; ++i) f(i, quad(i));
    }
    template <typename F> __device__ __forceinline__ void each(F f) const {
        each_turn([&](int, float4 v) { f(v.x); f(v.y); f(v.z); f(v.w); });
    }

    // the first read of the row: five turns' loads in flight, kept where they fit; this thread's largest
    __device__ __forceinline__ float fetch() const {
        float best = -INFINITY;
        for (int i0 = 0; i0 < r.turns; i0 += 5) {
            float4 v[5];
#pragma unroll
            for (int j = 0; j < 5; ++j) v[j] = i0 + j < r.turns ? load(i0 + j) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
#pragma unroll
            for (int j = 0; j < 5; ++j) {
                const float4 c = without_nan(v[j]);
                best = fmaxf(best, fmaxf(fmaxf(c.x, c.y), fmaxf(c.z, c.w)));
                if (r.cached && i0 + j < r.turns) kept[(warp * r.turns + i0 + j) * 32 + lane] = c;
            }
        }
        return best;
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

    __device__ __forceinline__ float depth(float x) const { return depth_of(x, mx, t); }
    __device__ __forceinline__ u64 mass(float x) const { return units_of(weight_of(x, mx, t)); }

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
                if (level == 0 || index >> 8 == prefix) add_to_bins(sh.bins[level & 1], index & (BINS - 1), by_mass, by_mass ? mass(x) : 0);
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
            each([&](float x) { if (inside(x)) remote_store(keys + remote_add(&sh.taken, 0), 0, ordered_key(x)); });
            barrier();
            found = 0;
            if (rank == 0) {
                sort_down(keys, tokens);
                u64 upto[PER_THREAD], own[PER_THREAD];
#pragma unroll
                for (int j = 0; j < PER_THREAD; ++j) {
                    const int i = j * THREADS + threadIdx.x;
                    upto[j] = own[j] = i >= tokens ? 0 : by_mass ? mass(of_key(keys[i])) : 1;
                }
                block_prefix(upto, tokens, sh.per_warp, warp, lane);
                found = keys[last_below(upto, own, keys, tokens, 0u, above, wanted, sh.per_warp, warp, lane)];
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

    // Draws among the tokens with a key of at least floor_key and a weight of at least `least`, over all blocks.
    __device__ void draw(int at, unsigned int floor_key, float least) {
        auto stays = [&](float x) -> u64 {
            if (ordered_key(x) < floor_key) return 0;
            const float w = weight_of(x, mx, t);
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
                give_answer(r, at, id + e, depth_of(e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w, mx, t), total);
            }
            running += all;
        }
    }
};

__global__ void __launch_bounds__(THREADS, 2) sample_filtered_kernel(const Rows r) {
    pdl_launch_dependents();
    if (r.blocks > 1) cluster_arrive_started();
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ Shared sh;
    // the first block's: tokens above the bound as (key, id), by block and in vocabulary order; behind them the blocks' parts of the row, where the keys are sorted later
    u64* list = reinterpret_cast<u64*>(smem);
    float4* kept = reinterpret_cast<float4*>(smem + LIST * sizeof(u64));
    const int blocks = r.blocks, rank = blockIdx.x % blocks, at = blockIdx.x / blocks, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_wait();
    const float* row = r.logits + at * r.row_stride;
    const int shift = (int)(((uintptr_t)row >> 2) & 3);
    Row w{r, sh, row, kept, reinterpret_cast<unsigned int*>(list), rank, blocks, warp, lane, shift, (r.vocab + shift + 3) / 4, 0, -INFINITY, r.temperature[at]};
    w.clear_bins(0);
    const float own_best = w.fetch();
    if (blocks > 1) cluster_wait_started();
    {
        unsigned int low = 0, high = ordered_key(own_best);
        w.row_ends(low, high);
        w.mx = of_key(high);
    }
    const float mx = w.mx, t = w.t;
    if (!(t > 0.f) || mx == -INFINITY) {                       // the lowest id of the largest logit
        unsigned int first = 0xffffffffu, unused = 0;
        for (int i = 0; i < r.turns; ++i) {
            const float4 v = w.quad(i);
            const unsigned int id = 4 * w.quad_at(i) - shift;
            if (first == 0xffffffffu) first = v.x == mx ? id : v.y == mx ? id + 1 : v.z == mx ? id + 2 : v.w == mx ? id + 3 : first;
        }
        w.row_ends(first, unused);
        if (rank == 0 && threadIdx.x == 0) {
            r.token[at] = mx == -INFINITY ? 0 : (int)first;
            if (r.logprob) r.logprob[at] = mx == -INFINITY ? -INFINITY : 0.f;
        }
        w.barrier();
        return;
    }
    const int k = r.top_k[at];
    const float p = r.top_p[at], m = r.min_p[at], least = m > 0.f ? fminf(m, 1.f) : 0.f;
    const bool by_count = k > 0 && k < r.vocab, by_mass = p < 1.f, by_weight = least > 0.f;
    if (!by_count && !by_mass && !by_weight) {
        w.draw(at, 0u, 0.f);
        w.barrier();
        return;
    }
    const float per_nat = LOG2E / t;
    const bool whole = blocks == 1 && r.vocab <= LIST;         // the list takes the row as it is
    bool fits = mx < INFINITY && per_nat < INFINITY && t < 1e30f;
    float bound = -INFINITY;
    double row_mass = 0.;                                      // for top_p alone, in units
    if (fits && !whole) {
        if (by_weight && !by_count) bound = mx + t * logf(least);
        if (by_count || by_mass) {
            const bool counting = by_count;
            if (own_best > -INFINITY) add_to_bins(sh.bins[0], min((int)(-w.depth(own_best) * BINS_PER_NAT), BINS - 1), !counting, counting ? 0 : w.mass(own_best));
            float sum = 0.f;
            if (!counting) {
                w.each([&](float x) {
                    float e;
                    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"((x - mx) * per_nat));
                    sum += e;
                });
                sum = warp_sum(sum);
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
        int n = 0;
        w.each([&](float x) { n += above(x); });
        n = __reduce_add_sync(0xffffffffu, n);
        __syncthreads();
        if (lane == 0) sh.per_warp[warp] = n;
        __syncthreads();
        int from = 0, mine = 0;
        for (int i = 0; i < WARPS; ++i) { if (i < warp) from += (int)sh.per_warp[i]; mine += (int)sh.per_warp[i]; }
        const int room = LIST / blocks;
        if (mine <= room && n > 0) {
            w.each_turn([&](int i, float4 v) {
                const bool hit[4] = {above(v.x), above(v.y), above(v.z), above(v.w)};
                const int own = hit[0] + hit[1] + hit[2] + hit[3];
                if (!__any_sync(0xffffffffu, own)) return;
                const int upto = (int)warp_prefix(own, lane);
                int slot = rank * room + from + upto - own;
                const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (hit[e]) {
                        const u64 entry = ((u64)ordered_key(x[e]) << 32) | (unsigned int)(4 * w.quad_at(i) - shift + e);
                        if (blocks > 1) remote_store(list + slot, 0, entry); else list[slot] = entry;
                        ++slot;
                    }
                from += __shfl_sync(0xffffffffu, upto, 31);
            });
        }
        const int slot = w.exchange(mine, 0);
        for (int b = 0; b < blocks; ++b) fits = fits && (int)sh.slots[slot][b][0] <= room;
        if (fits) {
            if (rank > 0) return;
            // the first block alone: places j THREADS + thread of the list a thread
            int count = 0;
            for (int b = 0; b < blocks; ++b) count += (int)sh.slots[slot][b][0];
            u64 entry[PER_THREAD] = {};
            unsigned int* keys = reinterpret_cast<unsigned int*>(kept);
#pragma unroll
            for (int j = 0; j < PER_THREAD; ++j) {
                int i = j * THREADS + threadIdx.x, b = 0;
                if (i >= count) break;
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
                        const int i = j * THREADS + threadIdx.x;
                        upto[j] = own[j] = i < count && keys[i] >= floor_key ? w.mass(of_key(keys[i])) : 0;
                    }
                    const u64 in_list = block_prefix(upto, count, sh.per_warp, warp, lane);
                    const double wanted = (double)p * (by_count || whole ? (double)in_list : row_mass);
                    // the likeliest token stays whatever p is
                    floor_key = max(floor_key, keys[last_below(upto, own, keys, count, floor_key, 0, wanted, sh.per_warp, warp, lane)]);
                }
            }
            u64 upto[PER_THREAD], own[PER_THREAD];
#pragma unroll
            for (int j = 0; j < PER_THREAD; ++j) {
                const unsigned int key = (unsigned int)(entry[j] >> 32);
                own[j] = 0;
                if (j * THREADS + threadIdx.x < count && key >= floor_key) {
                    const float weight = expf(w.depth(of_key(key)));
                    own[j] = weight < least ? 0 : units_of(weight);
                }
                upto[j] = own[j];
            }
            const u64 total = block_prefix(upto, count, sh.per_warp, warp, lane);
            const u64 target = target_of(total, r.uniform[at]);
#pragma unroll
            for (int j = 0; j < PER_THREAD; ++j)
                if (own[j] > 0 && upto[j] > target && upto[j] - own[j] <= target)
                    give_answer(r, at, (int)(unsigned int)entry[j], w.depth(of_key((unsigned int)(entry[j] >> 32))), total);
            return;
        }
    }
    unsigned int floor_key = 0;
    if (by_count) floor_key = w.threshold(false, (double)k, 0., 0u);
    if (by_mass) floor_key = p > 0.f ? w.threshold(true, 0., (double)p, floor_key) : ordered_key(mx);
    w.draw(at, floor_key, least);
    w.barrier();
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
    // so many blocks a row that two of them fit an SM, and more where rows are few, down to 4,096 ids a block
    int blocks = 1;
    while (blocks < MAX_BLOCKS && (vocab / blocks > 20480 || (vocab / blocks > 8192 && (long long)rows * blocks < sm_count()))) blocks *= 2;
    const int quads = (vocab + 3 + 3) / 4, turns = (quads + blocks * THREADS - 1) / (blocks * THREADS);
    size_t part = (size_t)turns * THREADS * sizeof(float4);
    const int cached = part <= 200 * 1024;                     // a longer part is read again
    if (!cached) part = 0;
    if (part < LIST * sizeof(unsigned int)) part = LIST * sizeof(unsigned int);
    const size_t smem = LIST * sizeof(u64) + part;
    const cudaError_t raised = raise_shared<sample_filtered_kernel>((int)smem);
    if (raised != cudaSuccess) QT_FAIL(QT_ERR_LAUNCH, "sample_filtered: cannot raise shared memory: %s", cudaGetErrorString(raised));
    const Rows r{logits, row_stride, temperature, top_k, top_p, min_p, uniform, token, logprob, vocab, blocks, turns, cached};
    launch_kernel_cluster(sample_filtered_kernel, dim3((unsigned)(rows * blocks)), dim3(THREADS), smem, (cudaStream_t)stream, (unsigned)blocks, r);
    QT_CHECK_LAUNCH("sample_filtered");
    return QT_OK;
}

QT_DEFINE_LAST_ERROR(sampling_filtered)
