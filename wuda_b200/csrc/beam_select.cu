// Beam selection: log-softmax over the vocabulary, cumulative scores, the k best continuations of a group's beams.
//
//   value[w, v] = score[w] + logit[w, v] - lse[w],   lse[w] = m + log sum_u exp(logit[w, u] - m)
//
// Within a beam the order of the values is that of the logits, so a beam's candidates are its k largest logits (ties to the lower
// token): keys of (order-preserving logit, ~token) are unique, and the largest key is the first candidate.  Only candidates of
// different beams are compared by value, in 64 bits.
//
// One launch.  A row of logits is cut into chunks, a CTA each, that are read once: 16 bytes per load, four loads per thread ahead of the
// four that it works on.  Every thread keeps a reference r and the sum of exp(x - r) of its elements; r follows the maximum only where a
// term would pass e^40, so a rescaling is rare and no term overflows.  x - r is formed before the product with log2 e: a
// logit equal to r counts exactly 1, a row of one token has log-probability 0, and logits of any magnitude will do.  Which element a
// thread gets depends on the element's number alone, not on the row's alignment, so equal rows have equal sums.
//
// Candidates: the k-th largest of 64 (k <= 32) or 128 maxima over disjoint parts of the tiles so far is a lower bound of the chunk's
// k-th largest logit, raised in front of the tiles 0, 2, 8, 26, .. (k > 32: 0, 1, 3, 7, ..); what a thread has of a tile in which it
// sees a logit beyond the bound is noted (a handful per tile) and looked at in the end, with the last bound.  No barrier besides.  A
// list that overflowed (sorted rows, rows of one value) is made again by exact selections.
//
// Rows that do not lie on 16 bytes: the aligned 16 bytes in which a vector begins are loaded as they are, and put together with the next
// lane's when the tile is worked on, so that the loads stay in flight (the shift at the loads themselves would wait for them).
//
// The CTA that completes a group's counter merges its lists the same way: the k-th largest of the maxima over 64 or 128 shares of the
// lists' first candidates bounds what can be among the k best, and the few that pass are ranked by counting.
//
// What bounds it (per launch in a graph, against a copy's 6.54 TB/s; plain calls one after the other take 0.4 to 1.3 us more): small calls
// the chain of launch, a chunk's loads, its fence and counter, and the merge's three round trips to L2 - 4 rows x 32000 bf16 8.2 us, of
// which the merge is 4.  Large ones the stream and what goes on beside it: 512 rows x 131072 bf16 (134 MB) 32.3 us with k = 8 and 34.3 with
// 16, 20.5 at the copy's rate.  Loads in this pattern alone take 22 us, the exponentials 2 on top, raising the bounds and notes 2 each,
// the merge 4.  256 rows x 131072 fp32, half the elements for the same bytes: 30.6.  The bf16 rows off 16 bytes: 39.2.
// More warps were worth more than anything else: a ring of bulk copies in shared memory left room for 5 or 6 CTAs per SM instead of 7
// (49-54 us instead of 40 at the time), and exponentials by polynomials for a part of the elements took more slots than they freed (42-47).
// Asking L2 for the tiles after the next one made it slower (35.4 to 38.5 us for two to eight tiles ahead, against 35.0 at the time).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cfloat>
#include <climits>
#include <type_traits>

#include "host.h"

namespace wuda {
namespace beams {

constexpr int kVectors = 4;                 // 16-byte loads per thread and tile
constexpr int kMostK = 64, kMostWidth = 32, kMostGroups = 256;
constexpr int kList = 1024;                 // candidates that a chunk's CTA holds
constexpr int kNotesOfBlock = 160, kNotesAllOfBlock = 1024; // notes of a CTA's warps with their contents, and without
constexpr int kEntries = 2048;              // candidates of all chunks of a group
constexpr int kMostChunks = 64;
constexpr int kMostLists = 256;             // of a group
constexpr int kFew = 512;                   // values that are ranked side by side
constexpr int kSms = 148;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kGrow = 40.f;               // e^40 * 2^24 elements are far from the largest fp32

using Key = unsigned long long;             // (ordered logit, ~token): unique, larger is better; 0 is none

struct Partial {
    double sum;                             // of exp(x - ref) over a chunk
    float ref;
    float unused;
};

struct Params {
    wuda_beam_select_args a;
    Key* lists;                             // [groups * width, chunks, k] in descending order, 0 behind them
    Partial* partials;                      // [groups * width, chunks]
    int chunks, chunk_vectors;              // vectors of 16 bytes per chunk, a multiple of the block's threads
};

template <typename T>
struct Type;
template <>
struct Type<float> {
    static constexpr int kVec = 4;
    static constexpr uint32_t kMasked = 0xff800000u;
};
template <>
struct Type<__half> {
    static constexpr int kVec = 8;
    static constexpr uint32_t kMasked = 0xfc00fc00u;
    using Pair = __half2;
};
template <>
struct Type<__nv_bfloat16> {
    static constexpr int kVec = 8;
    static constexpr uint32_t kMasked = 0xff80ff80u;
    using Pair = __nv_bfloat162;
};

// a word that grows with x (no NaN); 0 is below every number
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x);
    return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u); }
__device__ __forceinline__ Key key_of(float x, uint32_t token) { return (static_cast<Key>(ordered(x + 0.f)) << 32) | ~token; }      // (-0 counts as 0)
__device__ __forceinline__ uint32_t token_of(Key k) { return ~static_cast<uint32_t>(k); }

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 c;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(c.x), "=f"(c.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return c;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 c;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(c.x), "=f"(c.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return c;
}

// ---- a vector: 16 bytes of a row as four words, through L2: the kernel starts while the one that writes the logits runs, and a line
// in its SM's L1 may be older than them
__device__ __forceinline__ uint4 load16(const void* p) {
    uint4 v;
    asm volatile("ld.global.cg.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// Elements [at, at + kVec) of a row one by one, masked where they are not in [0, vocab).
template <typename T>
__device__ __noinline__ uint4 load_elements(const T* row, int at, int vocab) {
    uint32_t w[4] = {Type<T>::kMasked, Type<T>::kMasked, Type<T>::kMasked, Type<T>::kMasked};
#pragma unroll
    for (int i = 0; i < Type<T>::kVec; ++i) {
        if (at + i < 0 || at + i >= vocab) continue;
        if constexpr (sizeof(T) == 4) {
            w[i] = __ldcg(reinterpret_cast<const uint32_t*>(row) + at + i);
        } else {
            const uint32_t x = __ldcg(reinterpret_cast<const uint16_t*>(row) + at + i);
            w[i / 2] = i & 1 ? (w[i / 2] & 0xffffu) | (x << 16) : (w[i / 2] & 0xffff0000u) | x;
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
// The same sixteen bytes at a time, where row + at lies on 16 bytes (ALIGNED) or from the two such pieces that it lies in.
template <typename T, bool ALIGNED>
__device__ __forceinline__ uint4 load_vector(const T* row, int at, int vocab) {
    constexpr int kVec = Type<T>::kVec;
    if (at >= vocab) return make_uint4(Type<T>::kMasked, Type<T>::kMasked, Type<T>::kMasked, Type<T>::kMasked);
    const int off = ALIGNED ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(row + at) & 15), low = at - off / static_cast<int>(sizeof(T));
    if (off == 0 && at >= 0 && at + kVec <= vocab) return load16(row + at);
    if (off == 0 || low < 0 || low + 2 * kVec > vocab) return load_elements(row, at, vocab);
    const uint4 a = load16(row + low), b = load16(row + low + kVec);
    uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    if (off & 8) {
#pragma unroll
        for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
    }
    if (off & 4) {
#pragma unroll
        for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
    }
    const int bits = (off & 3) * 8;
    return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits), __funnelshift_r(w[2], w[3], bits),
                      __funnelshift_r(w[3], w[4], bits));
}

// NaN -> -inf in all elements of a word, and a word's elements as fp32
template <typename T>
__device__ __forceinline__ uint32_t without_nan(uint32_t w) {
    if constexpr (sizeof(T) == 4) {
        return __float_as_uint(fmaxf(__uint_as_float(w), -INFINITY));
    } else {
        using Pair = typename Type<T>::Pair;
        const uint32_t masked = Type<T>::kMasked;
        const Pair m = __hmax2(*reinterpret_cast<const Pair*>(&w), *reinterpret_cast<const Pair*>(&masked));
        return *reinterpret_cast<const uint32_t*>(&m);
    }
}
template <typename T>
__device__ __forceinline__ uint32_t max_words(uint32_t a, uint32_t b) {
    if constexpr (sizeof(T) == 4) {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    } else {
        using Pair = typename Type<T>::Pair;
        const Pair m = __hmax2(*reinterpret_cast<const Pair*>(&a), *reinterpret_cast<const Pair*>(&b));
        return *reinterpret_cast<const uint32_t*>(&m);
    }
}
template <typename T>
__device__ __forceinline__ float2 pair_of(uint32_t w) {       // of a 16-bit type
    if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(w), -INFINITY);
    else if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&w));
    else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
// a word that grows with the value; 0 is below every number
__device__ __forceinline__ Key ordered(double x) {
    const long long b = __double_as_longlong(x + 0.);      // (-0 counts as 0)
    return static_cast<Key>(b) ^ (static_cast<Key>(b >> 63) | (1ull << 63));
}
__device__ __forceinline__ double unordered(Key u) { return __longlong_as_double(u & (1ull << 63) ? u ^ (1ull << 63) : ~u); }

// The work of a CTA of kThreads threads
template <int kThreads>
struct Block {
static constexpr int kWarps = kThreads / 32, kNotes = kNotesOfBlock / kWarps, kNotesAll = kNotesAllOfBlock / kWarps;
// Candidates that are ranked side by side, a few per thread; beyond that the list is trimmed first.  It holds no more than kList.
static constexpr int kRanked = 3 * kThreads < kList ? 3 * kThreads : kList;

struct Shared {
    int count;                              // candidates (those beyond kList are lost)
    bool lost;                              // more was to be noted than there are places for
    alignas(16) uint32_t bound[kWarps];     // the least is the k-th largest logit so far, or less, as an ordered word
    uint32_t highest;                       // ... and the largest
    int hits[3];
    float warp_ref[kWarps];
    double warp_sum[kWarps];
    bool last;
    union {
        struct {                            // a chunk
            alignas(16) Key list[kList];
            alignas(16) uint4 note[kWarps][kNotes][kVectors];      // what a thread had of a tile in which a logit passed the bound
            alignas(16) uint32_t part_max[128];        // maxima of parts of the tiles, as ordered words
            int noted[kWarps][kNotesAll];              // ... whose: tile * 32 + lane
            float noted_top[kWarps][kNotesAll];        // ... and the largest logit of it
        };
        struct {                            // a group's lists
            Key entry[kEntries];
            alignas(16) Key value[kFew];               // what may be among the k best
            alignas(16) uint32_t front[128];           // largest values of shares of the entries, as ordered words
            alignas(16) Key tie[kFew];                 // ... and what decides between equal ones
            double sum[kMostLists], lse[kMostWidth], score[kMostWidth];
            float ref[kMostLists];
            int kind[kMostWidth];                      // 0 live, 1 finished, 2 dead
            uint32_t low[kMostWidth];
            int survivors, there;
        };
    };
};

// How many of n keys are larger, two at a time.
static __device__ __forceinline__ int larger_than(Key mine, const Key* keys, int n) {
    int rank = 0, i = 0;
#pragma unroll 4
    for (; i + 1 < n; i += 2) {
        const ulonglong2 other = *reinterpret_cast<const ulonglong2*>(keys + i);
        rank += (other.x > mine) + (other.y > mine);
    }
    if (i < n) rank += keys[i] > mine;
    return rank;
}

// Sum over the block, in turn `turn` of a sequence: three counters in rotation need one barrier per turn.
static __device__ __forceinline__ int block_total(int mine, int* hits, int turn) {
    const int n = __reduce_add_sync(0xffffffffu, mine);
    if ((threadIdx.x & 31) == 0 && n) atomicAdd(&hits[turn % 3], n);
    if (threadIdx.x == 0) hits[(turn + 1) % 3] = 0;
    __syncthreads();
    return hits[turn % 3];
}
static __device__ __forceinline__ void start_totals(int* hits) {
    __syncthreads();
    if (threadIdx.x < 3) hits[threadIdx.x] = 0;
    __syncthreads();
}

// The largest K such that at least `want` of the block's keys are at or above it, bit by bit; low <= K <= high is known (0 and ~0 where
// nothing is; low counts where they are fewer than `want`).  each(f) calls f(key) for every key of the thread.  All threads.
template <typename Each>
static __device__ __forceinline__ Key kth_largest(int want, Key low, Key high, int* hits, const Each& each) {
    start_totals(hits);
    int bit = 63 - __clzll(low ^ high);      // (-1: they are equal)
    Key least = bit < 63 ? low & ~((2ull << bit) - 1) : 0;
    for (int turn = 0; bit >= 0; --bit, ++turn) {
        const Key probe = least | (1ull << bit);
        int mine = 0;
        each([&](Key key) { mine += key >= probe; });
        const int total = block_total(mine, hits, turn);
        if (total >= want) least = probe;
        if (total == want) break;
    }
    return least;
}

// The k largest of the list and of the tile's keys (unique ones, 0 none) become the list, or all of them where they are fewer.  Returns
// the k-th.  All threads; ends behind a barrier.
template <int N>
static __device__ __forceinline__ Key select_exactly(Shared& sh, const Key (&tile)[N], int k) {
    Key held[kList / kThreads];
    const int count = min(sh.count, kList);
#pragma unroll
    for (int i = 0; i < kList / kThreads; ++i) held[i] = i * kThreads + threadIdx.x < count ? sh.list[i * kThreads + threadIdx.x] : 0;
    const auto each = [&](const auto& f) {
#pragma unroll
        for (int i = 0; i < kList / kThreads; ++i) f(held[i]);
#pragma unroll
        for (int i = 0; i < N; ++i) f(tile[i]);
    };
    const Key least = kth_largest(k, 0, ~0ull, sh.hits, each);
    __syncthreads();
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    each([&](Key key) {
        if (key != 0 && key >= least) sh.list[atomicAdd(&sh.count, 1)] = key;      // (k of them at most)
    });
    __syncthreads();
    return least;
}
static __device__ __noinline__ void trim_list(Shared& sh, int k) {
    const Key none[1] = {0};
    select_exactly(sh, none, k);
}

// A chunk's k largest keys where the list overflowed (rows sorted upwards, rows of one value, rows masked but for their end): tile by tile with
// exact selections, as far as a tile has a key above the k-th largest so far.
template <typename T>
static __device__ __noinline__ void candidates_exactly(Shared& sh, const T* row, int c0, int end, int vocab, int k) {
    constexpr int kVec = Type<T>::kVec;
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    Key least = 0;
    for (int at = c0; at < end; at += kThreads * kVec) {
        const int first = at + threadIdx.x * kVec;
        const uint4 v = load_elements(row, first, vocab);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        Key keys[kVec];
        bool above = false;
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
            const float2 f = pair_of<T>(w[e * 4 / kVec]);
            const float x = sizeof(T) == 2 && (e & 1) ? f.y : f.x;
            keys[e] = fabsf(x) < INFINITY ? key_of(x, static_cast<uint32_t>(first + e)) : 0;
            above = above || keys[e] > least;
        }
        if (__syncthreads_or(above)) {
            const Key now = select_exactly(sh, keys, k);
            if (sh.count == k) least = now;
            __syncthreads();
        }
    }
}

// The k-th largest of 64 (k <= 32) or 128 words: the least of those with fewer than k larger ones.  Each word is looked at by `by`
// neighbouring threads, which count a share of the others; every warp's least goes to `kth`, the largest of all to *first.  All
// threads, between two barriers of the caller's; then least_of(kth).
static __device__ __forceinline__ void kth_part(const uint32_t* parts, int k, uint32_t* kth, uint32_t* first) {
    const int tid = threadIdx.x, count = k <= 32 ? 64 : 128, by = kThreads / count, n = count / 4 / by;
    const uint32_t part = parts[tid / by];
    const uint4* share = reinterpret_cast<const uint4*>(parts) + tid % by * n;
    int larger = 0;
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
        const uint4 other = share[i];
        larger += (other.x > part) + (other.y > part) + (other.z > part) + (other.w > part);
    }
#pragma unroll
    for (int o = 1; o < kThreads / 64; o <<= 1)
        if (o < by) larger += __shfl_xor_sync(0xffffffffu, larger, o);
    if (larger == 0) *first = part;      // (equal ones write the same)
    const uint32_t least = __reduce_min_sync(0xffffffffu, larger < k ? part : 0xffffffffu);
    if ((tid & 31) == 0) kth[tid >> 5] = least;
}
static __device__ __forceinline__ uint32_t least_of(const uint32_t* kth) {
    if constexpr (kWarps > 4) return __reduce_min_sync(0xffffffffu, kth[threadIdx.x % kWarps]);
    const uint4 least = *reinterpret_cast<const uint4*>(kth);
    return min(min(least.x, least.y), min(least.z, least.w));
}

// The k-th largest of maxima over all that some threads each have seen: k logits so far are at or above it.
static __device__ __forceinline__ float raise_bound(Shared& sh, float so_far, int k, float bound, bool* raised) {
    atomicMax(&sh.part_max[threadIdx.x % (k <= 32 ? 64 : 128)], ordered(so_far));      // (what was there is of earlier tiles)
    __syncthreads();
    kth_part(sh.part_max, k, sh.bound, &sh.highest);
    __syncthreads();
    const float now = unordered(least_of(sh.bound));
    *raised = now > bound;
    return now;
}

// A chunk of a row: its partial sum, and its k largest keys in descending order.
template <typename T, bool ALIGNED>
static __device__ __forceinline__ void chunk(Shared& sh, const Params& p, const T* row, int row_number, int number) {
    constexpr int kVec = Type<T>::kVec;
    const wuda_beam_select_args& a = p.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, k = a.k;
    const int c0 = number * p.chunk_vectors * kVec, end = min(a.vocab, c0 + p.chunk_vectors * kVec);
    constexpr int kTile = kThreads * kVectors * kVec;
    const int tiles = (end - c0 + kTile - 1) / kTile, whole = (end - c0) / kTile;
    // A row's last, partial tile is spread over the threads, a vector each first, so that there are maxima of many parts of it.  In a
    // whole tile a warp's part is contiguous, vector after vector.  Where the row does not lie on 16 bytes, what is loaded are the aligned
    // 16 bytes in which a vector begins; its end is in the next lane's (for the last lane: in lane 0's next, and one more load of lane 0's).
    const int off = ALIGNED ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(row) & 15), back = off / static_cast<int>(sizeof(T));
    const auto element_of = [&](int tile, int u, int of_lane) {
        const int at = tile < whole ? (warp * kVectors + u) * 32 : u * kThreads + warp * 32;
        return c0 + (tile * kThreads * kVectors + at + of_lane) * kVec;
    };
    uint4 next[kVectors + !ALIGNED];
    const auto fetch = [&](int tile) {
        if (tile >= whole) {
#pragma unroll
            for (int u = 0; u < kVectors; ++u) next[u] = load_vector<T, ALIGNED>(row, element_of(tile, u, lane), a.vocab);
            return;
        }
        const int at = element_of(tile, 0, lane) - back;
        if (ALIGNED || (at - lane * kVec >= 0 && at + (kVectors * 32 + 1 - lane) * kVec <= a.vocab)) {      // (of the whole warp)
#pragma unroll
            for (int u = 0; u < kVectors; ++u) next[u] = load16(row + at + u * 32 * kVec);
            if constexpr (!ALIGNED) {
                if (lane == 0) next[kVectors] = load16(row + at + kVectors * 32 * kVec);
            }
        } else if constexpr (!ALIGNED) {      // the row's first bytes or last ones
#pragma unroll
            for (int u = 0; u < kVectors; ++u) next[u] = load_vector<T, true>(row, at + u * 32 * kVec, a.vocab);
            if (lane == 0) next[kVectors] = load_vector<T, true>(row, at + kVectors * 32 * kVec, a.vocab);
        }
    };
    // the words of a thread's vectors from what was loaded: SKIP whole words and off % 4 bytes of each are left out
    const auto shifted = [&](uint32_t (&w)[4 * kVectors], auto skip) {
        constexpr int SKIP = decltype(skip)::value;
        const int bits = (off & 3) * 8;
#pragma unroll
        for (int u = 0; u < kVectors; ++u) {
            const uint4 now = next[u], then = next[kVectors + !ALIGNED - 1 < u + 1 ? u : u + 1];
            uint32_t x[8] = {now.x, now.y, now.z, now.w};
            const uint32_t give[4] = {lane ? now.x : then.x, lane ? now.y : then.y, lane ? now.z : then.z, lane ? now.w : then.w};
#pragma unroll
            for (int i = 0; i <= SKIP; ++i) x[4 + i] = __shfl_sync(0xffffffffu, give[i], lane + 1);      // (of lane 0 for lane 31)
#pragma unroll
            for (int i = 0; i < 4; ++i) w[4 * u + i] = __funnelshift_r(x[SKIP + i], x[SKIP + i + 1], bits);
        }
    };
    if (a.finished && __ldcg(a.finished + row_number)) return;
    fetch(0);      // on its way while the score is
    if (!(fabsf(__ldcg(a.scores + row_number)) < INFINITY)) return;
    if (tid == 0) {
        sh.count = 0;
        sh.lost = false;
    }
    if (tid < 128) sh.part_max[tid] = ordered(-INFINITY);
    __syncthreads();
    float ref = -FLT_MAX, so_far = -INFINITY, bound = -INFINITY;
    float2 sum[2] = {{0.f, 0.f}, {0.f, 0.f}};
    int noted = 0;        // of the warp's vectors
    int refresh = 0;      // the next tile in front of which the bound is raised: 0, 2, 8, 26, .. or 0, 1, 3, 7, ..
    for (int tile = 0; tile < tiles; ++tile) {
        uint32_t w[4 * kVectors];
        if (ALIGNED || off == 0 || tile >= whole) {
#pragma unroll
            for (int u = 0; u < kVectors; ++u) w[4 * u] = next[u].x, w[4 * u + 1] = next[u].y, w[4 * u + 2] = next[u].z, w[4 * u + 3] = next[u].w;
        } else if constexpr (!ALIGNED) {
            switch (off >> 2) {      // (the same for the whole row)
                case 0: shifted(w, std::integral_constant<int, 0>()); break;
                case 1: shifted(w, std::integral_constant<int, 1>()); break;
                case 2: shifted(w, std::integral_constant<int, 2>()); break;
                default: shifted(w, std::integral_constant<int, 3>());
            }
        }
#pragma unroll
        for (int i = 0; i < 4 * kVectors; ++i) w[i] = without_nan<T>(w[i]);      // masked tokens are -inf from here on
        if (tile + 1 < tiles) fetch(tile + 1);
        // ---- the maximum
        const auto maximum = [&] {
            uint32_t m = w[0];
#pragma unroll
            for (int i = 1; i < 4 * kVectors; ++i) m = max_words<T>(m, w[i]);
            const float2 f = pair_of<T>(m);
            return fmaxf(f.x, f.y);
        };
        float top = maximum();
        if (top == INFINITY) {
#pragma unroll
            for (int i = 0; i < 4 * kVectors; ++i) {
                const float2 f = pair_of<T>(w[i]);
                if constexpr (sizeof(T) == 4) {
                    if (f.x == INFINITY) w[i] = Type<T>::kMasked;
                } else {
                    if (f.x == INFINITY) w[i] = (w[i] & 0xffff0000u) | (Type<T>::kMasked & 0xffffu);
                    if (f.y == INFINITY) w[i] = (w[i] & 0xffffu) | (Type<T>::kMasked & 0xffff0000u);
                }
            }
            top = maximum();
        }
        // ---- sum of exp(x - ref)
        if (top - ref > kGrow) {
            const float f = exp2_approx((ref - top) * kLog2e);
            ref = top;
#pragma unroll
            for (int i = 0; i < 2; ++i) sum[i] = make_float2(sum[i].x * f, sum[i].y * f);
        }
        const float2 minus = {-ref, -ref}, scale = {kLog2e, kLog2e};
#pragma unroll
        for (int i = 0; i < 4 * kVectors; i += sizeof(T) == 4 ? 2 : 1) {
            float2 x;
            if constexpr (sizeof(T) == 4) x = make_float2(__uint_as_float(w[i]), __uint_as_float(w[i + 1]));
            else x = pair_of<T>(w[i]);
            const float2 y = mul2(add2(x, minus), scale);
            const int to = sizeof(T) == 4 ? i / 2 & 1 : i & 1;
            sum[to] = add2(sum[to], make_float2(exp2_approx(y.x), exp2_approx(y.y)));
        }
        // ---- candidates
        so_far = fmaxf(so_far, top);
        bool with_equal = false;      // a logit equal to the bound is a candidate where the bound is this tile's
        if (tile == refresh) {
            refresh = k <= 32 ? 3 * refresh + 2 : 2 * refresh + 1;
            bound = raise_bound(sh, so_far, k, bound, &with_equal);
        }
        const bool hit = with_equal ? top >= bound : top > bound;
        const uint32_t hits = __ballot_sync(0xffffffffu, hit);
        if (hits) {      // places without atomics: each warp has a list of its own
            const int at = noted + __popc(hits & ((1u << lane) - 1));
            if (hit && at < kNotesAll) sh.noted[warp][at] = tile * 32 + lane, sh.noted_top[warp][at] = top;
            if (hit && at < kNotes) {
#pragma unroll
                for (int u = 0; u < kVectors; ++u) sh.note[warp][at][u] = make_uint4(w[4 * u], w[4 * u + 1], w[4 * u + 2], w[4 * u + 3]);
            }
            noted += __popc(hits);
        }
    }

    // ---- candidates: the noted elements that pass the last bound
    bool raised;
    if ((k <= 32 ? 3 * (tiles - 1) + 2 : 2 * (tiles - 1) + 1) != refresh) bound = raise_bound(sh, so_far, k, bound, &raised);
    else __syncthreads();      // (it was raised with the last tile)
    if (noted > kNotesAll) sh.lost = true;
    __syncwarp();
    int kept = 0;         // the notes that do, to the front of the list
    for (int i = 0; i < min(noted, kNotesAll); i += 32) {
        const bool keep = i + lane < min(noted, kNotesAll) && sh.noted_top[warp][i + lane] >= bound;
        const int of = keep ? sh.noted[warp][i + lane] : 0;
        const uint32_t keeps = __ballot_sync(0xffffffffu, keep);
        if (keep) sh.noted[warp][kept + __popc(keeps & ((1u << lane) - 1))] = of | (i + lane < kNotes ? (i + lane + 1) << 24 : 0);
        kept += __popc(keeps);
    }
    __syncwarp();
    for (int i = lane; i < kept * kVectors; i += 32) {
        const int u = i % kVectors, of = sh.noted[warp][i / kVectors], note = (of >> 24) - 1, from = of & 0xffffff;
        const int first = element_of(from / 32, u, from % 32);
        const uint4 v = note >= 0 ? sh.note[warp][note][u] : load_vector<T, ALIGNED>(row, first, a.vocab);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
            const float2 f = pair_of<T>(w[e * 4 / kVec]);
            const float x = sizeof(T) == 2 && (e & 1) ? f.y : f.x;
            if (x >= bound && fabsf(x) < INFINITY) {
                const int at = atomicAdd(&sh.count, 1);
                if (at < kList) sh.list[at] = key_of(x, static_cast<uint32_t>(first + e));
            }
        }
    }

    // ---- the chunk's sum, over the largest reference
    const float all = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
    float most = ref;
#pragma unroll
    for (int o = 16; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (lane == 0) sh.warp_ref[warp] = most;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWarps; ++i) most = fmaxf(most, sh.warp_ref[i]);
    double total = all * exp2_approx((ref - most) * kLog2e);
#pragma unroll
    for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    if (lane == 0) sh.warp_sum[warp] = total;
    if (sh.count > kRanked || sh.lost) {
        const bool lost = sh.count > kList || sh.lost;
        __syncthreads();
        if (kRanked == kList || lost) candidates_exactly<T>(sh, row, c0, end, a.vocab, k);
        else trim_list(sh, k);      // more than ranking each takes
    } else {
        __syncthreads();
    }
    const int64_t part = static_cast<int64_t>(row_number) * p.chunks + number;
    if (tid == 0) {
        double s = 0;
        for (int i = 0; i < kWarps; ++i) s += sh.warp_sum[i];
        p.partials[part] = {s, most, 0.f};
    }
    const int n = sh.count;
    Key* out = p.lists + part * k;
    for (int i = tid; i < n; i += kThreads) {
        const Key mine = sh.list[i];
        const int rank = larger_than(mine, sh.list, n);
        if (rank < k) out[rank] = mine;
    }
    if (tid >= n && tid < k) out[tid] = 0;
}

// All lists of a group, by the CTA that finished its last chunk.  (It runs once: loops that are not unrolled come out ahead of the
// instructions that an unrolled one would have to fetch.)
static __device__ __noinline__ void merge(Shared& sh, const Params& p, int g) {
    const wuda_beam_select_args& a = p.a;
    constexpr int kParts = (kMostLists + kThreads - 1) / kThreads;
    const int tid = threadIdx.x, lane = tid & 31, k = a.k, chunks = p.chunks;
    const int per_beam = chunks * k, lists = a.width * chunks, entries = lists * k;
    const float by_beam = 1.f / per_beam;
    const auto beam_of = [&](int e) { return static_cast<int>((e + 0.5f) * by_beam); };      // e / per_beam: exact for e < kEntries
    // ---- everything there is to read, then the beams' sums, eight lanes each
    const Key* keys = p.lists + static_cast<int64_t>(g) * entries;
    const Partial* partials = p.partials + static_cast<int64_t>(g) * lists;
    Key key[4];
    const auto load = [&](int e0) {
#pragma unroll
        for (int u = 0; u < 4; ++u) key[u] = e0 + u * kThreads < entries ? __ldcg(keys + e0 + u * kThreads) : 0;
    };
    const auto store = [&](int e0) {
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (e0 + u * kThreads < entries) sh.entry[e0 + u * kThreads] = key[u];
    };
    float ref[kParts], score = 0.f;
    double sum[kParts];
    bool ended = false;
#pragma unroll
    for (int i = 0; i < kParts; ++i)
        if (i * kThreads + tid < lists) ref[i] = __ldcg(&partials[i * kThreads + tid].ref), sum[i] = __ldcg(&partials[i * kThreads + tid].sum);
    load(tid);
    if (tid < a.width) {
        score = __ldcg(a.scores + g * a.width + tid);
        ended = a.finished && __ldcg(a.finished + g * a.width + tid);
    }
#pragma unroll
    for (int i = 0; i < kParts; ++i)
        if (i * kThreads + tid < lists) sh.ref[i * kThreads + tid] = ref[i], sh.sum[i * kThreads + tid] = sum[i];
    if (tid < a.width) {
        sh.kind[tid] = !(fabsf(score) < INFINITY) ? 2 : ended;
        sh.score[tid] = score;
    }
    if (tid == 0) sh.survivors = sh.there = 0;
    if (tid < 128) sh.front[tid] = 0;
    __syncthreads();
#pragma unroll 1
    for (int w0 = 0; w0 < a.width; w0 += kThreads / 8) {
        const int w = w0 + tid / 8, at = min(w, a.width - 1) * chunks;
        float most = -FLT_MAX;
        for (int i = lane & 7; i < chunks; i += 8) most = fmaxf(most, sh.ref[at + i]);
#pragma unroll
        for (int o = 4; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        double total = 0;
        for (int i = lane & 7; i < chunks; i += 8) total += sh.sum[at + i] * exp2_approx((sh.ref[at + i] - most) * kLog2e);
#pragma unroll
        for (int o = 4; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        if (w < a.width && (lane & 7) == 0) sh.lse[w] = most + log(total);      // (of a beam that was not read: not used)
    }
    store(tid);
#pragma unroll 1
    for (int e0 = tid + 4 * kThreads; e0 < entries; e0 += 4 * kThreads) {
        load(e0);
        store(e0);
    }
    __syncthreads();

    // ---- values as ordered words (0 none), in 64 bits where they are compared, in 32 where they are only bounded
    const auto value = [&](int e) -> Key {
        const Key key = sh.entry[e];
        const int w = beam_of(e);
        if (sh.kind[w] == 1) return e == w * per_beam ? ordered(sh.score[w]) : 0;      // (its lists hold nothing)
        return sh.kind[w] == 0 && key ? ordered((sh.score[w] + unordered(static_cast<uint32_t>(key >> 32))) - sh.lse[w]) : 0;
    };
    const auto rounded = [](Key v) -> uint32_t { return v ? ordered(static_cast<float>(unordered(v))) : 0u; };
    // the first of every list, 16 k or 256 together, in 64 or 128 shares (neighbours in a list in different ones): nothing below
    // the k-th largest of the shares' largest is among the k best
    const int deep = min(k, (max(16 * k, 256) + lists - 1) / lists);
    const float by_deep = 1.f / deep;
    uint32_t part = 0;
#pragma unroll 1
    for (int i = tid; i < lists * deep; i += kThreads) {
        const int list = static_cast<int>((i + 0.5f) * by_deep);      // i / deep
        part = max(part, rounded(value(list * k + i - list * deep)));
    }
    if (part) atomicMax(&sh.front[tid % (k <= 32 ? 64 : 128)], part);
    __syncthreads();
    kth_part(sh.front, k, sh.bound, &sh.highest);
    __syncthreads();
    const uint32_t least = max(least_of(sh.bound), 1u);
    // the bound as a logit of each beam, a little lower (what is compared with it is rounded in other places)
    if (tid < a.width) {
        const double logit = unordered(least) - sh.score[tid] + sh.lse[tid];
        const float low = static_cast<float>(logit - 1e-6 * (fabs(logit) + fabs(sh.score[tid]) + fabs(sh.lse[tid])));
        sh.low[tid] = sh.kind[tid] == 0 ? (least > 1u && low == low ? ordered(low) : 1u) : sh.kind[tid] == 1 ? 0u : 0xffffffffu;
    }
    __syncthreads();
    const auto pass = [&](int e, Key v) {
        const int at = atomicAdd(&sh.survivors, 1);
        // lower beam; within a beam larger logit, lower token (tokens have 24 bits)
        if (at < kFew) sh.value[at] = v, sh.tie[at] = static_cast<Key>(31 - beam_of(e)) << 56 | sh.entry[e] >> 32 << 24 | (sh.entry[e] & 0xffffff);
    };
#pragma unroll 4
    for (int e = tid; e < entries; e += kThreads) {
        if (static_cast<uint32_t>(sh.entry[e] >> 32) < sh.low[beam_of(e)]) continue;
        const Key v = value(e);
        if (rounded(v) >= least) pass(e, v);
    }
    __syncthreads();
    int n = sh.survivors;
    if (n > kFew) {
        // a few beams have most of the best: the k-th largest value, exactly but for its rounding
        uint32_t mine[kEntries / kThreads];
#pragma unroll
        for (int i = 0; i < kEntries / kThreads; ++i) mine[i] = i * kThreads + tid < entries ? rounded(value(i * kThreads + tid)) : 0;
        const uint32_t bound = static_cast<uint32_t>(kth_largest(k, least, sh.highest, sh.hits, [&](const auto& f) {
#pragma unroll
            for (int i = 0; i < kEntries / kThreads; ++i)
                if (i * kThreads < entries) f(static_cast<Key>(mine[i]));
        }));
        __syncthreads();
        if (tid == 0) sh.survivors = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kEntries / kThreads; ++i)
            if (mine[i] && mine[i] >= bound) pass(i * kThreads + tid, value(i * kThreads + tid));
        __syncthreads();
        n = sh.survivors;
    }
    if (n > kFew) {
        // many equal values: the k best by value, then by beam, then by logit and token
        const auto all = [&](const auto& f) {      // f(entry, value, beam)
#pragma unroll 1
            for (int e = tid; e < entries; e += kThreads)
                if (const Key v = value(e)) f(e, v, beam_of(e));
        };
        const auto count = [&](const auto& test) {
            int c = 0;
            all([&](int e, Key v, int w) { c += test(e, v, w); });
            start_totals(sh.hits);
            return block_total(c, sh.hits, 0);
        };
        const Key worst = kth_largest(k, 0, ~0ull, sh.hits, [&](const auto& f) { all([&](int, Key v, int) { f(v); }); });
        int wanted = k - count([&](int, Key v, int) { return v > worst; });
        const int beam = 31 - static_cast<int>(kth_largest(wanted, 0, 31, sh.hits, [&](const auto& f) {
            all([&](int, Key v, int w) { if (v == worst) f(static_cast<Key>(31 - w)); });
        }));
        wanted -= count([&](int, Key v, int w) { return v == worst && w < beam; });
        const Key last = kth_largest(wanted, 0, ~0ull, sh.hits, [&](const auto& f) {
            all([&](int e, Key v, int w) { if (v == worst && w == beam) f(sh.entry[e]); });
        });
        __syncthreads();
        if (tid == 0) sh.survivors = 0;
        __syncthreads();
        all([&](int e, Key v, int w) {
            if (v > worst || (v == worst && (w < beam || (w == beam && sh.entry[e] >= last)))) pass(e, v);
        });
        __syncthreads();
        n = min(sh.survivors, kFew);      // (k of them)
    }

    // ---- their order
    for (int i = tid; i < n; i += kThreads) {
        const Key v = sh.value[i], tie = sh.tie[i];
        int rank = 0, j = 0;
#pragma unroll 4
        for (; j + 1 < n; j += 2) {
            const ulonglong2 other = *reinterpret_cast<const ulonglong2*>(&sh.value[j]), ties = *reinterpret_cast<const ulonglong2*>(&sh.tie[j]);
            rank += (other.x > v || (other.x == v && ties.x > tie)) + (other.y > v || (other.y == v && ties.y > tie));
        }
        if (j < n) rank += sh.value[j] > v || (sh.value[j] == v && sh.tie[j] > tie);
        if (rank >= k) continue;
        atomicAdd(&sh.there, 1);
        const int64_t at = static_cast<int64_t>(g) * k + rank;
        const int w = 31 - static_cast<int>(tie >> 56);
        const bool done = sh.kind[w] == 1;
        const int token = done ? a.eos_token : static_cast<int>(~tie & 0xffffff);
        a.scores_out[at] = static_cast<float>(unordered(v));
        a.parents_out[at] = w;
        a.tokens_out[at] = token;
        a.finished_out[at] = done || token == a.eos_token;
    }
    __syncthreads();
    for (int j = sh.there + tid; j < k; j += kThreads) {
        const int64_t at = static_cast<int64_t>(g) * k + j;
        a.scores_out[at] = -INFINITY;
        a.parents_out[at] = a.tokens_out[at] = -1;
        a.finished_out[at] = 0;
    }
}
};

template <typename T, int kThreads, bool ALIGNED>
__global__ void __launch_bounds__(kThreads, 896 / kThreads) beam_select_kernel(const __grid_constant__ Params p) {
    using B = Block<kThreads>;
    __shared__ typename B::Shared sh;
    const wuda_beam_select_args& a = p.a;
    pdl_launch_dependents();
    pdl_wait();   // nothing of global memory is touched before the kernel ahead has finished
    const int number = blockIdx.x, g = blockIdx.z, row = g * a.width + blockIdx.y;
    const T* x = static_cast<const T*>(a.logits) + g * a.group_stride + blockIdx.y * a.beam_stride;
    B::template chunk<T, ALIGNED>(sh, p, x, row, number);
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        const unsigned all = a.width * p.chunks - 1;
        sh.last = atomicInc(reinterpret_cast<unsigned*>(a.counters + g), all) == all;      // (wraps back to zero)
    }
    __syncthreads();
    if (!sh.last) return;
    __threadfence();
    B::merge(sh, p, g);
}

// How the rows are cut, into chunks of whole tiles and lists that the merge can hold.
//   Up to 148 rows of more work than a tile of 128 threads per SM: CTAs of 512 threads, one per SM at most.  Fewer and longer lists make
//   the merge shorter, and a CTA alone on its SM needs the threads.  7 x 5 rows x 100003 fp16: 11.7 us (13.1 in CTAs of 128), 128 rows x
//   131072 bf16, k = 16: 16.0 (17.8); 64 rows x 131072 fp32, k = 4: 13.1 (14.2).  On the other side of both limits 152 rows x 131072
//   bf16: 17.9 us in CTAs of 128, 24.4 in those of 512; 4 rows of them 9.2 (8.8).
//   So, too, where the lists leave fewer than two fifths of the places of CTAs of 128 threads (wide groups, large k): 8 x 32 rows x
//   131072 bf16, k = 64: 41.7 us (49.0 in CTAs of 128), 12 x 32: 59.1 (70.1), 6 x 32 rows, k = 32: 28.3 (35.0).  Beyond that, 16 x 32 rows,
//   k = 64: 60.0 us in CTAs of 128, 76.2 in those of 512 (13 x 32, next to the limit, would gain: 78.0, 60.0).
//   Otherwise CTAs of 128 threads, as many as are resident together (seven per SM).  512 rows x 131072 bf16: 32.3 us in two chunks a row,
//   35.1 in three, 48.4 with 512 threads; 4 rows x 32000 bf16: 8.0 us in eight chunks of a tile (8.7 with 512 threads).  Rows that
//   fill half of the places or little more leave the others empty, so they are cut in three: 600 rows x 131072 51.1 -> 39.8 us, 800 rows
//   52.4 -> 49.3; 960 rows in one chunk 53.9 (56.1 in three).
struct Cut {
    int threads, chunks, chunk_vectors;
};
Cut cut(int groups, int width, int vocab, int k, int type) {
    const int rows = groups * width, of_128 = (type == 2 ? 4 : 8) * kVectors * 128;
    Cut c = {};
    const int tiles_of_128 = (vocab + of_128 - 1) / of_128;
    const int held = std::min(std::min(kMostChunks, kMostLists / width), kEntries / (width * k));      // chunks of a row that the merge can hold
    const bool few_rows = rows <= kSms && static_cast<int64_t>(rows) * tiles_of_128 > kSms;
    const bool few_lists = held < tiles_of_128 && rows * held * 5 < 7 * kSms * 2;
    c.threads = few_rows || few_lists ? 512 : 128;
    const int tile = of_128 * (c.threads / 128), tiles = (vocab + tile - 1) / tile;
    const int resident = (c.threads == 512 ? 1 : 7) * kSms;
    int n = std::max(resident / rows, 1);
    if (n == 1 && rows * 5 < resident * 4 && tiles >= 6) n = 3;
    n = std::min(std::min(n, tiles), held);
    const int per = (tiles + n - 1) / n;
    c.chunks = (tiles + per - 1) / per;
    c.chunk_vectors = per * c.threads * kVectors;
    return c;
}

bool sizes_fit(int groups, int width, int vocab, int k, int type) {
    return groups >= 0 && groups <= kMostGroups && width >= 1 && width <= kMostWidth && vocab >= 1 && vocab <= 1 << 24 && k >= 1 &&
           k <= kMostK && type >= 0 && type <= 2;
}

}  // namespace beams
}  // namespace wuda

extern "C" int64_t wuda_beam_select_workspace_bytes(int groups, int width, int vocab, int k, int logits_type) {
    using namespace wuda::beams;
    if (!sizes_fit(groups, width, vocab, k, logits_type)) return -1;
    if (groups == 0) return 0;
    return static_cast<int64_t>(groups) * width * cut(groups, width, vocab, k, logits_type).chunks * (k * sizeof(Key) + sizeof(Partial));
}

extern "C" int wuda_beam_select(const wuda_beam_select_args* args, void* stream) {
    using namespace wuda;
    using namespace wuda::beams;
    clear_error();
    WUDA_REQUIRE(args, "args must not be NULL");
    const wuda_beam_select_args& a = *args;
    WUDA_REQUIRE(a.groups >= 0 && a.groups <= kMostGroups, "groups must be in [0, %d] (got %d)", kMostGroups, a.groups);
    WUDA_REQUIRE(a.width >= 1 && a.width <= kMostWidth, "width must be in [1, %d] (got %d)", kMostWidth, a.width);
    WUDA_REQUIRE(a.k >= 1 && a.k <= kMostK, "k must be in [1, %d] (got %d)", kMostK, a.k);
    WUDA_REQUIRE(a.vocab >= 1 && a.vocab <= 1 << 24, "vocab must be in [1, 2^24] (got %d)", a.vocab);
    WUDA_REQUIRE(a.logits_type >= 0 && a.logits_type <= 2, "logits_type must be 0, 1 or 2 (got %d)", a.logits_type);
    if (a.groups == 0) return WUDA_OK;
    WUDA_REQUIRE(a.logits && a.scores && a.scores_out && a.parents_out && a.tokens_out && a.finished_out && a.workspace && a.counters,
                 "logits, scores, outputs, workspace and counters must not be NULL");
    WUDA_REQUIRE(a.group_stride >= 0 && a.beam_stride >= 0, "strides must not be negative");
    WUDA_REQUIRE((reinterpret_cast<uintptr_t>(a.logits) & (a.logits_type == 2 ? 3 : 1)) == 0, "logits are not aligned to their type");
    WUDA_REQUIRE(a.eos_token >= -1 && a.eos_token < a.vocab, "eos_token must be in [-1, vocab) (got %d)", a.eos_token);
    WUDA_REQUIRE(!a.finished || a.eos_token >= 0, "finished beams need an eos_token");
    const int64_t need = wuda_beam_select_workspace_bytes(a.groups, a.width, a.vocab, a.k, a.logits_type);
    WUDA_REQUIRE(a.workspace_bytes >= need && aligned16(a.workspace), "the workspace needs %lld bytes on 16 bytes (got %lld)",
                 static_cast<long long>(need), static_cast<long long>(a.workspace_bytes));
    // a group that ends writes its outputs while others still read their scores and flags
    const int64_t beams = static_cast<int64_t>(a.groups) * a.width, best = static_cast<int64_t>(a.groups) * a.k;
    const auto apart = [&](const void* out, const void* in, int64_t size) {
        const auto o = reinterpret_cast<uintptr_t>(out), i = reinterpret_cast<uintptr_t>(in);
        return (o == i && a.k == a.width) || o + best * size <= i || i + beams * size <= o;
    };
    WUDA_REQUIRE(apart(a.scores_out, a.scores, sizeof(float)), "scores_out must not overlap scores (but be them where k = width)");
    WUDA_REQUIRE(!a.finished || apart(a.finished_out, a.finished, 1), "finished_out must not overlap finished (but be it where k = width)");
    DeviceInfo dev;
    if (const int st = current_device_info(&dev)) return st;
    Params p;
    p.a = a;
    const Cut c = cut(a.groups, a.width, a.vocab, a.k, a.logits_type);
    p.chunks = c.chunks;
    p.chunk_vectors = c.chunk_vectors;
    const int64_t parts = static_cast<int64_t>(a.groups) * a.width * p.chunks;
    p.partials = static_cast<Partial*>(a.workspace);
    p.lists = reinterpret_cast<Key*>(p.partials + parts);
    // whether all rows lie on 16 bytes
    const int64_t in_16 = a.logits_type == 2 ? 4 : 8;
    const bool aligned = aligned16(a.logits) && (a.width == 1 || a.beam_stride % in_16 == 0) && (a.groups == 1 || a.group_stride % in_16 == 0);
    using Kernel = void (*)(Params);
    static const Kernel kernels[2][2][3] = {
        {{beam_select_kernel<__nv_bfloat16, 128, false>, beam_select_kernel<__half, 128, false>, beam_select_kernel<float, 128, false>},
         {beam_select_kernel<__nv_bfloat16, 512, false>, beam_select_kernel<__half, 512, false>, beam_select_kernel<float, 512, false>}},
        {{beam_select_kernel<__nv_bfloat16, 128, true>, beam_select_kernel<__half, 128, true>, beam_select_kernel<float, 128, true>},
         {beam_select_kernel<__nv_bfloat16, 512, true>, beam_select_kernel<__half, 512, true>, beam_select_kernel<float, 512, true>}}};
    WUDA_CUDA(launch_pdl(kernels[aligned][c.threads == 512][a.logits_type], dim3(c.chunks, a.width, a.groups), dim3(c.threads), 0,
                         static_cast<cudaStream_t>(stream), p));
    return WUDA_OK;
}
