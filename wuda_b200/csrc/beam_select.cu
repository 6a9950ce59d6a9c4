// Beam selection: log-softmax over the vocabulary, cumulative scores, the k best continuations of a group's beams.
//
//   value[w, v] = score[w] + logit[w, v] - lse[w],   lse[w] = m + log sum_u exp(logit[w, u] - m)
//
// Within a beam the order of the values is that of the logits, so a beam's candidates are its k largest logits (ties to the lower
// token): keys of (order-preserving logit, ~token) are unique, and the largest key is the first candidate.  Only candidates of
// different beams are compared by value, in 64 bits.
//
// One launch.  A row of logits is cut into chunks, a CTA each, that are read once: 16 bytes per load, four loads per thread ahead of the
// four that it works on.  Every thread keeps a reference r and the sum of exp(x - r) of its elements (r follows the maximum only
// where a term would pass e^40: a rescaling is rare, and no term overflows).  Which element a thread gets depends on the element's number
// alone, not on the row's alignment, so equal rows have equal sums.
//
// Candidates: the k-th largest of 64 or 128 maxima over disjoint parts of the tiles so far is a lower bound of the chunk's k-th largest
// logit, raised in front of the tiles 0, 3, 15, ..; a vector of loads that passes it (a handful per tile) is noted and looked at in the
// end, with the last bound.  No barrier besides.  A list that overflowed (sorted rows, rows of one value) is made again by exact selections.
//
// The CTA that completes a group's counter merges its lists: the k-th largest of the lists' first candidates bounds what can be among
// the k best, and the few that pass are ranked by counting.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cfloat>
#include <climits>
#include <type_traits>

#include "host.h"

namespace wuda {
namespace beams {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kVectors = 4;                 // 16-byte loads per thread and tile
constexpr int kMostK = 64, kMostWidth = 32, kMostGroups = 256;
constexpr int kList = 2048;                 // candidates that a CTA holds, and that a group's chunks may have together
constexpr int kMostChunks = 64;
constexpr int kMostLists = 1024;            // of a group
constexpr int kFront = kMostLists + kMostK; // the lists' first candidates, at least k of them
constexpr int kCtas = 1184;                 // CTAs of a launch: eight per SM, taken as SMs come free
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
__device__ __forceinline__ Key key_of(float x, uint32_t token) { return (static_cast<Key>(ordered(x)) << 32) | ~token; }
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

// ---- a vector: 16 bytes of a row as four words
__device__ __forceinline__ uint4 load16(const void* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// Elements [at, at + kVec) of a row; masked from `end` on.  ALIGNED: the row lies on 16 bytes.  Otherwise two aligned loads, both within
// the row [0, vocab), are shifted together.
template <typename T, bool ALIGNED>
__device__ __forceinline__ uint4 load_vector(const T* __restrict__ row, int at, int end, int vocab) {
    constexpr int kVec = Type<T>::kVec;
    const T* p = row + at;
    if (at + kVec <= end) {
        if (ALIGNED) return load16(p);
        const uintptr_t address = reinterpret_cast<uintptr_t>(p);
        const int off = static_cast<int>(address & 15);
        const T* low = reinterpret_cast<const T*>(address - off);
        if (off == 0) return load16(p);
        if (low >= row && low + 2 * kVec <= row + vocab) {
            const uint4 a = load16(low), b = load16(low + kVec);
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
    }
    uint32_t w[4] = {Type<T>::kMasked, Type<T>::kMasked, Type<T>::kMasked, Type<T>::kMasked};
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (at + i < end) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (at + i < end) {
                const uint32_t x = reinterpret_cast<const uint16_t*>(p)[i];
                w[i / 2] = i & 1 ? (w[i / 2] & 0xffffu) | (x << 16) : (w[i / 2] & 0xffff0000u) | x;
            }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
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
struct Shared {
    alignas(16) Key list[kList];
    int count, vectors;                     // candidates, and vectors that may hold some (those beyond kList are lost)
    float bound;                            // the k-th largest logit so far, or less
    alignas(16) float part_max[128];        // maxima of parts of the tiles
    int hits[2];
    float warp_ref[kWarps];
    double warp_sum[kWarps];
    bool last;
    // merging
    union {
        Key value[kList];
        int vector[kList];                  // (of a chunk: vectors with a logit beyond the bound of their tile)
    };
    alignas(16) Key front[kFront];
    uint16_t passed[kList];
    double lse[kMostWidth], score[kMostWidth];
    int kind[kMostWidth];
    Key least;
    int survivors, there;
};

// How many of n keys are larger, two at a time.
__device__ __forceinline__ int larger_than(Key mine, const Key* keys, int n) {
    int rank = 0, i = 0;
#pragma unroll 4
    for (; i + 1 < n; i += 2) {
        const ulonglong2 other = *reinterpret_cast<const ulonglong2*>(keys + i);
        rank += (other.x > mine) + (other.y > mine);
    }
    if (i < n) rank += keys[i] > mine;
    return rank;
}

__device__ __forceinline__ int block_total(int mine, int* hits, int turn) {
    const int n = __reduce_add_sync(0xffffffffu, mine);
    if ((threadIdx.x & 31) == 0 && n) atomicAdd(&hits[turn], n);
    __syncthreads();
    const int total = hits[turn];
    if (threadIdx.x == 0) hits[turn ^ 1] = 0;      // (the other one was read before this barrier)
    __syncthreads();
    return total;
}

// The k largest of the list and of the tile's keys, exactly: the largest K such that k of them are at or above it, bit by bit.  They become
// the list (all of them where they are fewer).  Returns K.  All threads; ends behind a barrier.
template <int N>
__device__ Key select_exactly(Shared& sh, const Key (&tile)[N], int k) {
    Key held[kList / kThreads];
    const int count = min(sh.count, kList);
#pragma unroll
    for (int i = 0; i < kList / kThreads; ++i) held[i] = i * kThreads + threadIdx.x < count ? sh.list[i * kThreads + threadIdx.x] : 0;
    if (threadIdx.x == 0) sh.hits[0] = sh.hits[1] = 0;
    __syncthreads();
    Key least = 0;
    for (int bit = 63, turn = 0; bit >= 0; --bit, turn ^= 1) {
        const Key want = least | (1ull << bit);
        int mine = 0;
#pragma unroll
        for (int i = 0; i < kList / kThreads; ++i) mine += held[i] >= want;
#pragma unroll
        for (int i = 0; i < N; ++i) mine += tile[i] >= want;
        const int total = block_total(mine, sh.hits, turn);
        if (total >= k) least = want;
        if (total == k) break;
    }
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    const auto keep = [&](Key key) {
        if (key != 0 && key >= least) sh.list[atomicAdd(&sh.count, 1)] = key;      // (k of them at most)
    };
#pragma unroll
    for (int i = 0; i < kList / kThreads; ++i) keep(held[i]);
#pragma unroll
    for (int i = 0; i < N; ++i) keep(tile[i]);
    __syncthreads();
    return least;
}
__device__ __noinline__ void trim_list(Shared& sh, int k) {
    const Key none[1] = {0};
    select_exactly(sh, none, k);
}

// A chunk's k largest keys where the list overflowed (rows sorted upwards, rows of one value, rows masked but for their end): tile by tile with
// exact selections, as far as a tile has a key above the k-th largest so far.
template <typename T>
__device__ __noinline__ void candidates_exactly(Shared& sh, const T* row, int c0, int end, int vocab, int k) {
    constexpr int kVec = Type<T>::kVec;
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    Key least = 0;
    for (int at = c0; at < end; at += kThreads * kVec) {
        const int first = at + threadIdx.x * kVec;
        const uint4 v = load_vector<T, false>(row, first, end, vocab);
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

// A chunk of a row: its partial sum, and its k largest keys in descending order.
template <typename T, bool ALIGNED>
__device__ __forceinline__ void chunk(Shared& sh, const Params& p, const T* row, int row_number, int number) {
    constexpr int kVec = Type<T>::kVec;
    const wuda_beam_select_args& a = p.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, k = a.k;
    const int c0 = number * p.chunk_vectors * kVec, end = min(a.vocab, c0 + p.chunk_vectors * kVec);
    if (tid == 0) {
        sh.count = sh.vectors = 0;
        sh.bound = -INFINITY;
    }
    const bool few = k <= 32;
    const int by = few ? 4 : 2;
    const int tiles = (end - c0 + kThreads * kVectors * kVec - 1) / (kThreads * kVectors * kVec);
    uint4 next[kVectors];
#pragma unroll
    for (int u = 0; u < kVectors; ++u) next[u] = load_vector<T, ALIGNED>(row, c0 + (u * kThreads + tid) * kVec, end, a.vocab);
    float ref = -FLT_MAX, so_far = -INFINITY, bound = -INFINITY;
    float2 sum[2] = {{0.f, 0.f}, {0.f, 0.f}};
    int refresh = 0;      // the next tile in front of which the bound is raised: 0, 3, 15, 63, ..
    for (int tile = 0; tile < tiles; ++tile) {
        uint32_t w[kVectors][4];
#pragma unroll
        for (int u = 0; u < kVectors; ++u) {
            w[u][0] = without_nan<T>(next[u].x), w[u][1] = without_nan<T>(next[u].y);
            w[u][2] = without_nan<T>(next[u].z), w[u][3] = without_nan<T>(next[u].w);
        }
        const int e0 = c0 + (tile * kThreads * kVectors + tid) * kVec;      // first element of the thread's first vector
        if (tile + 1 < tiles) {
#pragma unroll
            for (int u = 0; u < kVectors; ++u)
                next[u] = load_vector<T, ALIGNED>(row, e0 + (kVectors + u) * kThreads * kVec, end, a.vocab);
        }
        // ---- the vectors' maxima; masked tokens are -inf from here on
        float high[kVectors], top;
        const auto maxima = [&] {
            top = -INFINITY;
#pragma unroll
            for (int u = 0; u < kVectors; ++u) {
                const float2 f = pair_of<T>(max_words<T>(max_words<T>(w[u][0], w[u][1]), max_words<T>(w[u][2], w[u][3])));
                high[u] = fmaxf(f.x, f.y);
                top = fmaxf(top, high[u]);
            }
        };
        maxima();
        if (top == INFINITY) {
#pragma unroll
            for (int u = 0; u < kVectors; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 f = pair_of<T>(w[u][i]);
                    if constexpr (sizeof(T) == 4) {
                        if (f.x == INFINITY) w[u][i] = Type<T>::kMasked;
                    } else {
                        if (f.x == INFINITY) w[u][i] = (w[u][i] & 0xffff0000u) | (Type<T>::kMasked & 0xffffu);
                        if (f.y == INFINITY) w[u][i] = (w[u][i] & 0xffffu) | (Type<T>::kMasked & 0xffff0000u);
                    }
                }
            maxima();
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
        for (int u = 0; u < kVectors; ++u)
#pragma unroll
            for (int i = 0; i < 4; i += sizeof(T) == 4 ? 2 : 1) {
                float2 x;
                if constexpr (sizeof(T) == 4) x = make_float2(__uint_as_float(w[u][i]), __uint_as_float(w[u][i + 1]));
                else x = pair_of<T>(w[u][i]);
                const float2 y = mul2(add2(x, minus), scale);
                const int to = sizeof(T) == 4 ? i / 2 : i & 1;
                sum[to] = add2(sum[to], make_float2(exp2_approx(y.x), exp2_approx(y.y)));
            }
        // ---- candidates
        so_far = fmaxf(so_far, top);
        bool with_equal = false;      // a logit equal to the bound is a candidate where the bound is this tile's
        if (tile == refresh) {
            refresh = 4 * refresh + 3;
            // maxima over 2 or 4 neighbouring threads and all tiles so far, at least twice k of them: 8 warps look for the k-th largest
            float part = fmaxf(so_far, __shfl_xor_sync(0xffffffffu, so_far, 1));
            if (few) part = fmaxf(part, __shfl_xor_sync(0xffffffffu, part, 2));
            if (tid % by == 0) sh.part_max[tid / by] = part;
            __syncthreads();
            int larger = 0, not_smaller = 0;      // than the thread's own part, among a quarter or half of them
#pragma unroll 4
            for (int i = 0; i < kThreads / 16; i += 4) {
                const float4 other = *reinterpret_cast<const float4*>(&sh.part_max[few ? tid % 4 * 4 + i * 4 : tid % 2 * 4 + i * 2]);
                larger += (other.x > part) + (other.y > part) + (other.z > part) + (other.w > part);
                not_smaller += (other.x >= part) + (other.y >= part) + (other.z >= part) + (other.w >= part);
            }
            if (!few) {
#pragma unroll 4
                for (int i = kThreads / 16; i < kThreads / 4; i += 4) {
                    const float4 other = *reinterpret_cast<const float4*>(&sh.part_max[tid % 2 * 4 + i * 2]);
                    larger += (other.x > part) + (other.y > part) + (other.z > part) + (other.w > part);
                    not_smaller += (other.x >= part) + (other.y >= part) + (other.z >= part) + (other.w >= part);
                }
            }
            int both = larger | not_smaller << 16;
            both += __shfl_xor_sync(0xffffffffu, both, 1);
            if (few) both += __shfl_xor_sync(0xffffffffu, both, 2);
            if ((both & 0xffff) < k && k <= both >> 16) sh.bound = part;      // (equal ones write the same)
            __syncthreads();
            with_equal = sh.bound > bound;
            bound = sh.bound;
        }
        if (with_equal ? top >= bound : top > bound) {
#pragma unroll
            for (int u = 0; u < kVectors; ++u)
                if (with_equal ? high[u] >= bound : high[u] > bound) {
                    const int at = atomicAdd(&sh.vectors, 1);
                    if (at < kList) sh.vector[at] = (tile * kVectors + u) * kThreads + tid;
                }
        }
    }

    // ---- candidates: the elements of the noted vectors that pass the last bound
    __syncthreads();
    const int vectors = sh.vectors;
    if (vectors <= kList)
        for (int i = tid; i < vectors; i += kThreads) {
            const int first = c0 + sh.vector[i] * kVec;
            const uint4 v = load_vector<T, ALIGNED>(row, first, end, a.vocab);
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
    if (sh.count > kThreads || vectors > kList) {
        const bool lost = sh.count > kList || vectors > kList;
        __syncthreads();
        if (lost) candidates_exactly<T>(sh, row, c0, end, a.vocab, k);
        else trim_list(sh, k);      // more than a thread each: down to the k largest
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
    if (tid < n) {
        const Key mine = sh.list[tid];
        const int rank = larger_than(mine, sh.list, n);
        if (rank < k) out[rank] = mine;
    }
    if (tid >= n && tid < k) out[tid] = 0;
}

// a word that grows with the value; 0 is below every number
__device__ __forceinline__ Key ordered(double x) {
    const long long b = __double_as_longlong(x);
    return static_cast<Key>(b) ^ (static_cast<Key>(b >> 63) | (1ull << 63));
}
__device__ __forceinline__ double unordered(Key u) { return __longlong_as_double(u & (1ull << 63) ? u ^ (1ull << 63) : ~u); }

// All lists of a group, by the CTA that finished its last chunk.
__device__ __noinline__ void merge(Shared& sh, const Params& p, int g) {
    const wuda_beam_select_args& a = p.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, k = a.k, chunks = p.chunks;
    const int per_beam = chunks * k, lists = a.width * chunks, entries = lists * k;
    // the lists' keys are on their way while the beams' sums are added
    const Key* keys = p.lists + static_cast<int64_t>(g) * entries;
    Key mine[kList / kThreads];
#pragma unroll
    for (int i = 0; i < kList / kThreads; ++i) mine[i] = i * kThreads + tid < entries ? __ldcg(keys + i * kThreads + tid) : 0;
    for (int w = warp; w < a.width; w += kWarps) {
        const int row = g * a.width + w;
        const float score = a.scores[row];
        const bool dead = !(fabsf(score) < INFINITY), done = !dead && a.finished && a.finished[row];
        double lse = 0;
        if (!dead && !done) {
            const Partial* parts = p.partials + static_cast<int64_t>(row) * chunks;
            float ref[kMostChunks / 32], most = -FLT_MAX;
            double sum[kMostChunks / 32], total = 0;
#pragma unroll
            for (int i = 0; i < kMostChunks / 32; ++i) {
                const int at = i * 32 + lane;
                ref[i] = at < chunks ? __ldcg(&parts[at].ref) : -FLT_MAX;
                sum[i] = at < chunks ? __ldcg(&parts[at].sum) : 0;
                most = fmaxf(most, ref[i]);
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
#pragma unroll
            for (int i = 0; i < kMostChunks / 32; ++i) total += sum[i] * exp(static_cast<double>(ref[i]) - most);
#pragma unroll
            for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
            lse = most + log(total);
        }
        if (lane == 0) sh.lse[w] = lse, sh.score[w] = score, sh.kind[w] = dead ? 2 : done;
    }
    if (tid == 0) sh.survivors = sh.there = 0, sh.least = 0;
    __syncthreads();
    // values as ordered words; the first `deep` of every list also side by side
    const int deep = (k + lists - 1) / lists, pool = lists * deep;
#pragma unroll
    for (int i = 0; i < kList / kThreads; ++i) {
        const int e = i * kThreads + tid;
        if (e >= entries) break;
        const int list = e / k, w = list / chunks;
        Key v = 0;
        if (sh.kind[w] == 0) {
            if (mine[i]) v = ordered((sh.score[w] + unordered(static_cast<uint32_t>(mine[i] >> 32))) - sh.lse[w]);
        } else if (sh.kind[w] == 1 && e == w * per_beam) {
            v = ordered(sh.score[w]);
            mine[i] = key_of(0.f, static_cast<uint32_t>(a.eos_token));
        }
        sh.list[e] = mine[i];
        sh.value[e] = v;
        if (e - list * k < deep) sh.front[list * deep + e - list * k] = v;
    }
    __syncthreads();
    // the k-th largest of the front: nothing below it is among the k best
    for (int i = tid; i < pool; i += kThreads) {
        const Key v = sh.front[i];
        int larger = 0, not_smaller = 0, j = 0;
#pragma unroll 4
        for (; j + 1 < pool; j += 2) {
            const ulonglong2 other = *reinterpret_cast<const ulonglong2*>(&sh.front[j]);
            larger += (other.x > v) + (other.y > v);
            not_smaller += (other.x >= v) + (other.y >= v);
        }
        if (j < pool) larger += sh.front[j] > v, not_smaller += sh.front[j] >= v;
        if (larger < k && k <= not_smaller) sh.least = v;
    }
    __syncthreads();
    const Key least = max(sh.least, 1ull);
    // (the front's places are free now: the values that pass, side by side)
    for (int e = tid; e < entries; e += kThreads)
        if (sh.value[e] >= least) sh.passed[atomicAdd(&sh.survivors, 1)] = static_cast<uint16_t>(e);
    __syncthreads();
    const int n = sh.survivors;
    const bool few = n <= kFront;
    if (few)
        for (int i = tid; i < n; i += kThreads) sh.front[i] = sh.value[sh.passed[i]];
    __syncthreads();
    for (int i = tid; i < n; i += kThreads) {
        const int e = sh.passed[i], w = e / per_beam;
        const Key v = sh.value[e];
        int rank = 0, equal = 0;
        if (few) {
            int j = 0;
#pragma unroll 4
            for (; j + 1 < n; j += 2) {
                const ulonglong2 other = *reinterpret_cast<const ulonglong2*>(&sh.front[j]);
                rank += (other.x > v) + (other.y > v);
                equal += (other.x == v) + (other.y == v);
            }
            if (j < n) rank += sh.front[j] > v, equal += sh.front[j] == v;
        } else {
            for (int j = 0; j < n; ++j) {
                const Key other = sh.value[sh.passed[j]];
                rank += other > v;
                equal += other == v;
            }
        }
        if (rank >= k) continue;
        if (equal > 1) {      // lower beam; within a beam larger logit, lower token
            const Key key = sh.list[e];
            for (int j = 0; j < n; ++j) {
                const int o = sh.passed[j], ow = o / per_beam;
                if (sh.value[o] == v && o != e) rank += ow != w ? ow < w : sh.list[o] > key;
            }
            if (rank >= k) continue;
        }
        atomicAdd(&sh.there, 1);
        const int64_t at = static_cast<int64_t>(g) * k + rank;
        const int token = static_cast<int>(token_of(sh.list[e]));
        a.scores_out[at] = static_cast<float>(unordered(v));
        a.parents_out[at] = w;
        a.tokens_out[at] = token;
        a.finished_out[at] = sh.kind[w] == 1 || token == a.eos_token;
    }
    __syncthreads();
    for (int j = sh.there + tid; j < k; j += kThreads) {
        const int64_t at = static_cast<int64_t>(g) * k + j;
        a.scores_out[at] = -INFINITY;
        a.parents_out[at] = a.tokens_out[at] = -1;
        a.finished_out[at] = 0;
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 3) beam_select_kernel(const __grid_constant__ Params p) {
    __shared__ Shared sh;
    const wuda_beam_select_args& a = p.a;
    pdl_launch_dependents();
    pdl_wait();   // nothing of global memory is touched before the kernel ahead has finished
    const int number = blockIdx.x % p.chunks, row = blockIdx.x / p.chunks, g = row / a.width;
    const float score = a.scores[row];
    if (fabsf(score) < INFINITY && !(a.finished && a.finished[row])) {
        const T* x = static_cast<const T*>(a.logits) + g * a.group_stride + (row - g * a.width) * a.beam_stride;
        if ((reinterpret_cast<uintptr_t>(x) & 15) == 0) chunk<T, true>(sh, p, x, row, number);
        else chunk<T, false>(sh, p, x, row, number);
    }
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        const unsigned all = a.width * p.chunks - 1;
        sh.last = atomicInc(reinterpret_cast<unsigned*>(a.counters + g), all) == all;      // (wraps back to zero)
    }
    __syncthreads();
    if (!sh.last) return;
    __threadfence();
    merge(sh, p, g);
}

// Chunks of a row: enough CTAs for the device and whole rounds of loads for each, and lists that the merge can hold.
void cut(int groups, int width, int vocab, int k, int type, int* chunks, int* chunk_vectors) {
    const int vec = type == 2 ? 4 : 8, rows = groups * width;
    const int blocks = (vocab + vec * kThreads - 1) / (vec * kThreads);      // rounds of one load per thread
    int n = (kCtas + rows - 1) / rows;
    n = std::min(std::min(n, blocks), std::min(std::min(kMostChunks, kMostLists / width), kList / (width * k)));
    const int per = (blocks + n - 1) / n;
    *chunks = (blocks + per - 1) / per;
    *chunk_vectors = per * kThreads;
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
    int chunks, vectors;
    cut(groups, width, vocab, k, logits_type, &chunks, &vectors);
    return static_cast<int64_t>(groups) * width * chunks * (k * sizeof(Key) + sizeof(Partial));
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
    DeviceInfo dev;
    if (const int st = current_device_info(&dev)) return st;
    Params p;
    p.a = a;
    cut(a.groups, a.width, a.vocab, a.k, a.logits_type, &p.chunks, &p.chunk_vectors);
    const int64_t parts = static_cast<int64_t>(a.groups) * a.width * p.chunks;
    p.partials = static_cast<Partial*>(a.workspace);
    p.lists = reinterpret_cast<Key*>(p.partials + parts);
    void (*kernel)(Params) = a.logits_type == 0 ? beam_select_kernel<__nv_bfloat16> : a.logits_type == 1 ? beam_select_kernel<__half> : beam_select_kernel<float>;
    WUDA_CUDA(launch_pdl(kernel, dim3(static_cast<unsigned>(parts)), dim3(kThreads), 0, static_cast<cudaStream_t>(stream), p));
    return WUDA_OK;
}
