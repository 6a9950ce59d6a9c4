// The request slots of a batch in shared memory: which rows have one, and which row has it first.  Every CTA of a kernel finds
// that out for itself (a few hundred cycles beside the loads that it waits for anyway), so that no launch is needed in front.
//
// What an earlier kernel may have written is read through L2 (__ldcg) here and in the kernels that include this: they start while
// that kernel runs, and a line in their SM's L1 may be older than its writes.
#pragma once
#include <climits>

#include "host.h"

namespace wuda {

constexpr int kMostSlots = 16384;      // one word of shared memory per slot
constexpr int kMostRows = 4096;

// Division of a 32-bit number by one that the host knows: a high product, an add and two shifts instead of some thirty
// instructions (T. Granlund and P. Montgomery, "Division by invariant integers using multiplication", figure 4.1).
struct Divisor {
    uint32_t by, factor;
    int shift1, shift2;
    Divisor() = default;
    explicit Divisor(uint32_t d) : by(d) {
        int l = 0;
        while (l < 32 && (1ull << l) < d) ++l;
        factor = static_cast<uint32_t>(((1ull << 32) * ((1ull << l) - d)) / d + 1);
        shift1 = l < 1 ? l : 1;
        shift2 = l > 1 ? l - 1 : 0;
    }
#ifdef __CUDACC__
    __device__ __forceinline__ uint32_t quotient(uint32_t n) const {
        const uint32_t t = __umulhi(factor, n);
        return (t + ((n - t) >> shift1)) >> shift2;
    }
    __device__ __forceinline__ uint32_t rest(uint32_t n) const { return n - quotient(n) * by; }
    __device__ __forceinline__ uint32_t quotient_up(uint32_t n) const {      // of n / by
        const uint32_t q = quotient(n);
        return q + (q * by != n);
    }
#endif
};

#ifdef __CUDACC__
__device__ __forceinline__ void report(int32_t* status, int code) {
    if (status) atomicCAS(status, 0, code);
}

// slot[b] = given(b), or -1 where it is outside [0, capacity) or an earlier row has it.  `first`: capacity words, whatever they
// hold.  All threads of the block; the rows of a thread are [b0, b1), and what it leaves of them only that thread may read before the
// next barrier.
template <typename Given>
__device__ __forceinline__ void take_slots(const Given& given, int b0, int b1, int capacity, int* slot, int* first, int32_t* status) {
    for (int b = b0; b < b1; ++b) {
        const int s = given(b);
        const bool inside = s >= 0 && s < capacity;
        if (!inside && s != -1) report(status, WUDA_DEV_BAD_SLOT);
        slot[b] = inside ? s : -1;
        if (inside) first[s] = INT_MAX;
    }
    __syncthreads();
    for (int b = b0; b < b1; ++b)
        if (slot[b] >= 0) atomicMin(&first[slot[b]], b);
    __syncthreads();
    for (int b = b0; b < b1; ++b)
        if (slot[b] >= 0 && first[slot[b]] != b) {
            report(status, WUDA_DEV_BAD_SLOT);
            slot[b] = -1;
        }
}

// Exclusive sums of N counts over the block's threads, in thread order, and the totals.  `scratch`: N * 33 words.
template <int N, int THREADS>
__device__ __forceinline__ void block_exclusive_sum(int (&v)[N], int (&total)[N], int* scratch) {
    static_assert(THREADS % 32 == 0 && THREADS <= 1024, "whole warps");
    constexpr int kWarps = THREADS / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int inclusive[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        int x = v[i];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        inclusive[i] = x;
        if (lane == 31) scratch[i * 33 + warp] = x;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        int x = lane < kWarps ? scratch[i * 33 + lane] : 0;      // every warp adds the warps' sums for itself
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        total[i] = __shfl_sync(0xffffffffu, x, 31);
        const int before = __shfl_sync(0xffffffffu, x, warp == 0 ? 0 : warp - 1);
        v[i] = inclusive[i] - v[i] + (warp == 0 ? 0 : before);
    }
}
#endif

}  // namespace wuda
