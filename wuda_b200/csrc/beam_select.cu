// Beam selection: log-softmax over the vocabulary, cumulative scores, the k best continuations of a group's beams.
//
//   value[w, v] = score[w] + logit[w, v] - lse[w],   lse[w] = m + log sum_u exp(logit[w, u] - m)
//
// Within a beam the order of the values is that of the logits, so a beam's candidates are its k largest logits (ties to the lower
// token): keys of (order-preserving logit, ~token) are unique, and the largest key is the first candidate.  Only candidates of
// different beams are compared by value, in 64 bits.
//
// One CTA per beam finds maximum, sum and its k largest keys, one after the other; one CTA per group merges the beams' lists.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "host.h"

namespace wuda {
namespace beams {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMostK = 64, kMostWidth = 32, kMostGroups = 256;

struct Params {
    wuda_beam_select_args a;
    unsigned long long* lists;      // [groups * width, k] keys in descending order, 0 behind them
    double* lse;                    // [groups * width]
};

__device__ __forceinline__ float value_of(float x) { return x; }
__device__ __forceinline__ float value_of(__half x) { return __half2float(x); }
__device__ __forceinline__ float value_of(__nv_bfloat16 x) { return __bfloat162float(x); }

// a word that grows with x (no NaN); 0 is below every number
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x);
    return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u); }

template <typename T>
__device__ __forceinline__ float finite_or_lowest(T raw) {      // a masked token is -inf
    const float x = value_of(raw);
    return fabsf(x) < INFINITY ? x : -INFINITY;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) beam_rows_kernel(const Params p) {
    __shared__ float red_max[kWarps];
    __shared__ double red_sum[kWarps];
    __shared__ unsigned long long red_key[kWarps];
    const wuda_beam_select_args& a = p.a;
    pdl_launch_dependents();
    pdl_wait();
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (!(fabsf(a.scores[row]) < INFINITY) || (a.finished && a.finished[row])) return;
    const T* x = static_cast<const T*>(a.logits) + (row / a.width) * a.group_stride + (row % a.width) * a.beam_stride;
    float m = -INFINITY;
    for (int i = tid; i < a.vocab; i += kThreads) m = fmaxf(m, finite_or_lowest(x[i]));
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) red_max[warp] = m;
    __syncthreads();
    for (int i = 0; i < kWarps; ++i) m = fmaxf(m, red_max[i]);
    float s = 0.f;
    for (int i = tid; i < a.vocab; i += kThreads) {
        const float v = finite_or_lowest(x[i]);
        if (v > -INFINITY) s += expf(v - m);
    }
    double d = s;
#pragma unroll
    for (int o = 16; o; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
    if (lane == 0) red_sum[warp] = d;
    __syncthreads();
    if (tid == 0) {
        double total = 0;
        for (int i = 0; i < kWarps; ++i) total += red_sum[i];
        p.lse[row] = m > -INFINITY ? static_cast<double>(m) + log(total) : 0.0;
    }
    unsigned long long below = ~0ull;
    for (int j = 0; j < a.k; ++j) {
        unsigned long long best = 0;
        for (int i = tid; i < a.vocab; i += kThreads) {
            const float v = finite_or_lowest(x[i]);
            const unsigned long long key = v > -INFINITY ? (static_cast<unsigned long long>(ordered(v)) << 32) | ~static_cast<uint32_t>(i) : 0;
            if (key < below && key > best) best = key;
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
        if (lane == 0) red_key[warp] = best;
        __syncthreads();
        for (int i = 0; i < kWarps; ++i) best = max(best, red_key[i]);
        if (tid == 0) p.lists[static_cast<int64_t>(row) * a.k + j] = best;
        below = best;
        __syncthreads();
    }
}

// Position of each entry among all: how many come before it in (value descending, beam, logit descending, token).
__global__ void __launch_bounds__(kThreads) beam_merge_kernel(const Params p) {
    __shared__ double value[kMostWidth * kMostK];
    const wuda_beam_select_args& a = p.a;
    pdl_launch_dependents();
    pdl_wait();
    const int g = blockIdx.x, tid = threadIdx.x, entries = a.width * a.k;
    int there = 0;
    for (int e = tid; e < entries; e += kThreads) {
        const int row = g * a.width + e / a.k;
        const double score = a.scores[row];
        double v = -INFINITY;
        if (fabs(score) < INFINITY) {
            if (a.finished && a.finished[row]) {
                if (e % a.k == 0) v = score;
            } else if (const unsigned long long key = p.lists[static_cast<int64_t>(row) * a.k + e % a.k]) {
                v = (score + unordered(static_cast<uint32_t>(key >> 32))) - p.lse[row];
            }
        }
        value[e] = v;
    }
    __syncthreads();
    for (int e = 0; e < entries; ++e) there += value[e] > -INFINITY;
    for (int e = tid; e < entries; e += kThreads) {
        const double v = value[e];
        if (v == -INFINITY) continue;
        int rank = 0;
        for (int o = 0; o < entries; ++o) rank += value[o] > v || (value[o] == v && o < e);
        if (rank >= a.k) continue;
        const int beam = e / a.k, row = g * a.width + beam;
        const bool done = a.finished && a.finished[row];
        const int token = done ? a.eos_token : static_cast<int>(~static_cast<uint32_t>(p.lists[static_cast<int64_t>(row) * a.k + e % a.k]));
        const int64_t at = static_cast<int64_t>(g) * a.k + rank;
        a.scores_out[at] = static_cast<float>(v);
        a.parents_out[at] = beam;
        a.tokens_out[at] = token;
        a.finished_out[at] = done || token == a.eos_token;
    }
    for (int j = there + tid; j < a.k; j += kThreads) {
        const int64_t at = static_cast<int64_t>(g) * a.k + j;
        a.scores_out[at] = -INFINITY;
        a.parents_out[at] = a.tokens_out[at] = -1;
        a.finished_out[at] = 0;
    }
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
    return static_cast<int64_t>(groups) * width * (k + 1) * 8;
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
    const int rows = a.groups * a.width;
    Params p;
    p.a = a;
    p.lists = static_cast<unsigned long long*>(a.workspace);
    p.lse = reinterpret_cast<double*>(p.lists + static_cast<int64_t>(rows) * a.k);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (a.logits_type == 0) WUDA_CUDA(launch_pdl(beam_rows_kernel<__nv_bfloat16>, dim3(rows), dim3(kThreads), 0, s, p));
    if (a.logits_type == 1) WUDA_CUDA(launch_pdl(beam_rows_kernel<__half>, dim3(rows), dim3(kThreads), 0, s, p));
    if (a.logits_type == 2) WUDA_CUDA(launch_pdl(beam_rows_kernel<float>, dim3(rows), dim3(kThreads), 0, s, p));
    WUDA_CUDA(launch_pdl(beam_merge_kernel, dim3(a.groups), dim3(kThreads), 0, s, p));
    return WUDA_OK;
}
