// Beam reordering: slots of the new beams, and the copies of what forks take over from their parents.
//
// Of a group's W <= 32 beams lane j of a warp looks at new beam j: match_any finds the children of one parent (the lowest keeps the
// parent's slot), one OR over the lanes the parents that have a child; the other beams' slots go to the further children in order.
// Sources (parents) and destinations (beams without a child) are different slots, so all copies run at the same time and in place.
//
// Every CTA works out all groups for itself in shared memory, with the number of pieces that each fork's copy has (a few KB
// each: rows of the states, entries of one page of a pool); a scan over the forks numbers the pieces and the CTAs take them in turn.
#include "batch_slots.cuh"

namespace wuda {
namespace reorder {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kPieceBytes = 16384;

struct Params {
    wuda_beam_reorder_args a;
    const int32_t* parents;
    const int32_t* slots;
    int32_t* slots_out;
    int groups;
    int state_pieces;                            // pieces of all state rows
    int piece_entries[WUDA_BEAM_MAX_POOLS];      // entries of a page that are copied at a time, a multiple of 4
    int32_t* status;
};

inline size_t shared_bytes(int rows, int capacity) { return sizeof(int) * (4ull * rows + 1 + capacity); }

__device__ __forceinline__ int lowest_but(uint32_t set, int n) {      // the n-th lowest member, -1 where there are fewer
    for (; n > 0 && set; --n) set &= set - 1;
    return set ? __ffs(set) - 1 : -1;
}

struct Span {
    int first_page, pages, entries;      // pages [first_page, pages), entries in all pages
};
__device__ __forceinline__ Span span_of(const wuda_beam_pool& pool, int length, int shared) {
    Span s;
    s.entries = pool.ring > 0 ? min(length / pool.tokens_per_entry, pool.ring) : length / pool.tokens_per_entry;
    s.pages = (s.entries + pool.entries_per_block - 1) / pool.entries_per_block;
    s.first_page = pool.ring > 0 ? 0 : min(shared / pool.tokens_per_entry / pool.entries_per_block, s.pages);
    return s;
}
__device__ __forceinline__ int pieces_of(const wuda_beam_pool& pool, const Span& s, int piece_entries) {
    if (s.first_page >= s.pages) return 0;
    const int per_page = (pool.entries_per_block + piece_entries - 1) / piece_entries;
    const int last = s.entries - (s.pages - 1) * pool.entries_per_block;
    return (s.pages - 1 - s.first_page) * per_page + (last + piece_entries - 1) / piece_entries;
}

// bytes (a multiple of 4) from src to dst by all threads of the block; 16 at a time where both lie on 16 bytes
__device__ __forceinline__ void copy_block(uint8_t* dst, const uint8_t* src, int64_t bytes) {
    int64_t done = 0;
    if (((reinterpret_cast<uintptr_t>(dst) | reinterpret_cast<uintptr_t>(src)) & 15) == 0) {
        const int64_t n = bytes / 16;
        for (int64_t i = threadIdx.x; i < n; i += kThreads) reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(src)[i];
        done = n * 16;
    }
    for (int64_t i = done / 4 + threadIdx.x; i < bytes / 4; i += kThreads)
        reinterpret_cast<uint32_t*>(dst)[i] = reinterpret_cast<const uint32_t*>(src)[i];
}

__global__ void __launch_bounds__(kThreads) beam_reorder_kernel(const __grid_constant__ Params p) {
    extern __shared__ int mem[];
    __shared__ int scan[33];
    const wuda_beam_reorder_args& a = p.a;
    const int width = a.width, rows = p.groups * width, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int* slot = mem;                 // of the beams now
    int* source = slot + rows;       // of new beam j: the slot that its own is filled from, -1 no fork
    int* own = source + rows;        // of new beam j: its slot
    int* begin = own + rows;         // of new beam j: the number of its first piece
    int* first = begin + rows + 1;   // (load_slots)
    int32_t* status = blockIdx.x == 0 ? p.status : nullptr;
    pdl_launch_dependents();
    pdl_wait();   // nothing of global memory is touched before the kernel ahead has finished
    const int per = (rows + kThreads - 1) / kThreads;
    const int b0 = min(tid * per, rows), b1 = min(b0 + per, rows);
    load_slots(p.slots, b0, b1, a.capacity, slot, first, status);
    for (int b = b0; b < b1; ++b) source[b] = p.parents[b];
    __syncthreads();

    // ---- new slots and forks, a group per warp
    for (int g = warp; g < p.groups; g += kWarps) {
        const int at = g * width + lane;
        const bool mine = lane < width;
        const int now = mine ? slot[at] : -1;
        int parent = mine ? source[at] : -1;
        if (parent < -1 || parent >= width) {
            report(status, WUDA_DEV_BAD_PARENT);
            parent = -1;
        }
        const int from = __shfl_sync(0xffffffffu, now, max(parent, 0));
        if (parent >= 0 && from < 0) parent = -1;
        const uint32_t children = __match_any_sync(0xffffffffu, parent);
        const bool keeps = parent >= 0 && lane == __ffs(children) - 1;
        const uint32_t has_child = __reduce_or_sync(0xffffffffu, parent >= 0 ? 1u << parent : 0u);
        const uint32_t places = __ballot_sync(0xffffffffu, now >= 0) & ~has_child;
        const uint32_t further = __ballot_sync(0xffffffffu, parent >= 0 && !keeps);
        const uint32_t orphans = __ballot_sync(0xffffffffu, mine && parent < 0);
        const uint32_t below = (1u << lane) - 1;
        // (a parent's further children are at most as many as there are places, unless slots were refused)
        const int place = keeps ? parent : (parent >= 0 ? lowest_but(places, __popc(further & below))
                                                        : lowest_but(places, __popc(further) + __popc(orphans & below)));
        int to = __shfl_sync(0xffffffffu, now, max(place, 0));
        if (place < 0) to = -1;
        __syncwarp();
        if (mine) {
            source[at] = parent >= 0 && !keeps && to >= 0 ? from : -1;
            own[at] = to;
        }
    }
    __syncthreads();

    // ---- how much each fork copies
    int sum[1] = {0}, total[1];
    for (int b = b0; b < b1; ++b) {
        begin[b] = sum[0];
        if (source[b] < 0) continue;
        const int length = a.lengths[source[b]], shared = a.shared_lengths ? a.shared_lengths[source[b]] : 0;
        bool good = length >= 0 && shared >= 0 && a.lengths[own[b]] == length && (!a.shared_lengths || a.shared_lengths[own[b]] == shared);
        int pieces = p.state_pieces;
        for (int i = 0; i < a.num_pools; ++i) {
            const Span s = span_of(a.pools[i], length, shared);
            good = good && s.pages <= a.pools[i].table_width;
            if (good) pieces += pieces_of(a.pools[i], s, p.piece_entries[i]);
        }
        if (!good) {
            report(status, WUDA_DEV_BAD_LENGTH);
            source[b] = own[b] = -1;
            continue;
        }
        sum[0] += pieces;
    }
    block_exclusive_sum<1, kThreads>(sum, total, scan);
    for (int b = b0; b < b1; ++b) {
        begin[b] += sum[0];
        if (blockIdx.x == 0) p.slots_out[b] = own[b];
    }
    __syncthreads();

    // ---- the copies
    for (int unit = blockIdx.x; unit < total[0]; unit += gridDim.x) {
        int b = 0;       // the last beam whose pieces start at or before this one: the fork that it belongs to
        for (int lo = 0, hi = rows; lo < hi;) {
            const int mid = (lo + hi) >> 1;
            if (begin[mid] <= unit) b = mid, lo = mid + 1;
            else hi = mid;
        }
        const int src = source[b], dst = own[b];
        int piece = unit - begin[b];
        if (piece < p.state_pieces) {
            for (int i = 0; i < a.num_states; ++i) {
                const int64_t bytes = a.states[i].row_bytes;
                const int n = static_cast<int>((bytes + kPieceBytes - 1) / kPieceBytes);
                if (piece < n) {
                    const int64_t at = static_cast<int64_t>(piece) * kPieceBytes;
                    uint8_t* data = static_cast<uint8_t*>(a.states[i].data);
                    copy_block(data + dst * bytes + at, data + src * bytes + at, min(static_cast<int64_t>(kPieceBytes), bytes - at));
                    break;
                }
                piece -= n;
            }
            continue;
        }
        piece -= p.state_pieces;
        const int length = a.lengths[src], shared = a.shared_lengths ? a.shared_lengths[src] : 0;
        for (int i = 0; i < a.num_pools; ++i) {
            const wuda_beam_pool& pool = a.pools[i];
            const Span s = span_of(pool, length, shared);
            const int step = p.piece_entries[i], n = pieces_of(pool, s, step);
            if (piece >= n) {
                piece -= n;
                continue;
            }
            const int per_page = (pool.entries_per_block + step - 1) / step;
            const int page = s.first_page + piece / per_page, e0 = piece % per_page * step;
            const int e1 = min(min(e0 + step, pool.entries_per_block), s.entries - page * pool.entries_per_block);
            const int from = pool.table[static_cast<int64_t>(src) * pool.table_width + page];
            const int to = pool.table[static_cast<int64_t>(dst) * pool.table_width + page];
            if (from < 0 || from >= pool.num_blocks || to < 0 || to >= pool.num_blocks) {
                report(p.status, WUDA_DEV_BAD_PAGE_INDEX);
                break;
            }
            uint8_t* data = static_cast<uint8_t*>(pool.data);
            int64_t offset = 0;
            for (int k = 0; k < 2; ++k) {
                const int64_t size = pool.segment_bytes[k];
                copy_block(data + to * pool.stride_bytes + offset + e0 * size, data + from * pool.stride_bytes + offset + e0 * size,
                           (e1 - e0) * size);
                offset += pool.entries_per_block * size;
            }
            break;
        }
    }
}

}  // namespace reorder
}  // namespace wuda

extern "C" int wuda_beam_reorder(const wuda_beam_reorder_args* args, const int32_t* parents, const int32_t* slots, int32_t* slots_out,
                                 int groups, int32_t* status_word, void* stream) {
    using namespace wuda;
    using namespace wuda::reorder;
    clear_error();
    WUDA_REQUIRE(args, "args must not be NULL");
    const wuda_beam_reorder_args& a = *args;
    WUDA_REQUIRE(a.width >= 1 && a.width <= 32, "width must be in [1, 32] (got %d)", a.width);
    WUDA_REQUIRE(groups >= 0 && groups <= kMostRows / a.width, "groups * width must be in [0, %d] (got %d * %d)", kMostRows, groups, a.width);
    WUDA_REQUIRE(a.capacity >= 1 && a.capacity <= kMostSlots, "capacity must be in [1, %d] (got %d)", kMostSlots, a.capacity);
    WUDA_REQUIRE(a.num_states >= 0 && a.num_states <= WUDA_BEAM_MAX_STATES, "num_states must be in [0, %d]", WUDA_BEAM_MAX_STATES);
    WUDA_REQUIRE(a.num_pools >= 0 && a.num_pools <= WUDA_BEAM_MAX_POOLS, "num_pools must be in [0, %d]", WUDA_BEAM_MAX_POOLS);
    WUDA_REQUIRE(a.lengths, "lengths must not be NULL");
    WUDA_REQUIRE(groups == 0 || (parents && slots && slots_out), "parents, slots and slots_out must not be NULL");
    WUDA_REQUIRE(groups == 0 || (slots_out != slots && slots_out != parents), "slots_out must be an array of its own");
    Params p = {};
    p.a = a;
    p.parents = parents, p.slots = slots, p.slots_out = slots_out, p.groups = groups, p.status = status_word;
    int64_t pieces = 0;
    for (int i = 0; i < a.num_states; ++i) {
        const wuda_beam_state& s = a.states[i];
        WUDA_REQUIRE(s.data && s.row_bytes > 0 && s.row_bytes % 4 == 0 && (reinterpret_cast<uintptr_t>(s.data) & 3) == 0,
                     "state %d must be 4-byte aligned rows of a multiple of 4 bytes", i);
        pieces += (s.row_bytes + kPieceBytes - 1) / kPieceBytes;
    }
    for (int i = 0; i < a.num_pools; ++i) {
        const wuda_beam_pool& q = a.pools[i];
        const int64_t record = static_cast<int64_t>(q.segment_bytes[0]) + q.segment_bytes[1];
        WUDA_REQUIRE(q.data && q.table && aligned16(q.data) && q.stride_bytes % 16 == 0, "pool %d must be 16-byte aligned pages", i);
        WUDA_REQUIRE(q.num_blocks >= 1 && q.table_width >= 1 && q.entries_per_block >= 1 && q.tokens_per_entry >= 1 && q.ring >= 0,
                     "pool %d: sizes must be positive", i);
        WUDA_REQUIRE(q.segment_bytes[0] > 0 && q.segment_bytes[0] % 4 == 0 && q.segment_bytes[1] >= 0 && q.segment_bytes[1] % 4 == 0,
                     "pool %d: segments must be multiples of 4 bytes", i);
        WUDA_REQUIRE(q.segment_bytes[1] == 0 || static_cast<int64_t>(q.entries_per_block) * q.segment_bytes[0] % 16 == 0,
                     "pool %d: the second segment must start on 16 bytes", i);
        WUDA_REQUIRE(q.stride_bytes >= q.entries_per_block * record, "pool %d: a page does not hold its entries", i);
        int step = 4;      // entries of a piece: a power of two of them up to kPieceBytes (20 % more where that halves the pieces)
        while (step * 2 * record <= kPieceBytes * 6 / 5 && step < q.entries_per_block) step *= 2;
        p.piece_entries[i] = step;
        // the table's pages bound the pieces of a fork
        pieces += static_cast<int64_t>(q.table_width) * ((q.entries_per_block + step - 1) / step);
    }
    WUDA_REQUIRE(pieces * groups * a.width < INT_MAX, "a reordering of more than 2^31 pieces");
    for (int i = 0; i < a.num_states; ++i) p.state_pieces += static_cast<int>((a.states[i].row_bytes + kPieceBytes - 1) / kPieceBytes);
    if (groups == 0) return WUDA_OK;
    DeviceInfo dev;
    if (const int st = current_device_info(&dev)) return st;
    const int rows = groups * a.width;
    const size_t smem = shared_bytes(rows, a.capacity);
    if (smem > 48 * 1024 - 1024)
        WUDA_CUDA(cudaFuncSetAttribute(beam_reorder_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(shared_bytes(kMostRows, kMostSlots))));
    const int64_t most = pieces * rows;
    const int grid = static_cast<int>(most < 4 * dev.num_sms ? (most > 0 ? most : 1) : 4 * dev.num_sms);
    WUDA_CUDA(launch_pdl(beam_reorder_kernel, dim3(grid), dim3(kThreads), smem, static_cast<cudaStream_t>(stream), p));
    return WUDA_OK;
}
