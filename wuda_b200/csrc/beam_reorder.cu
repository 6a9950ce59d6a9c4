// Beam reordering: slots of the new beams, and the copies of what forks take over from their parents.
//
// A lane looks at one new beam: match_any finds the children of one parent, of which the first keeps the parent's slot; one OR over the
// lanes gives the parents that have a child, and the slots of the other beams go to the further children in order.  Sources (parents)
// and destinations (beams without a child) are different slots, so all copies run at the same time and in place.
//
// Every CTA works out all groups for itself in shared memory, with the number of pieces that each fork's copy has (a few KB
// each: rows of the states, entries of one page of a pool); a scan over the forks numbers the pieces and the CTAs take them in turn.
//
// What bounds it: about 5 us of launch, slots, lengths, page tables and first loads, then HBM.  Per launch in a graph: 4 beams with two
// forks (0.8 MB moved) 5.7 us; 16 x 8 beams, 64 forks (32 MB) 9.9; 8 x 32 beams, 160 MB 31.3 - 5.1 TB/s with the start, 6.1 without,
// where a copy reaches 6.54.  Four loads of 16 bytes per thread and five CTAs of 256 threads per SM: four CTAs, or eight loads, were
// 1-3 us slower at 160 MB; plain stores took 34.6 us (they push out of L2 what is still to be read).
#include "batch_slots.cuh"

namespace wuda {
namespace reorder {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kUnroll = 4;                   // units of a thread in flight
constexpr int kResident = 5;                 // CTAs of an SM
constexpr int kBatch = 32;                   // pieces that a CTA plans at a time
constexpr int kPieceBytes = 16384;           // 16 bytes x kUnroll x kThreads

struct Params {
    wuda_beam_reorder_args a;
    const int32_t* parents;
    const int32_t* slots;
    int32_t* slots_out;
    int groups;
    int state_first[WUDA_BEAM_MAX_STATES + 1];   // the first piece of each state's rows, the pieces of all
    int state_pieces;
    int piece_shift[WUDA_BEAM_MAX_POOLS];        // entries of a page that are copied at a time: 2 ^ this, at least 4
    Divisor per_group;                           // beams
    Divisor per_entry[WUDA_BEAM_MAX_POOLS], per_block[WUDA_BEAM_MAX_POOLS], per_page[WUDA_BEAM_MAX_POOLS];      // tokens, entries, pieces
    int32_t* status;
};

inline size_t shared_bytes(int rows, int capacity) { return sizeof(int) * (8ull * rows + capacity); }
constexpr size_t kPlainBytes = 44 * 1024;    // of 48 KB that a launch may take without asking: the rest holds the static arrays

// The n-th lowest member of a set, -1 where there are fewer: halves, by their members.
__device__ __forceinline__ int lowest_but(uint32_t set, int n) {
    if (n >= __popc(set)) return -1;
    int at = 0;
#pragma unroll
    for (int half = 16; half; half >>= 1) {
        const int below = __popc(set & ((1u << half) - 1));
        if (n >= below) n -= below, set >>= half, at += half;
    }
    return at;
}

struct Span {
    int first_page, pages, entries;      // pages [first_page, pages), entries in all pages
};
__device__ __forceinline__ Span span_of(const Params& p, int pool, int length, int shared) {
    const int ring = p.a.pools[pool].ring;
    Span s;
    s.entries = static_cast<int>(p.per_entry[pool].quotient(length));
    if (ring > 0) s.entries = min(s.entries, ring);
    s.pages = static_cast<int>(p.per_block[pool].quotient_up(s.entries));
    s.first_page = ring > 0 ? 0 : min(static_cast<int>(p.per_block[pool].quotient(p.per_entry[pool].quotient(shared))), s.pages);
    return s;
}
__device__ __forceinline__ int pieces_of(const Params& p, int pool, const Span& s) {
    if (s.first_page >= s.pages) return 0;
    const int last = s.entries - (s.pages - 1) * p.a.pools[pool].entries_per_block;
    return (s.pages - 1 - s.first_page) * static_cast<int>(p.per_page[pool].by) + ((last + (1 << p.piece_shift[pool]) - 1) >> p.piece_shift[pool]);
}

// What one piece copies: up to two runs of units of 16 bytes, or of 4 where not everything lies on 16.
struct Piece {
    const uint8_t* src[2];
    uint8_t* dst[2];
    int units[2];
    bool wide;
    __device__ __forceinline__ void in_units() {      // of bytes
        uintptr_t bits = units[0] | units[1];
#pragma unroll
        for (int k = 0; k < 2; ++k) bits |= reinterpret_cast<uintptr_t>(src[k]) | reinterpret_cast<uintptr_t>(dst[k]);
        wide = (bits & 15) == 0;
        units[0] >>= wide ? 4 : 2;
        units[1] >>= wide ? 4 : 2;
    }
};

// By all threads of the block: four units in flight per thread, loads first.  Addresses by constant steps from two pointers: an index
// into either run for every unit takes five times the instructions.
template <typename Unit>
__device__ __forceinline__ void copy_units(const Piece& c) {
    const int tid = threadIdx.x, n1 = c.units[1];
    const Unit* src = reinterpret_cast<const Unit*>(c.src[0]) + tid;
    Unit* dst = reinterpret_cast<Unit*>(c.dst[0]) + tid;
    for (int rest = c.units[0] - tid; rest > 0; rest -= kUnroll * kThreads) {
        Unit v[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
            if (u * kThreads < rest) v[u] = __ldcg(src + u * kThreads);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
            if (u * kThreads < rest) __stcs(dst + u * kThreads, v[u]);
        src += kUnroll * kThreads;
        dst += kUnroll * kThreads;
    }
    // the second run from the last threads, which have least of the first
    for (int i = kThreads - 1 - tid; i < n1; i += kThreads)
        reinterpret_cast<Unit*>(c.dst[1])[i] = __ldcg(reinterpret_cast<const Unit*>(c.src[1]) + i);
}

__global__ void __launch_bounds__(kThreads, kResident) beam_reorder_kernel(const __grid_constant__ Params p) {
    extern __shared__ int mem[];
    __shared__ int scan[33];
    __shared__ Piece pieces[kBatch];
    static_assert(sizeof scan + sizeof pieces + 16 <= 48 * 1024 - kPlainBytes, "static and dynamic shared memory pass 48 KB together");
    const wuda_beam_reorder_args& a = p.a;
    const int width = a.width, rows = p.groups * width, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int* slot = mem;                 // of the beams now
    int* length = slot + rows;       // ... their tokens
    int* common = length + rows;     // ... and shared tokens
    int* parents = common + rows;    // of new beam j: the beam of its group that it continues
    int* source = parents + rows;    // the slot that its own is filled from, -1: no fork
    int* donor = source + rows;      // ... and the beam that has it
    int* own = donor + rows;         // its slot
    int* begin = own + rows;         // the number of its first piece
    int* first = begin + rows;       // (take_slots)
    int32_t* status = blockIdx.x == 0 ? p.status : nullptr;
    pdl_launch_dependents();
    pdl_wait();   // nothing of global memory is touched before the kernel ahead has finished
    const int per = (rows + kThreads - 1) / kThreads;
    const int b0 = min(tid * per, rows), b1 = min(b0 + per, rows);
    for (int b = b0; b < b1; ++b) {
        parents[b] = __ldcg(p.parents + b);
        const int s = slot[b] = __ldcg(p.slots + b);
        const bool inside = s >= 0 && s < a.capacity;
        length[b] = inside ? __ldcg(a.lengths + s) : -1;
        common[b] = inside && a.shared_lengths ? __ldcg(a.shared_lengths + s) : 0;
    }
    take_slots([&](int b) { return slot[b]; }, b0, b1, a.capacity, slot, first, status);
    __syncthreads();

    // ---- new slots and forks, and how much each fork copies: a lane per new beam, as many whole groups to a warp as fit
    const int together = static_cast<int>(p.per_group.quotient(32)), in_warp = static_cast<int>(p.per_group.quotient(lane));
    for (int g0 = warp * together; g0 < p.groups; g0 += kWarps * together) {
        const int at = (g0 + in_warp) * width, base = in_warp * width, j = lane - base, b = at + j;
        const bool mine = in_warp < together && g0 + in_warp < p.groups;
        const uint32_t below = (1u << lane) - 1, group = mine ? (width < 32 ? (1u << width) - 1 : 0xffffffffu) << base : 0;
        int parent = mine ? parents[b] : -1;
        const bool live = mine && slot[b] >= 0;
        const uint32_t all_live = __ballot_sync(0xffffffffu, live);
        if (parent < -1 || parent >= width) report(status, WUDA_DEV_BAD_PARENT);
        if (parent < 0 || parent >= width || !(all_live >> (base + parent) & 1)) parent = -1;
        const uint32_t siblings = __match_any_sync(0xffffffffu, parent >= 0 ? base + parent : -1);
        const bool keeps = parent >= 0 && lane == __ffs(siblings) - 1;
        const uint32_t has_child = __reduce_or_sync(0xffffffffu, parent >= 0 ? 1u << (base + parent) : 0u);
        const uint32_t further = __ballot_sync(0xffffffffu, parent >= 0 && !keeps) & group;
        const uint32_t orphans = __ballot_sync(0xffffffffu, mine && parent < 0) & group;
        if (!mine) continue;
        // (there are at least as many places as further children, unless slots were refused)
        const uint32_t places = (all_live & ~has_child & group) >> base;
        const int place = keeps ? parent : lowest_but(places, parent >= 0 ? __popc(further & below) : __popc(further) + __popc(orphans & below));
        int to = place >= 0 ? slot[at + place] : -1, from = -1, pieces = 0;
        if (parent >= 0 && !keeps && to >= 0) {
            const int tokens = length[at + parent], shared = common[at + parent];
            bool good = tokens >= 0 && shared >= 0 && length[at + place] == tokens && common[at + place] == shared;
            if (good) {
                from = slot[at + parent];
                pieces = p.state_pieces;
#pragma unroll
                for (int i = 0; i < WUDA_BEAM_MAX_POOLS; ++i) {
                    if (i >= a.num_pools) break;
                    const Span s = span_of(p, i, tokens, shared);
                    good = good && s.pages <= a.pools[i].table_width;
                    if (good) pieces += pieces_of(p, i, s);
                }
            }
            if (!good) {
                report(status, WUDA_DEV_BAD_LENGTH);
                to = from = -1;
                pieces = 0;
            }
        }
        source[b] = from;
        own[b] = to;
        donor[b] = from >= 0 ? at + parent : 0;
        begin[b] = pieces;
    }
    __syncthreads();
    int sum[1] = {0}, total[1];
    for (int b = b0; b < b1; ++b) {
        const int pieces = begin[b];
        begin[b] = sum[0];
        sum[0] += pieces;
    }
    block_exclusive_sum<1, kThreads>(sum, total, scan);
    for (int b = b0; b < b1; ++b) {
        begin[b] += sum[0];
        if (blockIdx.x == 0) p.slots_out[b] = own[b];
    }
    __syncthreads();

    // ---- the copies.  What a piece is takes divisions and two dependent loads: a thread per piece works that out for the CTA's next kBatch.
    const auto piece_of = [&](int unit) {
        Piece c = {};
        int b = 0;       // the last beam whose pieces start at or before this one: the fork that it belongs to
        for (int lo = 0, hi = rows; lo < hi;) {
            const int mid = (lo + hi) >> 1;
            if (begin[mid] <= unit) b = mid, lo = mid + 1;
            else hi = mid;
        }
        const int src = source[b], dst = own[b], tokens = length[donor[b]], shared = common[donor[b]];
        int piece = unit - begin[b];
        if (piece < p.state_pieces) {
            int i = 0;
            while (piece >= p.state_first[i + 1]) ++i;
            const int64_t bytes = a.states[i].row_bytes, at = static_cast<int64_t>(piece - p.state_first[i]) * kPieceBytes;
            uint8_t* data = static_cast<uint8_t*>(a.states[i].data);
            c.src[0] = data + src * bytes + at, c.dst[0] = data + dst * bytes + at;
            c.units[0] = static_cast<int>(min(static_cast<int64_t>(kPieceBytes), bytes - at));
            return c;
        }
        piece -= p.state_pieces;
#pragma unroll
        for (int i = 0; i < WUDA_BEAM_MAX_POOLS; ++i) {
            if (i >= a.num_pools) break;
            const wuda_beam_pool& pool = a.pools[i];
            const Span s = span_of(p, i, tokens, shared);
            const int n = pieces_of(p, i, s);
            if (piece >= n) {
                piece -= n;
                continue;
            }
            const int of = static_cast<int>(p.per_page[i].quotient(piece)), page = s.first_page + of;
            const int e0 = (piece - of * static_cast<int>(p.per_page[i].by)) << p.piece_shift[i];
            const int e1 = min(min(e0 + (1 << p.piece_shift[i]), pool.entries_per_block), s.entries - page * pool.entries_per_block);
            const int from = __ldcg(pool.table + static_cast<int64_t>(src) * pool.table_width + page);
            const int to = __ldcg(pool.table + static_cast<int64_t>(dst) * pool.table_width + page);
            if (from < 0 || from >= pool.num_blocks || to < 0 || to >= pool.num_blocks) {
                report(p.status, WUDA_DEV_BAD_PAGE_INDEX);
                return c;
            }
            int64_t offset = 0;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int64_t size = pool.segment_bytes[k], at = offset + e0 * size;
                c.src[k] = static_cast<const uint8_t*>(pool.data) + from * pool.stride_bytes + at;
                c.dst[k] = static_cast<uint8_t*>(pool.data) + to * pool.stride_bytes + at;
                c.units[k] = static_cast<int>((e1 - e0) * size);
                offset += pool.entries_per_block * size;
            }
            return c;
        }
        return c;
    };
    for (int64_t unit = blockIdx.x; unit < total[0]; unit += static_cast<int64_t>(kBatch) * gridDim.x) {
        const int64_t last = total[0] - 1 - unit;
        const int n = static_cast<int>(min(last / gridDim.x + 1, static_cast<int64_t>(kBatch)));
        if (tid < n) {
            Piece c = piece_of(static_cast<int>(unit + static_cast<int64_t>(tid) * gridDim.x));
            c.in_units();
            pieces[tid] = c;
        }
        __syncthreads();
        for (int i = 0; i < n; ++i) {
            if (pieces[i].wide) copy_units<uint4>(pieces[i]);
            else copy_units<uint32_t>(pieces[i]);
        }
        __syncthreads();
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
    const int beams = groups * a.width;
    WUDA_REQUIRE(groups == 0 || ((slots_out + beams <= slots || slots + beams <= slots_out) && (slots_out + beams <= parents || parents + beams <= slots_out)),
                 "slots_out must be an array of its own");
    Params p = {};
    p.a = a;
    p.per_group = Divisor(a.width);
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
        WUDA_REQUIRE(record <= 1 << 24, "pool %d: an entry of more than 16 MB", i);
        WUDA_REQUIRE(q.segment_bytes[1] == 0 || static_cast<int64_t>(q.entries_per_block) * q.segment_bytes[0] % 16 == 0,
                     "pool %d: the second segment must start on 16 bytes", i);
        WUDA_REQUIRE(q.stride_bytes >= q.entries_per_block * record, "pool %d: a page does not hold its entries", i);
        int shift = 2;      // entries of a piece: a power of two of them up to kPieceBytes
        while ((2 * record << shift) <= kPieceBytes && 1 << shift < q.entries_per_block) ++shift;
        p.piece_shift[i] = shift;
        p.per_entry[i] = Divisor(q.tokens_per_entry);
        p.per_block[i] = Divisor(q.entries_per_block);
        p.per_page[i] = Divisor((q.entries_per_block + (1 << shift) - 1) >> shift);
        // the table's pages bound the pieces of a fork
        pieces += static_cast<int64_t>(q.table_width) * p.per_page[i].by;
    }
    WUDA_REQUIRE(pieces < INT_MAX && pieces * groups * a.width < INT_MAX, "a reordering of more than 2^31 pieces");
    for (int i = 0; i < a.num_states; ++i) {
        p.state_pieces += static_cast<int>((a.states[i].row_bytes + kPieceBytes - 1) / kPieceBytes);
        p.state_first[i + 1] = p.state_pieces;
    }
    if (groups == 0) return WUDA_OK;
    DeviceInfo dev;
    if (const int st = current_device_info(&dev)) return st;
    const int rows = beams;
    const size_t smem = shared_bytes(rows, a.capacity);
    if (smem > kPlainBytes)
        WUDA_CUDA(cudaFuncSetAttribute(beam_reorder_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(shared_bytes(kMostRows, kMostSlots))));
    const int64_t most = pieces * rows;
    const int grid = static_cast<int>(most < kResident * dev.num_sms ? (most > 0 ? most : 1) : kResident * dev.num_sms);
    WUDA_CUDA(launch_pdl(beam_reorder_kernel, dim3(grid), dim3(kThreads), smem, static_cast<cudaStream_t>(stream), p));
    return WUDA_OK;
}
