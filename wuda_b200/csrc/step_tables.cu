// Step tables: positions, cache destinations, block tables and window entries of a step from the lengths of its requests, with the
// pages that growing requests take from the free stacks.
//
// For a row (slot, n tokens) with old = lengths[slot], now = old + n:  pages(x) = ceil((x / ratio) / entries_per_block) of each
// compressed pool are held at length x, so a row takes need = pages(now) - pages(old) pages; with `first` the sum of the needs of the rows
// in front of it, its page j >= pages(old) is free[count - 1 - (first + j - pages(old))].  Everything else follows from
// positions, divisions and the page tables, token by token and column by column.
//
// Every CTA works out all rows (slots, lengths, a scan over the needs) in shared memory, then the warps of all CTAs write the outputs.
// A launch of its own for the rows would cost more (2-3 us) than doing them 148 times side by side; what each CTA repeats are loads that
// all have to be waited for once.
//
// What bounds it is that chain: launch, slots, lengths, scan, tables or free pages, stores - four dependent round trips to L2.  Per launch
// in a graph, state in place / to other tensors: 1 request 4.0 / 4.1 us, 64 requests of 32768 tokens 4.6 / 4.2, 128 of a million tokens
// (tables of 4096 pages, 6.5 MB read and written: 1.0 us at 6.54 TB/s) 6.2 / 5.5, 37 requests with 65521 tokens between them - / 6.1 (in
// place costs a counter, a barrier and a write behind both).  In one CTA the latter two took 447 and 150 us.
// kPiece = 256: eight loads of a lane in flight, and 128 x 2 x 16 pieces give each of the 2368 warps two.
#include "batch_slots.cuh"

namespace wuda {
namespace steptables {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kPiece = 256;      // columns of a block table that a warp writes at a time

struct Params {
    wuda_step_tables_args a;
    const int32_t* slots;
    const int32_t* new_tokens;
    int rows;
    int32_t* status;
    Divisor ratio, ring, window, idx_epb, cmp_epb, swa_epb, pieces;
};

// What is known of a row, in shared memory
struct Rows {
    int* slot;        // -1: left out
    int* old_len;
    int* new_len;
    int* idx_first;   // pages that the rows in front of it take
    int* cmp_first;
    int* idx_need;    // and that it takes itself
    int* cmp_need;
    int* count;       // tokens
    int* start;       // rows + 1
    int* first;       // (take_slots)
    __device__ Rows(int* mem, int rows) {
        slot = mem, old_len = slot + rows, new_len = old_len + rows, idx_first = new_len + rows, cmp_first = idx_first + rows;
        idx_need = cmp_first + rows, cmp_need = idx_need + rows, count = cmp_need + rows, start = count + rows, first = start + rows + 1;
    }
};
inline size_t shared_bytes(int rows, int capacity) { return sizeof(int) * (9ull * rows + 1 + capacity); }

__device__ __forceinline__ int pages_of(const Params& p, uint32_t tokens, const Divisor& epb) {
    return static_cast<int>(epb.quotient_up(p.ratio.quotient(tokens)));
}

__device__ __forceinline__ int cut_count(int count, int capacity, int32_t* status) {
    if (count >= 0 && count <= capacity) return count;
    report(status, WUDA_DEV_BAD_LENGTH);
    return count < 0 ? 0 : capacity;
}

// Page `page` of a row: held before, or taken from the free stack in this step.
struct PoolView {
    const int32_t* table;   // the slot's row
    const int32_t* free;
    int held, top;          // page `held` is free[top], the next one free[top - 1]
    __device__ int operator()(int page) const { return __ldcg(page < held ? table + page : free + (top - (page - held))); }
};

// entry `entry` of a request, in page `page` of it, as an entry of the pool
__device__ __forceinline__ int64_t entry_of(int pool_page, const Divisor& epb, uint32_t page, uint32_t entry) {
    return static_cast<int64_t>(pool_page) * epb.by + (entry - page * epb.by);
}

__global__ void __launch_bounds__(kThreads) step_tables_kernel(const __grid_constant__ Params p) {
    extern __shared__ int mem[];
    __shared__ int scan[3 * 33];
    __shared__ int taken[2], stacks[2];
    __shared__ bool last;
    const wuda_step_tables_args& a = p.a;
    const int rows = p.rows, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const Rows r(mem, rows);
    pdl_launch_dependents();
    pdl_wait();   // nothing of global memory is touched before the kernel ahead has finished
    int32_t* status = blockIdx.x == 0 ? p.status : nullptr;

    // ---- the rows
    const int per = (rows + kThreads - 1) / kThreads;
    const int b0 = min(tid * per, rows), b1 = min(b0 + per, rows);
    // (one thread of a CTA reads the counts: all of them, of all CTAs, would queue for one address of L2)
    if (tid == 0) stacks[0] = __ldcg(a.free_counts), stacks[1] = __ldcg(a.free_counts + 1);
    take_slots([&](int b) { return __ldcg(p.slots + b); }, b0, b1, a.capacity, r.slot, r.first, status);
    const int free_idx = cut_count(stacks[0], a.idx_free_capacity, tid == 0 ? status : nullptr);
    const int free_cmp = cut_count(stacks[1], a.cmp_free_capacity, tid == 0 ? status : nullptr);
    int sum[3] = {0, 0, 0}, total[3];      // tokens, pages of both pools
    for (int b = b0; b < b1; ++b) {
        const int n = p.new_tokens ? __ldcg(p.new_tokens + b) : 1;
        const int counted = min(max(n, 0), a.max_tokens + 1);
        r.start[b] = sum[0];
        r.count[b] = n;
        sum[0] += counted;
        const int slot = r.slot[b];
        if (slot < 0) continue;
        const int old = __ldcg(a.lengths + slot);
        const int64_t now = static_cast<int64_t>(old) + n;
        const bool counts = old >= 0 && n >= 0 && now <= INT_MAX;
        const int idx_pages = counts ? pages_of(p, static_cast<uint32_t>(now), p.idx_epb) : 0;
        const int cmp_pages = counts ? pages_of(p, static_cast<uint32_t>(now), p.cmp_epb) : 0;
        if (!counts || idx_pages > a.table_width || cmp_pages > a.table_width) {
            report(status, WUDA_DEV_BAD_LENGTH);
            r.slot[b] = -1;
            continue;
        }
        r.old_len[b] = old;
        r.new_len[b] = static_cast<int>(now);
        r.idx_first[b] = sum[1];
        r.cmp_first[b] = sum[2];
        sum[1] += r.idx_need[b] = idx_pages - pages_of(p, old, p.idx_epb);
        sum[2] += r.cmp_need[b] = cmp_pages - pages_of(p, old, p.cmp_epb);
    }
    block_exclusive_sum<3, kThreads>(sum, total, scan);
    if (tid == 0) {
        taken[0] = taken[1] = 0;
        r.start[rows] = min(total[0], a.max_tokens);
    }
    __syncthreads();
    // Rows that would reach beyond the buffers or the stacks.  Their needs are in the sums of the rows behind them, which is the rule:
    // of the rows that need pages none behind the first that finds too few is served.  (Tokens beyond the buffers are a suffix, too.)
    for (int b = b0; b < b1; ++b) {
        const int n = max(r.count[b], 0);
        const int begin = r.start[b] + sum[0];
        r.start[b] = min(begin, a.max_tokens);
        if (r.slot[b] < 0) continue;
        const int idx_first = r.idx_first[b] + sum[1], cmp_first = r.cmp_first[b] + sum[2];
        const int idx_need = r.idx_need[b], cmp_need = r.cmp_need[b];
        if (begin + static_cast<int64_t>(n) > a.max_tokens) {
            report(status, WUDA_DEV_BAD_LENGTH);
            r.slot[b] = -1;
        } else if (idx_need + cmp_need > 0 && (idx_first + idx_need > free_idx || cmp_first + cmp_need > free_cmp)) {
            report(status, WUDA_DEV_NO_FREE_PAGE);
            r.slot[b] = -1;
        } else {
            r.idx_first[b] = free_idx - 1 - idx_first;      // (kept as the place of its first page in the stack)
            r.cmp_first[b] = free_cmp - 1 - cmp_first;
            if (idx_need + cmp_need > 0) {
                atomicMax(&taken[0], idx_first + idx_need);
                atomicMax(&taken[1], cmp_first + cmp_need);
            }
        }
    }
    __syncthreads();

    // ---- the state after the step.  In place it is written by the CTA that comes last here, when every CTA has read it.
    const bool in_place = a.lengths_out == a.lengths || a.free_counts_out == a.free_counts;
    bool mine = blockIdx.x == 0;
    if (in_place && gridDim.x > 1) {
        if (tid == 0) last = atomicInc(reinterpret_cast<unsigned*>(a.counter), gridDim.x - 1) == gridDim.x - 1;   // (wraps back to zero)
        __syncthreads();
        mine = last;
    }
    if (mine) {
        if (a.lengths_out != a.lengths) {
            for (int s = tid; s < a.capacity; s += kThreads) a.lengths_out[s] = __ldcg(a.lengths + s);
            __syncthreads();
        }
        for (int b = b0; b < b1; ++b)
            if (r.slot[b] >= 0) a.lengths_out[r.slot[b]] = r.new_len[b];
        if (tid == 0) {
            a.free_counts_out[0] = free_idx - taken[0];
            a.free_counts_out[1] = free_cmp - taken[1];
        }
    }
    if (blockIdx.x == 0)
        for (int b = tid; b <= rows; b += kThreads) a.token_starts[b] = r.start[b];

    // ---- the outputs, a task per warp: 256 columns of one pool's block table, a row's values and window entries, or 32 tokens
    const int window_pages = (a.window + a.swa_entries_per_block - 1) / a.swa_entries_per_block;
    const int tokens = r.start[rows];
    const int pieces = static_cast<int>(p.pieces.by), tables = rows * 2 * pieces;
    const int tasks = tables + rows + (tokens + 31) / 32;
    for (int task = blockIdx.x * kWarps + warp; task < tasks; task += gridDim.x * kWarps) {
        if (task < tables) {
            const int of = static_cast<int>(p.pieces.quotient(task)), piece = task - of * pieces, b = of >> 1;
            const bool cmp = of & 1;
            const Divisor epb = cmp ? p.cmp_epb : p.idx_epb;
            const int slot = r.slot[b];
            int32_t* out = (cmp ? a.cmp_block_table : a.idx_block_table) + b * a.block_table_stride;
            PoolView pool = {};
            int pages = 0;
            int32_t* table = nullptr;
            if (slot >= 0) {
                table = (cmp ? a.cmp_table : a.idx_table) + slot * a.table_stride;
                pages = pages_of(p, r.new_len[b], epb);
                pool = {table, cmp ? a.cmp_free : a.idx_free, pages - (cmp ? r.cmp_need[b] : r.idx_need[b]),
                        cmp ? r.cmp_first[b] : r.idx_first[b]};
            }
            int page[kPiece / 32];
#pragma unroll
            for (int i = 0; i < kPiece / 32; ++i) {      // all loads, then all stores
                const int column = piece * kPiece + i * 32 + lane;
                page[i] = column < pages ? pool(column) : 0;
            }
#pragma unroll
            for (int i = 0; i < kPiece / 32; ++i) {
                const int column = piece * kPiece + i * 32 + lane;
                if (column < a.table_width) out[column] = page[i];
                if (column < pages && column >= pool.held) table[column] = page[i];
            }
        } else if (task < tables + rows) {
            const int b = task - tables;
            const int slot = r.slot[b], now = slot >= 0 ? r.new_len[b] : 0;
            const int valid = min(now, a.window);
            const int32_t* pages = a.swa_table + static_cast<int64_t>(max(slot, 0)) * window_pages;
            const int only = window_pages == 1 ? __ldcg(pages) : 0;
            for (int i = lane; i < a.window; i += 32) {
                const uint32_t ring = i < valid ? p.window.rest(now - valid + i) : 0, page = p.swa_epb.quotient(ring);
                a.swa_indices[static_cast<int64_t>(b) * a.window + i] = i < valid ? static_cast<int>(((window_pages == 1 ? only : __ldcg(pages + page)) - page) * p.swa_epb.by + ring) : -1;
            }
            if (lane == 0) {
                const int entries = static_cast<int>(p.ratio.quotient(now));
                a.n_compressed[b] = entries;
                a.cmp_lengths[b] = min(entries, a.topk);
                a.swa_lengths[b] = valid;
            }
        } else if (const int t = (task - tables - rows) * 32 + lane; t < tokens) {
            int b = 0;       // the last row that starts at or before t (rows without tokens start where the next one does)
            for (int lo = 0, hi = rows; lo < hi;) {
                const int mid = (lo + hi) >> 1;
                if (r.start[mid] <= t) b = mid, lo = mid + 1;
                else hi = mid;
            }
            const int slot = r.slot[b];
            int pos = 0;
            int64_t state = -1, idx = -1, cmp = -1, swa = -1;
            if (slot >= 0) {
                const int old = r.old_len[b], now = r.new_len[b];
                pos = old + t - r.start[b];
                if (pos >= now - a.ring_entries) state = static_cast<int64_t>(slot) * a.ring_entries + p.ring.rest(pos);
                if (pos >= now - a.window) {
                    const uint32_t ring = p.window.rest(pos), page = p.swa_epb.quotient(ring);
                    swa = entry_of(__ldcg(a.swa_table + static_cast<int64_t>(slot) * window_pages + page), p.swa_epb, page, ring);
                }
                const uint32_t done = p.ratio.quotient(pos + 1u);
                if (done * p.ratio.by == pos + 1u) {
                    const uint32_t entry = done - 1, idx_page = p.idx_epb.quotient(entry), cmp_page = p.cmp_epb.quotient(entry);
                    const PoolView ip = {a.idx_table + slot * a.table_stride, a.idx_free, pages_of(p, old, p.idx_epb), r.idx_first[b]};
                    const PoolView cp = {a.cmp_table + slot * a.table_stride, a.cmp_free, pages_of(p, old, p.cmp_epb), r.cmp_first[b]};
                    idx = entry_of(ip(idx_page), p.idx_epb, idx_page, entry);
                    cmp = entry_of(cp(cmp_page), p.cmp_epb, cmp_page, entry);
                }
            }
            a.pos[t] = pos;
            a.q_pos[t] = pos;
            a.state_row[t] = state;
            a.idx_dst[t] = idx;
            a.cmp_dst[t] = cmp;
            a.swa_dst[t] = swa;
        }
    }
}

}  // namespace steptables
}  // namespace wuda

extern "C" int wuda_step_tables(const wuda_step_tables_args* args, const int32_t* slots, const int32_t* new_tokens, int rows,
                                int32_t* status_word, void* stream) {
    using namespace wuda;
    using namespace wuda::steptables;
    clear_error();
    WUDA_REQUIRE(args, "args must not be NULL");
    const wuda_step_tables_args& a = *args;
    WUDA_REQUIRE(rows >= 0 && rows <= kMostRows, "rows must be in [0, %d] (got %d)", kMostRows, rows);
    WUDA_REQUIRE(a.capacity >= 1 && a.capacity <= kMostSlots, "capacity must be in [1, %d] (got %d)", kMostSlots, a.capacity);
    WUDA_REQUIRE(a.table_width >= 1 && a.table_width <= 262144, "table_width must be in [1, 262144] (got %d)", a.table_width);
    WUDA_REQUIRE(a.max_tokens >= 0 && a.max_tokens <= 262144, "max_tokens must be in [0, 262144] (got %d)", a.max_tokens);
    WUDA_REQUIRE(new_tokens || rows <= a.max_tokens, "%d rows of one token do not fit max_tokens = %d", rows, a.max_tokens);
    WUDA_REQUIRE(a.table_stride >= a.table_width && a.block_table_stride >= a.table_width, "the tables' rows are shorter than table_width");
    WUDA_REQUIRE(a.idx_free_capacity >= 0 && a.cmp_free_capacity >= 0, "a free stack of negative size");
    WUDA_REQUIRE(a.idx_entries_per_block >= 1 && a.cmp_entries_per_block >= 1 && a.swa_entries_per_block >= 1,
                 "entries per block must be positive");
    WUDA_REQUIRE(a.ratio >= 1 && a.ring_entries >= 1 && a.window >= 1 && a.window <= 65536 && a.topk >= 0,
                 "ratio, ring_entries and window must be positive, window at most 65536, topk not negative");
    WUDA_REQUIRE(a.lengths && a.lengths_out && a.idx_table && a.cmp_table && a.swa_table && a.free_counts && a.free_counts_out &&
                     a.token_starts && a.n_compressed && a.cmp_lengths && a.swa_lengths && a.swa_indices && a.idx_block_table &&
                     a.cmp_block_table && a.counter,
                 "state, row outputs and counter must not be NULL");
    WUDA_REQUIRE(a.max_tokens == 0 || (a.pos && a.q_pos && a.state_row && a.idx_dst && a.cmp_dst && a.swa_dst),
                 "token outputs must not be NULL");
    WUDA_REQUIRE((a.idx_free || a.idx_free_capacity == 0) && (a.cmp_free || a.cmp_free_capacity == 0), "free stacks must not be NULL");
    WUDA_REQUIRE(a.idx_table != a.cmp_table, "the two pools must not share a page table");
    if (rows == 0 && a.lengths_out == a.lengths && a.free_counts_out == a.free_counts) return WUDA_OK;      // (there is nothing to write)
    WUDA_REQUIRE(slots || rows == 0, "slots must not be NULL");
    DeviceInfo dev;
    if (const int st = current_device_info(&dev)) return st;
    const size_t smem = shared_bytes(rows, a.capacity);
    if (smem > 48 * 1024 - 1024)
        WUDA_CUDA(cudaFuncSetAttribute(step_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(shared_bytes(kMostRows, kMostSlots))));
    Params p = {a, slots, new_tokens, rows, status_word};
    p.ratio = Divisor(a.ratio), p.ring = Divisor(a.ring_entries), p.window = Divisor(a.window);
    p.idx_epb = Divisor(a.idx_entries_per_block), p.cmp_epb = Divisor(a.cmp_entries_per_block), p.swa_epb = Divisor(a.swa_entries_per_block);
    p.pieces = Divisor((a.table_width + kPiece - 1) / kPiece);
    const int64_t tokens = new_tokens && rows ? a.max_tokens : rows;
    const int64_t tasks = static_cast<int64_t>(rows) * (2 * ((a.table_width + kPiece - 1) / kPiece) + 1) + (tokens + 31) / 32;
    const int grid = static_cast<int>(tasks < static_cast<int64_t>(dev.num_sms) * kWarps ? (tasks + kWarps - 1) / kWarps + (tasks == 0) : dev.num_sms);
    WUDA_CUDA(launch_pdl(step_tables_kernel, dim3(grid), dim3(kThreads), smem, static_cast<cudaStream_t>(stream), p));
    return WUDA_OK;
}
