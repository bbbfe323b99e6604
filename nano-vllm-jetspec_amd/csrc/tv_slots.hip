// Block tables and slot maps built on the device from request lengths, for gfx950.
//
//   block_tables_kernel  a batch's page tables after an admission or a growth step: request r of
//                        lengths[r] tokens needs ceil(lengths[r] / B) pages, holds held_counts[r]
//                        already and takes the rest from the free list, in request order.
//   slot_maps_kernel     the packed rows of a batch: row offsets, each row's request and index in
//                        it, its position and its cache slot, through the block tables (prefill,
//                        decode) or through a packed arena (draft trees).
//
// Both are prefix sums over the requests followed by independent rows.  The sums are a few KB that
// stay in the L2, so every workgroup recomputes what it needs of them instead of waiting for a
// launch that publishes them: one launch each, no workspace, no atomics.  Latency bounds both (three
// dependent loads, two scans): tables of 2048 entries for 512 requests 5.7 us (6.3 MB, 1.1 TB/s), the maps of 250
// rows 3.9 us, of 531 thousand rows 8.7 us (1.5 TB/s).
#include <stdint.h>

#include "tv_internal.h"

namespace tv {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

// Inclusive prefix sum over the workgroup; *total receives the sum.  `part` is kWaves words of LDS
// that no earlier use of may still be in flight.
__device__ __forceinline__ int64_t block_scan(int64_t x, int64_t* part, int64_t* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t y = __shfl_up(x, o);
        if (lane >= o) x += y;
    }
    if (lane == 63) part[wave] = x;
    __syncthreads();
    int64_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        if (w < wave) before += part[w];
        all += part[w];
    }
    __syncthreads();
    *total = all;
    return x + before;
}

struct TableParams {
    const int32_t* lengths;
    const int32_t* held;       // [R, held_stride], held_width entries a row
    int64_t held_stride;
    int32_t held_width;
    const int32_t* held_counts;
    const int32_t* free_pages;
    const int32_t* free_count; // live entries of free_pages, or null: free_capacity
    int32_t free_capacity;
    int32_t num_requests, block_size, width;
    int32_t* tables;           // [R, width]
    int32_t* counts;
    int32_t* taken;
    int32_t* status;
};

struct Need {
    int32_t held;
    int64_t pages;   // pages the length needs
    int64_t grow;    // pages to take from the free list
    bool bad;
};

__device__ __forceinline__ Need need_of(const TableParams& p, int r) {
    Need n;
    const int32_t len = p.lengths[r];
    const int32_t held = p.held_counts ? p.held_counts[r] : 0;
    n.bad = len < 0 || held < 0 || held > p.held_width;
    n.held = held < 0 ? 0 : held > p.held_width ? p.held_width : held;
    n.pages = len <= 0 ? 0 : (static_cast<int64_t>(len) + p.block_size - 1) / p.block_size;
    n.grow = n.pages > p.width || n.pages <= n.held ? 0 : n.pages - n.held;
    return n;
}

// Workgroup w writes the rows of requests [w*R/G, (w+1)*R/G): it sums the growth of all earlier
// requests, scans its own, and fills one row after the other.  A request is granted its pages iff
// they fit the table and the free list still holds them, so once the list is short every later
// request that grows is refused too, and what is taken is a prefix of the list.
__global__ void __launch_bounds__(kThreads)
block_tables_kernel(const TableParams p) {
    __shared__ int64_t part[kWaves];
    __shared__ int64_t row_at[kThreads];
    __shared__ int32_t row_held[kThreads], row_count[kThreads];
    const int tid = threadIdx.x;
    const int64_t R = p.num_requests, G = gridDim.x;
    const int first = static_cast<int>(blockIdx.x * R / G), last = static_cast<int>((blockIdx.x + 1) * R / G);
    int64_t free_pages = p.free_capacity;
    if (p.free_count) {
        const int32_t live = *p.free_count;
        if (live < 0 || live > p.free_capacity) {
            if (blockIdx.x == 0 && tid == 0) set_status(p.status, TV_STATUS_BAD_REQUEST);
        }
        free_pages = live < 0 ? 0 : live < p.free_capacity ? live : p.free_capacity;
    }
    int64_t sum = 0;
    for (int r = tid; r < first; r += kThreads) sum += need_of(p, r).grow;
    int64_t base = 0;
    block_scan(sum, part, &base);
    if (R == 0 && tid == 0) *p.taken = 0;
    for (int at = first; at < last; at += kThreads) {
        const int r = at + tid;
        Need n = {0, 0, 0, false};
        if (r < last) n = need_of(p, r);
        int64_t total = 0;
        const int64_t end = base + block_scan(n.grow, part, &total);
        if (r < last) {
            const bool granted = n.pages <= p.width && end <= free_pages;
            const int32_t count = granted && n.pages > n.held ? static_cast<int32_t>(n.pages) : n.held;
            row_at[tid] = end - n.grow;
            row_held[tid] = n.held;
            row_count[tid] = count;
            p.counts[r] = count;
            if (n.bad) set_status(p.status, TV_STATUS_BAD_REQUEST);
            if (!granted && n.pages > n.held) set_status(p.status, TV_STATUS_NO_PAGES);
            // One request ends what is taken: the first that the list is short for, else the last.
            if (end > free_pages ? end - n.grow <= free_pages : r == R - 1) {
                *p.taken = static_cast<int32_t>(end > free_pages ? end - n.grow : end);
            }
        }
        __syncthreads();
        const int rows = last - at < kThreads ? last - at : kThreads;
        for (int i = 0; i < rows; ++i) {
            const int held = row_held[i], count = row_count[i];
            const int32_t* own = p.held + static_cast<int64_t>(at + i) * p.held_stride;
            const int32_t* pages = p.free_pages + row_at[i] - held;
            int32_t* out = p.tables + static_cast<int64_t>(at + i) * p.width;
            for (int j = tid; j < p.width; j += kThreads) {
                out[j] = j < held ? own[j] : j < count ? pages[j] : -1;
            }
        }
        __syncthreads();
        base += total;
    }
}

struct MapParams {
    const int32_t* cache_lens;
    const int32_t* query_lens;
    const int32_t* tables;     // [R, tables_stride] of tables_width pages, or null: the arena
    int64_t tables_stride;
    int32_t tables_width;
    const int32_t* arena;
    int32_t arena_pages;
    const int32_t* depths;     // per packed row, or null
    int32_t num_requests, block_size;
    int64_t num_blocks, total_rows;
    int32_t* cu;
    int32_t* request;
    int32_t* local;
    int64_t* positions;
    int64_t* slots;
    int32_t* status;
};

// Requests whose offsets a workgroup holds in LDS at a time.
constexpr int kRequestChunk = 4 * kThreads;

// Workgroup w maps rows [w*kThreads*RPT, ...): it scans the requests chunk by chunk until its rows
// are covered, and each row finds its request among a chunk's offsets by bisection.  Workgroup 0
// also writes the offsets.  Rows past the last request's are padding: request -1, slot -1.
template <int RPT>
__global__ void __launch_bounds__(kThreads)
slot_maps_kernel(const MapParams p) {
    __shared__ int64_t part[kWaves];
    __shared__ int64_t offset[kRequestChunk + 1];
    const int tid = threadIdx.x;
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kThreads * RPT;
    const int64_t row_end = row0 + kThreads * RPT < p.total_rows ? row0 + kThreads * RPT : p.total_rows;
    const bool lead = blockIdx.x == 0;
    const int32_t R = p.num_requests;
    int32_t bad = 0;
    int64_t base = 0;
    for (int chunk = 0; chunk < R && (lead || base < row_end); chunk += kRequestChunk) {
        const int n = R - chunk < kRequestChunk ? R - chunk : kRequestChunk;
        int64_t len[4], mine = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = 4 * tid + i;
            int32_t q = r < n ? p.query_lens[chunk + r] : 0;
            if (q < 0) {
                bad |= TV_STATUS_BAD_REQUEST;
                q = 0;
            }
            len[i] = q;
            mine += q;
        }
        int64_t total = 0;
        int64_t at = base + block_scan(mine, part, &total) - mine;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = 4 * tid + i;
            if (r < n) {
                offset[r] = at;
                if (lead) p.cu[chunk + r] = static_cast<int32_t>(at < 0x7fffffff ? at : 0x7fffffff);
            }
            at += len[i];
        }
        const int64_t end = base + total;
        if (tid == 0) offset[n] = end;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
            const int64_t row = row0 + i * kThreads + tid;
            if (row < base || row >= end || row >= row_end) continue;
            int lo = 0, hi = n;   // offset[lo] <= row < offset[hi]
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (offset[mid] <= row) lo = mid; else hi = mid;
            }
            const int r = chunk + lo;
            const int64_t l = row - offset[lo];
            const int64_t cached = p.cache_lens[r], at_pos = cached + l;
            const int64_t position = p.depths ? cached + p.depths[row] : at_pos;
            int64_t slot = -1;
            if (cached < 0 || position < 0) {
                bad |= TV_STATUS_BAD_POSITION;
            } else {
                const int64_t of = p.tables ? at_pos : row;
                const bool small = of <= 0x7fffffff;
                const uint32_t index = small ? static_cast<uint32_t>(of) / static_cast<uint32_t>(p.block_size) : 0;
                const int32_t inside = static_cast<int32_t>(static_cast<uint32_t>(of) - index * static_cast<uint32_t>(p.block_size));
                int64_t page = -1;
                if (small) {
                    if (p.tables) {
                        if (index < static_cast<uint32_t>(p.tables_width)) page = p.tables[r * p.tables_stride + index];
                    } else if (index < static_cast<uint32_t>(p.arena_pages)) {
                        page = p.arena[index];
                    }
                }
                if (page < 0 || page >= p.num_blocks) bad |= TV_STATUS_BAD_SLOT;
                else slot = page * p.block_size + inside;
            }
            p.request[row] = r;
            p.local[row] = static_cast<int32_t>(l);
            p.positions[row] = position < 0 ? 0 : position;
            p.slots[row] = slot;
        }
        __syncthreads();
        base = end;
    }
    // Every request is behind these rows, or there is none.
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
        const int64_t row = row0 + i * kThreads + tid;
        if (row >= base && row < row_end) {
            p.request[row] = -1;
            p.local[row] = 0;
            p.positions[row] = 0;
            p.slots[row] = -1;
        }
    }
    if (lead && tid == 0) {
        p.cu[R] = static_cast<int32_t>(base < 0x7fffffff ? base : 0x7fffffff);
        if (base > p.total_rows) bad |= TV_STATUS_BAD_REQUEST;
    }
    if (bad) set_status(p.status, bad);
}

}  // namespace
}  // namespace tv

using namespace tv;

extern "C" int tv_build_block_tables(const int32_t* lengths, const int32_t* held_tables, int64_t held_stride,
                                     int32_t held_width, const int32_t* held_counts, const int32_t* free_pages,
                                     const int32_t* free_count, int32_t free_capacity, int32_t num_requests,
                                     int32_t block_size, int32_t width, int32_t* tables, int32_t* counts,
                                     int32_t* taken, int32_t* status, void* stream) {
    clear_error();
    if (num_requests < 0 || block_size < 1 || width < 1 || free_capacity < 0 || held_width < 0 || held_width > width ||
        held_stride < 0) {
        return fail(TV_ERR_INVALID, "build_block_tables: invalid sizes (%d requests, block size %d, width %d, held width %d)",
                    num_requests, block_size, width, held_width);
    }
    if (!taken || (free_capacity > 0 && !free_pages)) return fail(TV_ERR_INVALID, "build_block_tables: null pointer");
    if (num_requests > 0 && (!lengths || !tables || !counts || (held_counts && held_width > 0 && !held_tables))) {
        return fail(TV_ERR_INVALID, "build_block_tables: null pointer");
    }
    TableParams p;
    p.lengths = lengths;
    p.held = held_tables;
    p.held_stride = held_stride;
    p.held_width = held_counts ? held_width : 0;
    p.held_counts = held_counts;
    p.free_pages = free_pages;
    p.free_count = free_count;
    p.free_capacity = free_capacity;
    p.num_requests = num_requests;
    p.block_size = block_size;
    p.width = width;
    p.tables = tables;
    p.counts = counts;
    p.taken = taken;
    p.status = status;
    // A workgroup per request while the sums that each recomputes stay small beside its row: 512 requests 5.7 us
    // against 6.5 with 256 workgroups, 2000 requests 13.0 against 19.4.
    const int groups = num_requests < 1 ? 1 : num_requests < 1024 ? num_requests : 1024;
    hipLaunchKernelGGL(block_tables_kernel, dim3(groups), dim3(kThreads), 0, as_stream(stream), p);
    return check_launch("build_block_tables");
}

extern "C" int tv_packed_slot_maps(const int32_t* cache_lens, const int32_t* query_lens, const int32_t* block_tables,
                                   int64_t table_stride, int32_t table_width, const int32_t* arena_pages,
                                   int32_t num_arena_pages, const int32_t* depths, int32_t num_requests,
                                   int64_t total_rows, int32_t block_size, int64_t num_blocks, int32_t* cu_seqlens,
                                   int32_t* query_to_request, int32_t* query_local_row, int64_t* positions,
                                   int64_t* slots, int32_t* status, void* stream) {
    clear_error();
    if (num_requests < 0 || total_rows < 0 || total_rows > 0x7fffffff || block_size < 1 || num_blocks < 1 ||
        table_width < 0 || table_stride < 0 || num_arena_pages < 0) {
        return fail(TV_ERR_INVALID, "packed_slot_maps: invalid sizes (%d requests, %lld rows, block size %d)", num_requests,
                    static_cast<long long>(total_rows), block_size);
    }
    if (!cu_seqlens || (num_requests > 0 && (!cache_lens || !query_lens)) ||
        (total_rows > 0 && (!query_to_request || !query_local_row || !positions || !slots))) {
        return fail(TV_ERR_INVALID, "packed_slot_maps: null pointer");
    }
    if (num_requests > 0 && total_rows > 0 && (block_tables != nullptr) == (arena_pages != nullptr)) {
        return fail(TV_ERR_INVALID, "packed_slot_maps: needs either block tables or an arena");
    }
    MapParams p;
    p.cache_lens = cache_lens;
    p.query_lens = query_lens;
    p.tables = block_tables;
    p.tables_stride = table_stride;
    p.tables_width = table_width;
    p.arena = arena_pages;
    p.arena_pages = arena_pages ? num_arena_pages : 0;
    p.depths = depths;
    p.num_requests = num_requests;
    p.block_size = block_size;
    p.num_blocks = num_blocks;
    p.total_rows = total_rows;
    p.cu = cu_seqlens;
    p.request = query_to_request;
    p.local = query_local_row;
    p.positions = positions;
    p.slots = slots;
    p.status = status;
    // A row a thread while that gives the chip no more workgroups than it holds, then four, which share a
    // workgroup's scan.  One against four: 130 thousand rows of 61 requests 4.7 / 6.4 us, 508 thousand of 250 7.9 / 8.6, 531
    // thousand of 61 8.0 / 8.7, 576 thousand of 16 7.8 / 8.0, 608 thousand of 4 7.8 / 7.5, a million of one 9.6 / 8.3, of
    // 1000 13.6 / 11.8.  The two meet near 600 thousand rows: from the border, 262 thousand, up to there four cost up to 9 %.
    const int64_t one = (total_rows + kThreads - 1) / kThreads;
    if (one <= 1024) {
        hipLaunchKernelGGL(slot_maps_kernel<1>, dim3(one < 1 ? 1 : one), dim3(kThreads), 0, as_stream(stream), p);
    } else {
        hipLaunchKernelGGL(slot_maps_kernel<4>, dim3((one + 3) / 4), dim3(kThreads), 0, as_stream(stream), p);
    }
    return check_launch("packed_slot_maps");
}
