// A paged cache's block tables and slots, from the requests' lengths, on the device.
//
//   block_tables  new_r = max(0, ceil(length_r / block) - held_r); the scan of new_r says which
//                 ids of the free pool a request takes: table[r][held_r + j] = pool[scan_r + j]
//   slot_map      the scan of fresh_r packs the requests' new tokens; token i of request r
//                 at position p = start_r + i has slot table[r][p / block] * block + p % block
//
// Both turn one number per request into a ragged list: a scan over the requests, then a
// search of the scan per list entry. The lists are a few megabytes at most, so the calls
// are bound by the launch and by one chain of dependent reads. Up to kScanInBlock
// requests every CTA scans all of them itself into shared memory -- one launch, no wait on
// another CTA; past it the scan is a kernel of its own (one CTA) that leaves it in scratch.
#include "sequences.cuh"

#include <algorithm>

#define EB_API extern "C" __attribute__((visibility("default")))

namespace eb {
namespace {

constexpr int kThreads = 1024;
constexpr uint32_t kItems = 8;                           // requests a thread scans
constexpr uint32_t kScanInBlock = kThreads * kItems;     // 8192
constexpr uint32_t kWarps = kThreads / 32;

struct PagedArgs {
    uint32_t requests;
    int64_t width, tableStride;
    int64_t room;  // width * block: the positions a row of the table covers
    FastDiv perBlock;
    int32_t* table;
    const uint8_t* terminated;
    const void* lengths;
    const int32_t* held;
    const int32_t* pool;
    const uint32_t* count;
    int64_t poolSize;
    uint8_t* used;
    int64_t usedSize;
    int32_t* blocks;
    uint32_t* cells;
    const void* start;
    const void* fresh;
    uint32_t capacity;
    void* slots;
    void* positions;
    int32_t* tokenRequests;
    int32_t* offsets;
    uint32_t* upto;  // scratch: the inclusive scan (more than kScanInBlock requests)
};

template <class Len>
__device__ __forceinline__ int64_t lengthAt(const void* p, uint32_t r)
{
    const int64_t v = int64_t(__ldg(reinterpret_cast<const Len*>(p) + r));
    return v < 0 ? 0 : v;
}

// ------------------------------------------------------------------ what each request adds

/** A request's state: its reads do not wait for one another. */
struct Blocks {
    uint32_t held;   // clipped to the row
    uint32_t need;   // width + 1 where the row cannot hold them
    bool live;
    bool wide;       // more than the row holds

    template <class Len>
    __device__ __forceinline__ void read(const PagedArgs& a, uint32_t r)
    {
        const uint8_t ended = a.terminated != nullptr ? __ldg(a.terminated + r) : uint8_t(0);
        const int64_t length = lengthAt<Len>(a.lengths, r);
        const int64_t h = __ldg(a.held + r);
        held = uint32_t(h < 0 ? 0 : (h < a.width ? h : a.width));
        live = ended == 0;
        wide = live && length > a.room;
        const uint32_t l = uint32_t(length < a.room ? length : a.room);
        const uint32_t whole = a.perBlock(l);
        need = live ? whole + (whole * a.perBlock.d != l ? 1u : 0u) : 0u;
    }
    /** The blocks it asks for. */
    __device__ __forceinline__ uint32_t adds() const { return wide || need <= held ? 0u : need - held; }
};

struct Tokens {
    uint32_t fresh;

    template <class Len>
    __device__ __forceinline__ void read(const PagedArgs& a, uint32_t r)
    {
        const uint8_t ended = a.terminated != nullptr ? __ldg(a.terminated + r) : uint8_t(0);
        const int64_t f = lengthAt<Len>(a.fresh, r);
        fresh = ended != 0 ? 0u : uint32_t(f < 0x7fffffffll ? f : 0x7fffffffll);
    }
    __device__ __forceinline__ uint32_t adds() const { return fresh; }
};

// ------------------------------------------------------------------ the scan

/** Sums past this read as this: no pool and no list is as long. */
constexpr uint64_t kMost = 0x7fffffffull;

/** Requests [from, from + kScanInBlock): thread t reads ``items`` neighbours from ``t * items`` on
 *  (as few as cover them), all at once; their inclusive sums on top of ``carry`` go to
 *  ``upto``. Returns the new carry. */
template <class What, class Len>
__device__ __forceinline__ uint64_t scanBlock(const PagedArgs& a, uint32_t from, uint64_t carry, What (&what)[kItems],
    uint32_t* upto, uint64_t* scratch)
{
    const uint32_t m = min(a.requests - from, kScanInBlock);
    const uint32_t items = (m + kThreads - 1) / kThreads, first = threadIdx.x * items;
#pragma unroll
    for (uint32_t k = 0; k < kItems; ++k)
        if (k < items && first + k < m)
            what[k].template read<Len>(a, from + first + k);
    uint64_t mine = 0;
#pragma unroll
    for (uint32_t k = 0; k < kItems; ++k)
        if (k < items && first + k < m)
            mine += what[k].adds();
    uint64_t total = 0;
    uint64_t sum = carry + blockExclusiveSum(mine, total, scratch);
#pragma unroll
    for (uint32_t k = 0; k < kItems; ++k)
        if (k < items && first + k < m) {
            sum += what[k].adds();
            upto[first + k] = uint32_t(sum < kMost ? sum : kMost);
        }
    __syncthreads();
    return carry + total;
}

/** The scan of any number of requests by one CTA, into scratch. */
template <class What, class Len>
__global__ __launch_bounds__(kThreads) void scanKernel(PagedArgs a)
{
    __shared__ uint32_t upto[kScanInBlock];
    __shared__ uint64_t scratch[33];
    letNextKernelStart();
    if (threadIdx.x == 0 && a.cells != nullptr)
        a.cells[1] = 0;
    uint64_t carry = 0;
    for (uint32_t from = 0; from < a.requests; from += kScanInBlock) {
        What what[kItems];
        carry = scanBlock<What, Len>(a, from, carry, what, upto, scratch);
        for (uint32_t i = threadIdx.x; i < min(a.requests - from, kScanInBlock); i += kThreads)
            a.upto[from + i] = upto[i];
        __syncthreads();
    }
}

/** The first request from ``low`` on whose inclusive sum is above ``q`` (the requests' number
 *  if none is). */
__device__ __forceinline__ uint32_t requestOf(const uint32_t* upto, uint32_t requests, uint32_t q, uint32_t low = 0)
{
    uint32_t high = requests;
    while (low < high) {
        const uint32_t mid = (low + high) >> 1;
        if (upto[mid] > q)
            high = mid;
        else
            low = mid + 1;
    }
    return low;
}

/** The same from a request ``r`` at or before it: mostly that one or the next; a row of requests
 *  that add nothing is searched over. */
__device__ __forceinline__ uint32_t requestFrom(const uint32_t* upto, uint32_t requests, uint32_t q, uint32_t r)
{
    if (r < requests && upto[r] <= q && ++r < requests && upto[r] <= q)
        r = requestOf(upto, requests, q, r + 1u);
    return r;
}

// ------------------------------------------------------------------ block tables

constexpr uint32_t kEntries = 128;  // of the pool's front per warp and step: one search for all of them

/** Every CTA scans the requests (or reads the scan from scratch) and takes its share of the
 *  lists; the last one also writes what each request holds and the cells. */
template <class Len, bool InBlock>
__global__ __launch_bounds__(kThreads) void blockTablesKernel(PagedArgs a)
{
    __shared__ uint32_t sUpto[InBlock ? kScanInBlock : 1];
    __shared__ uint32_t sGone[InBlock ? kScanInBlock / 32 : 1];  // a bit per terminated request
    __shared__ uint64_t scratch[33];
    __shared__ uint32_t sShort;
    const uint32_t* upto = InBlock ? sUpto : a.upto;
    const bool returns = a.used != nullptr && a.terminated != nullptr;
    const uint32_t lane = threadIdx.x & 31u, warp = blockIdx.x * kWarps + (threadIdx.x >> 5),
                   warps = gridDim.x * kWarps;
    if constexpr (!InBlock)
        waitForKernelBefore();
    const uint32_t given = __ldg(a.count);
    const uint32_t available = uint64_t(given) > uint64_t(a.poolSize) ? 0u : given;
    if (threadIdx.x == 0)
        sShort = 0;
    Blocks what[kItems];
    if constexpr (InBlock) {
        for (uint32_t i = threadIdx.x; returns && i < (a.requests + 31) / 32; i += kThreads)
            sGone[i] = 0;
        (void)scanBlock<Blocks, Len>(a, 0, 0, what, sUpto, scratch);
    } else {
        __syncthreads();
    }
    // the sums never fall, so the requests that fit with new blocks are the first ones, up to
    // the last sum within the pool
    const uint32_t fitting = requestOf(upto, a.requests, available);
    const uint32_t taken = fitting == 0 ? 0u : upto[fitting - 1];

    const bool last = blockIdx.x == gridDim.x - 1;
    uint32_t missed = 0;
    auto settle = [&](const Blocks& w, uint32_t r) {
        const bool fits = !w.wide && (w.need <= w.held || upto[r] <= available);
        a.blocks[r] = int32_t(!w.live ? 0u : (fits && w.need > w.held ? w.need : w.held));
        missed += fits ? 0u : 1u;
    };
    if constexpr (InBlock) {
        const uint32_t items = (a.requests + kThreads - 1) / kThreads, first = threadIdx.x * items;
#pragma unroll
        for (uint32_t k = 0; k < kItems; ++k) {
            if (k < items && first + k < a.requests) {
                if (last)
                    settle(what[k], first + k);
                if (returns && !what[k].live && what[k].held > 0)
                    atomicOr(sGone + ((first + k) >> 5), 1u << ((first + k) & 31u));
            }
        }
        __syncthreads();
    } else {
        for (uint32_t r = blockIdx.x * kThreads + threadIdx.x; r < a.requests; r += gridDim.x * kThreads) {
            Blocks w;
            w.read<Len>(a, r);
            settle(w, r);
        }
    }

    // the blocks of terminated requests, a warp per request
    if (returns) {
        for (uint32_t r = warp; r < a.requests; r += warps) {
            if (InBlock ? ((sGone[r >> 5] >> (r & 31u)) & 1u) == 0 : __ldg(a.terminated + r) == 0)
                continue;
            const int64_t h = __ldg(a.held + r);
            const int64_t held = h < a.width ? h : a.width;
            const int32_t* row = a.table + int64_t(r) * a.tableStride;
#pragma unroll 4
            for (int64_t j = lane; j < held; j += 32) {
                const int64_t id = row[j];
                if (id >= 0 && id < a.usedSize)
                    a.used[id] = 0;
            }
        }
    }

    // the front of the pool
    for (uint64_t q0 = uint64_t(warp) * kEntries; q0 < taken; q0 += uint64_t(warps) * kEntries) {
        const uint32_t r0 = requestOf(upto, a.requests, uint32_t(q0));
        int32_t id[kEntries / 32];
#pragma unroll
        for (uint32_t k = 0; k < kEntries / 32; ++k) {
            const uint64_t q = q0 + 32u * k + lane;
            id[k] = q < taken ? __ldg(a.pool + q) : -1;
        }
        uint32_t r = r0;
#pragma unroll
        for (uint32_t k = 0; k < kEntries / 32; ++k) {
            const uint64_t q = q0 + 32u * k + lane;
            if (q >= taken)
                break;
            r = requestFrom(upto, a.requests, uint32_t(q), r);
            const uint32_t before = r == 0 ? 0u : upto[r - 1];
            const int64_t h = __ldg(a.held + r);
            a.table[int64_t(r) * a.tableStride + (h < 0 ? 0 : h) + (uint32_t(q) - before)] = id[k];
            if (a.used != nullptr && id[k] >= 0 && int64_t(id[k]) < a.usedSize)
                a.used[id[k]] = 1;
        }
    }

    if (InBlock && !last)
        return;
    missed = warpSum(missed);
    if (lane == 0 && missed != 0)
        atomicAdd(&sShort, missed);
    __syncthreads();
    if (threadIdx.x == 0) {
        if (last)
            a.cells[0] = taken;
        if (InBlock)
            a.cells[1] = sShort;
        else if (sShort != 0)  // zeroed by the scan
            atomicAdd(a.cells + 1, sShort);
    }
}

// ------------------------------------------------------------------ slots

constexpr uint32_t kTokens = 4;  // neighbouring tokens per thread and step

template <class Len, class Slot, bool InBlock>
__global__ __launch_bounds__(kThreads) void slotMapKernel(PagedArgs a)
{
    __shared__ uint32_t sUpto[InBlock ? kScanInBlock : 1];
    __shared__ uint64_t scratch[33];
    const uint32_t* upto = InBlock ? sUpto : a.upto;
    if constexpr (InBlock) {
        Tokens what[kItems];
        (void)scanBlock<Tokens, Len>(a, 0, 0, what, sUpto, scratch);
    } else {
        waitForKernelBefore();
    }
    const uint32_t lane = threadIdx.x & 31u, warp = blockIdx.x * kWarps + (threadIdx.x >> 5),
                   warps = gridDim.x * kWarps;
    for (uint64_t w0 = uint64_t(warp) * 32u * kTokens; w0 < a.capacity; w0 += uint64_t(warps) * 32u * kTokens) {
        const uint32_t r0 = requestOf(upto, a.requests, uint32_t(w0));  // one search for the warp's tokens
        const uint64_t q0 = w0 + lane * kTokens;
        uint32_t r = r0;
        if (q0 < a.capacity)
            r = requestFrom(upto, a.requests, uint32_t(q0), r);
        Pack<Slot, kTokens> slot;
        Pack<Len, kTokens> position;
        Pack<int32_t, kTokens> request;
#pragma unroll
        for (uint32_t k = 0; k < kTokens; ++k) {
            const uint32_t q = uint32_t(q0) + k;
            r = requestFrom(upto, a.requests, q, r);
            slot.e[k] = Slot(-1);
            position.e[k] = 0;
            request.e[k] = -1;
            if (r < a.requests) {
                const uint32_t before = r == 0 ? 0u : upto[r - 1];
                const uint64_t p = uint64_t(lengthAt<Len>(a.start, r)) + (q - before);
                position.e[k] = Len(p);
                request.e[k] = int32_t(r);
                if (p < uint64_t(a.room)) {
                    const uint32_t b = a.perBlock(uint32_t(p));
                    const int64_t id = __ldg(a.table + int64_t(r) * a.tableStride + b);
                    const int64_t at = id * a.perBlock.d + (uint32_t(p) - b * a.perBlock.d);
                    if (id >= 0 && int64_t(Slot(at)) == at)
                        slot.e[k] = Slot(at);
                }
            }
        }
        if (q0 + kTokens <= a.capacity) {
            *reinterpret_cast<Pack<Slot, kTokens>*>(reinterpret_cast<Slot*>(a.slots) + q0) = slot;
            *reinterpret_cast<Pack<Len, kTokens>*>(reinterpret_cast<Len*>(a.positions) + q0) = position;
            *reinterpret_cast<Pack<int32_t, kTokens>*>(a.tokenRequests + q0) = request;
        } else {
#pragma unroll
            for (uint32_t k = 0; k < kTokens; ++k) {
                if (q0 + k < a.capacity) {
                    reinterpret_cast<Slot*>(a.slots)[q0 + k] = slot.e[k];
                    reinterpret_cast<Len*>(a.positions)[q0 + k] = position.e[k];
                    a.tokenRequests[q0 + k] = request.e[k];
                }
            }
        }
    }
    for (uint32_t r = blockIdx.x * kThreads + threadIdx.x; r <= a.requests; r += gridDim.x * kThreads)
        a.offsets[r] = r == 0 ? 0 : int32_t(upto[r - 1]);
}

// ------------------------------------------------------------------ host side

PagedArgs pagedArgs(const eagle_b200_paged_desc& d, const char* who)
{
    const std::string w(who);
    (void)indexBytes(d.length_type, who);
    if (d.reserved0 != 0)
        invalid(w + ": reserved0 must be zero");
    if (d.requests < 0 || d.requests > (1ll << 20))
        invalid(w + ": requests must lie in [0, 2^20]");
    if (d.block < 1 || d.width < 0 || d.block > 0x7fffffffll || d.width > 0x7fffffffll / d.block)
        invalid(w + ": block must be at least 1 and width * block at most 2^31 - 1");
    if (d.requests > 1 && d.table_stride < d.width)
        invalid(w + ": the table's rows overlap (table_stride below width)");
    PagedArgs a{};
    a.requests = uint32_t(d.requests);
    a.width = d.width;
    a.tableStride = d.table_stride;
    a.room = d.width * d.block;
    a.perBlock = FastDiv(uint32_t(d.block));
    a.table = reinterpret_cast<int32_t*>(d.table);
    a.terminated = reinterpret_cast<const uint8_t*>(d.terminated);
    a.upto = reinterpret_cast<uint32_t*>(d.scratch);
    return a;
}

int64_t pagedScratch(const eagle_b200_paged_desc& d) { return d.requests > int64_t(kScanInBlock) ? d.requests * 4 : 16; }

template <class F>
void withLength(uint32_t type, F&& f)
{
    if (type == EAGLE_B200_TYPE_I32)
        f(int32_t{});
    else
        f(int64_t{});
}

template <class What, class Len>
void launchScan(const PagedArgs& a, cudaStream_t s, const char* who)
{
    scanKernel<What, Len><<<1, kThreads, 0, s>>>(a);
    launchCheck(who);
}

}  // namespace
}  // namespace eb

using namespace eb;

EB_API eagle_backend_status eagle_backend_x_b200_block_tables(eagle_b200_paged_desc* desc)
{
    return guarded([&] {
        const char* who = "eagle_backend_x_b200_block_tables";
        const eagle_b200_paged_desc d = readDesc(desc, 0u, who);
        if (desc->struct_size < sizeof d)
            invalid(std::string(who) + ": struct_size too small for the query's answer");
        PagedArgs a = pagedArgs(d, who);
        if (d.pool_size < 0 || d.pool_size > 0x7ffffffell || d.used_size < 0)
            invalid(std::string(who) + ": pool_size must lie in [0, 2^31 - 2] and used_size not be negative");
        if (d.scratch == 0) {
            desc->scratch_bytes = pagedScratch(d);
            return;
        }
        requireAddress(d.scratch, 16, who, "scratch");
        requireAddress(d.count, 4, who, "count");
        requireAddress(d.cells, 4, who, "cells");
        if (d.pool_size > 0)
            requireAddress(d.pool, 4, who, "pool");
        const int64_t bytes = indexBytes(d.length_type, who);
        if (d.requests > 0) {
            requireAddress(d.lengths, uint64_t(bytes), who, "lengths");
            requireAddress(d.held, 4, who, "held");
            requireAddress(d.blocks, 4, who, "blocks");
            if (d.blocks == d.held)
                invalid(std::string(who) + ": blocks may not be held: every CTA reads all of held");
            if (d.width > 0)
                requireAddress(d.table, 4, who, "table");
        }
        requireDevice();
        DeviceScope scope(resolveDevice(d.device, d.cells));
        a.lengths = reinterpret_cast<const void*>(d.lengths);
        a.held = reinterpret_cast<const int32_t*>(d.held);
        a.pool = reinterpret_cast<const int32_t*>(d.pool);
        a.count = reinterpret_cast<const uint32_t*>(d.count);
        a.poolSize = d.pool_size;
        a.used = reinterpret_cast<uint8_t*>(d.used);
        a.usedSize = d.used_size;
        a.blocks = reinterpret_cast<int32_t*>(d.blocks);
        a.cells = reinterpret_cast<uint32_t*>(d.cells);
        const cudaStream_t s = seamStream(d.stream);
        // the entries the call can write at most, an SM per CTA
        const int64_t most = std::max(std::min(d.pool_size, d.requests * d.width), d.requests);
        const int64_t grid = std::max<int64_t>(1, std::min<int64_t>(smCount(), (most + kWarps * kEntries - 1) / (kWarps * kEntries)));
        withLength(d.length_type, [&](auto len) {
            using Len = decltype(len);
            if (d.requests <= int64_t(kScanInBlock)) {
                blockTablesKernel<Len, true><<<unsigned(grid), kThreads, 0, s>>>(a);
                launchCheck(who);
            } else {
                launchScan<Blocks, Len>(a, s, who);
                launchBehind(blockTablesKernel<Len, false>, unsigned(grid), kThreads, 0, s, a, who);
            }
        });
    });
}

EB_API eagle_backend_status eagle_backend_x_b200_slot_map(eagle_b200_paged_desc* desc)
{
    return guarded([&] {
        const char* who = "eagle_backend_x_b200_slot_map";
        const eagle_b200_paged_desc d = readDesc(desc, 0u, who);
        if (desc->struct_size < sizeof d)
            invalid(std::string(who) + ": struct_size too small for the query's answer");
        PagedArgs a = pagedArgs(d, who);
        (void)indexBytes(d.slot_type, who);
        if (d.capacity < 0 || d.capacity > 0x7ffffff0ll)
            invalid(std::string(who) + ": capacity must lie in [0, 2^31 - 16]");
        if (d.scratch == 0) {
            desc->scratch_bytes = pagedScratch(d);
            return;
        }
        requireAddress(d.scratch, 16, who, "scratch");
        requireAddress(d.offsets, 4, who, "offsets");
        if (d.capacity > 0) {
            requireAddress(d.slots, 16, who, "slots");
            requireAddress(d.positions, 16, who, "positions");
            requireAddress(d.token_requests, 16, who, "token_requests");
        }
        const int64_t bytes = indexBytes(d.length_type, who);
        if (d.requests > 0) {
            requireAddress(d.start, uint64_t(bytes), who, "start");
            requireAddress(d.fresh, uint64_t(bytes), who, "fresh");
            if (d.width > 0)
                requireAddress(d.table, 4, who, "table");
        }
        requireDevice();
        DeviceScope scope(resolveDevice(d.device, d.offsets));
        a.start = reinterpret_cast<const void*>(d.start);
        a.fresh = reinterpret_cast<const void*>(d.fresh);
        a.capacity = uint32_t(d.capacity);
        a.slots = reinterpret_cast<void*>(d.slots);
        a.positions = reinterpret_cast<void*>(d.positions);
        a.tokenRequests = reinterpret_cast<int32_t*>(d.token_requests);
        a.offsets = reinterpret_cast<int32_t*>(d.offsets);
        const cudaStream_t s = seamStream(d.stream);
        const int64_t per = int64_t(kThreads) * kTokens;
        const int64_t grid = std::max<int64_t>(1, std::min<int64_t>(2 * smCount(), (d.capacity + per - 1) / per));
        withLength(d.length_type, [&](auto len) {
            withLength(d.slot_type, [&](auto slot) {
                using Len = decltype(len);
                using Slot = decltype(slot);
                if (d.requests <= int64_t(kScanInBlock)) {
                    slotMapKernel<Len, Slot, true><<<unsigned(grid), kThreads, 0, s>>>(a);
                    launchCheck(who);
                } else {
                    launchScan<Tokens, Len>(a, s, who);
                    launchBehind(slotMapKernel<Len, Slot, false>, unsigned(grid), kThreads, 0, s, a, who);
                }
            });
        });
    });
}
