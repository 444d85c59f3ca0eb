// A paged cache's block tables and slots, from the requests' lengths, on the device.
//
//   block_tables  new_r = max(0, ceil(length_r / block) - held_r); the scan of new_r says which
//                 ids of the free pool a request takes: table[r][held_r + j] = pool[scan_r + j]
//   slot_map      the scan of fresh_r packs the requests' new tokens; token i of request r
//                 at position p = start_r + i has slot table[r][p / block] * block + p % block
//
// Both turn one number per request into a ragged list by a scan over the requests. The lists
// are a few megabytes at most, so the calls are bound by the launch and by one chain of
// dependent reads. Up to kScanInBlock requests every CTA scans all of them itself into shared
// memory: one launch, no wait on another CTA. Past it the scan is a kernel of its own, of one
// CTA, that leaves it in scratch: 300 CTAs that each read 8191 requests took 7 us over that,
// one CTA and the start of a second kernel 4.
#include "sequences.cuh"

#include <algorithm>

#define EB_API extern "C" __attribute__((visibility("default")))

namespace eb {
namespace {

constexpr int kThreads = 512, kItems = 4;            // requests a thread scans where every CTA scans
constexpr int kScanThreads = 1024, kScanItems = 8;   // where one does
constexpr uint32_t kScanInBlock = kThreads * kItems;         // 2048
constexpr uint32_t kScanAtOnce = kScanThreads * kScanItems;  // 8192
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
    const int64_t v = int64_t(reinterpret_cast<const Len*>(p)[r]);
    return v < 0 ? 0 : v;
}

// ------------------------------------------------------------------ what each request adds

/** A request's blocks, from what is read of it (Raw: so that the reads of several are in flight
 *  together). */
struct Blocks {
    uint32_t held;  // clipped to the row
    uint32_t need;  // width + 1 where the row cannot hold them
    bool live;

    using Kept = uint2;  // {held, need}, the highest bit of held set where it is terminated
    template <class Len>
    struct Raw {
        Len length;
        int32_t held;
        uint8_t ended;
        __device__ __forceinline__ void read(const PagedArgs& a, uint32_t r)
        {
            ended = a.terminated != nullptr ? a.terminated[r] : uint8_t(0);
            length = reinterpret_cast<const Len*>(a.lengths)[r];
            held = a.held[r];
        }
    };
    template <class Len>
    __device__ __forceinline__ void take(const PagedArgs& a, const Raw<Len>& raw)
    {
        const int64_t length = raw.length < 0 ? 0 : int64_t(raw.length), h = raw.held;
        held = uint32_t(h < 0 ? 0 : (h < a.width ? h : a.width));
        live = raw.ended == 0;
        const uint32_t l = uint32_t(length < a.room ? length : a.room);
        const uint32_t whole = a.perBlock(l);
        need = length > a.room ? uint32_t(a.width) + 1u : whole + (whole * a.perBlock.d != l ? 1u : 0u);
        need = live ? need : 0u;
    }
    /** The blocks it asks for. */
    __device__ __forceinline__ uint32_t adds(const PagedArgs& a) const
    {
        return need > uint32_t(a.width) || need <= held ? 0u : need - held;
    }
    __device__ __forceinline__ Kept kept() const { return make_uint2(held | (live ? 0u : 0x80000000u), need); }
    static __device__ __forceinline__ Blocks of(Kept k)
    {
        Blocks b;
        b.held = k.x & 0x7fffffffu;
        b.live = (k.x >> 31) == 0;
        b.need = k.y;
        return b;
    }
};

/** A request's new tokens. */
struct Tokens {
    uint32_t fresh;
    int64_t start;

    using Kept = int64_t;
    template <class Len>
    struct Raw {
        Len fresh, start;
        uint8_t ended;
        __device__ __forceinline__ void read(const PagedArgs& a, uint32_t r)
        {
            ended = a.terminated != nullptr ? a.terminated[r] : uint8_t(0);
            fresh = reinterpret_cast<const Len*>(a.fresh)[r];
            start = reinterpret_cast<const Len*>(a.start)[r];
        }
    };
    template <class Len>
    __device__ __forceinline__ void take(const PagedArgs&, const Raw<Len>& raw)
    {
        const int64_t f = raw.fresh;
        start = raw.start < 0 ? 0 : int64_t(raw.start);
        fresh = raw.ended != 0 || f < 0 ? 0u : uint32_t(f < 0x7fffffffll ? f : 0x7fffffffll);
    }
    __device__ __forceinline__ uint32_t adds(const PagedArgs&) const { return fresh; }
    __device__ __forceinline__ Kept kept() const { return start; }
};

// ------------------------------------------------------------------ the scan

/** Sums past this read as this: no pool and no list is as long. So 32 bits hold them. */
constexpr uint32_t kMost = 0x7fffffffu;

__device__ __forceinline__ uint32_t addUpTo(uint32_t a, uint32_t b) { return min(a + b, kMost); }  // both at most kMost

__device__ __forceinline__ uint32_t warpInclusive(uint32_t v)
{
    const uint32_t lane = threadIdx.x & 31u;
#pragma unroll
    for (uint32_t off = 1; off < 32; off <<= 1) {
        const uint32_t o = __shfl_up_sync(kFull, v, off);
        if (lane >= off)
            v = addUpTo(v, o);
    }
    return v;
}

constexpr uint32_t kMaxSegments = kScanItems * (kScanThreads / 32);

/** Requests [from, from + Threads * Items), Threads neighbours at a time (a thread reading its own
 *  neighbours instead took 13 us for 8191 requests), all read at once: their inclusive sums on
 *  top of ``carry`` go to ``upto`` and what they keep to ``kept``. Every warp scans its 32 of each
 *  step, the first one those segments' sums. Returns the new carry. ``segment`` is kMaxSegments
 *  + 1 words of shared memory. */
template <int Threads, int Items, class What, class Len>
__device__ __forceinline__ uint32_t scanBlock(const PagedArgs& a, uint32_t from, uint32_t carry, uint32_t* upto,
    typename What::Kept* kept, uint32_t* segment)
{
    constexpr uint32_t kOwn = Threads / 32;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const uint32_t m = min(a.requests - from, uint32_t(Threads * Items));
    const uint32_t items = (m + Threads - 1) / Threads;
    typename What::template Raw<Len> raw[Items];
    uint32_t sum[Items];
#pragma unroll
    for (uint32_t k = 0; k < uint32_t(Items); ++k)
        if (k < items)
            raw[k].read(a, from + min(k * Threads + threadIdx.x, m - 1u));
#pragma unroll
    for (uint32_t k = 0; k < uint32_t(Items); ++k) {
        if (k < items) {
            const uint32_t i = k * Threads + threadIdx.x;
            What what;
            what.template take<Len>(a, raw[k]);
            sum[k] = i < m ? what.adds(a) : 0u;
            if (kept != nullptr && i < m)
                kept[i] = what.kept();
            sum[k] = warpInclusive(sum[k]);
            if (lane == 31)
                segment[k * kOwn + warp] = sum[k];
        }
    }
    __syncthreads();
    if (warp == 0) {
        constexpr uint32_t kEach = Items * kOwn / 32;  // segments a lane adds up
        uint32_t mine[kEach], total = 0;
#pragma unroll
        for (uint32_t e = 0; e < kEach; ++e) {
            mine[e] = total;
            const uint32_t s = lane * kEach + e;
            total = addUpTo(total, s < items * kOwn ? segment[s] : 0u);
        }
        const uint32_t through = warpInclusive(total);
        const uint32_t before = __shfl_up_sync(kFull, through, 1);
        __syncwarp();
#pragma unroll
        for (uint32_t e = 0; e < kEach; ++e)
            segment[lane * kEach + e] = addUpTo(carry, addUpTo(lane == 0 ? 0u : before, mine[e]));
        if (lane == 31)
            segment[kMaxSegments] = addUpTo(carry, through);
    }
    __syncthreads();
#pragma unroll
    for (uint32_t k = 0; k < uint32_t(Items); ++k)
        if (k < items && k * Threads + threadIdx.x < m)
            upto[k * Threads + threadIdx.x] = addUpTo(segment[k * kOwn + warp], sum[k]);
    __syncthreads();
    return segment[kMaxSegments];
}

/** The scan of any number of requests by one CTA, into scratch. */
template <class What, class Len>
__global__ __launch_bounds__(kScanThreads) void scanKernel(PagedArgs a)
{
    __shared__ uint32_t upto[kScanAtOnce];
    __shared__ uint32_t segment[kMaxSegments + 1];
    letNextKernelStart();
    waitForKernelBefore();
    if (threadIdx.x == 0 && a.cells != nullptr)
        a.cells[1] = 0;
    uint32_t carry = 0;
    for (uint32_t from = 0; from < a.requests; from += kScanAtOnce) {
        carry = scanBlock<kScanThreads, kScanItems, What, Len>(a, from, carry, upto, nullptr, segment);
        for (uint32_t i = threadIdx.x; i < min(a.requests - from, kScanAtOnce); i += kScanThreads)
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

/** A warp, or several where there are more warps than requests, takes one request's blocks: those
 *  it gets are copied from the pool, and those a terminated one gives back are cleared. (One
 *  search per entry of the pool's front instead, 100 instructions per 32 entries against 15,
 *  took twice as long.) The requests are spread over the CTAs for what they hold now, too. */
template <class Len, bool InBlock>
__global__ __launch_bounds__(kThreads) void blockTablesKernel(PagedArgs a)
{
    __shared__ uint32_t segment[InBlock ? kMaxSegments + 1 : 1];
    __shared__ uint32_t sShort;
    __shared__ Blocks::Kept kept[InBlock ? kScanInBlock : 1];
    __shared__ uint32_t sUpto[InBlock ? kScanInBlock : 1];
    const uint32_t* upto = InBlock ? sUpto : a.upto;
    const uint32_t lane = threadIdx.x & 31u, warp = blockIdx.x * kWarps + (threadIdx.x >> 5),
                   warps = gridDim.x * kWarps;
    letNextKernelStart();
    waitForKernelBefore();
    const uint32_t given = *a.count;
    const uint32_t available = uint64_t(given) > uint64_t(a.poolSize) ? 0u : given;
    if (threadIdx.x == 0)
        sShort = 0;
    if constexpr (InBlock)
        (void)scanBlock<kThreads, kItems, Blocks, Len>(a, 0, 0, sUpto, kept, segment);
    else
        __syncthreads();
    auto request = [&](uint32_t r) {
        Blocks b;
        if constexpr (InBlock) {
            b = Blocks::of(kept[r]);
        } else {
            Blocks::Raw<Len> raw;
            raw.read(a, r);
            b.take<Len>(a, raw);
        }
        return b;
    };

    constexpr int kAhead = InBlock ? 4 : 8;
    constexpr uint32_t kEntries = 32u * kAhead;
    // ``share`` warps to a request where there are as many
    const uint32_t share = a.requests == 0 ? 0u : max(1u, warps / a.requests);
    const uint32_t part = share > 1 ? warp / a.requests : 0u;
    for (uint32_t r = warp - part * a.requests; r < a.requests && part < share; r += warps) {
        const Blocks b = request(r);
        int32_t* row = a.table + int64_t(r) * a.tableStride;
        if (b.live) {
            const uint32_t adds = b.adds(a), sum = upto[r];
            if (sum > available)
                continue;
            const int32_t* from = a.pool + (sum - adds);
            for (uint32_t j = part * kEntries + lane; j < adds; j += share * kEntries) {
                int32_t id[kAhead];
#pragma unroll
                for (int u = 0; u < kAhead; ++u)
                    id[u] = j + 32u * u < adds ? from[j + 32u * u] : -1;
#pragma unroll
                for (int u = 0; u < kAhead; ++u) {
                    if (j + 32u * u < adds) {
                        row[b.held + j + 32u * u] = id[u];
                        if (a.used != nullptr && id[u] >= 0 && int64_t(id[u]) < a.usedSize)
                            a.used[id[u]] = 1;
                    }
                }
            }
        } else if (a.used != nullptr) {
            for (uint32_t j = part * kEntries + lane; j < b.held; j += share * kEntries) {
                int32_t id[kAhead];
#pragma unroll
                for (int u = 0; u < kAhead; ++u)
                    id[u] = j + 32u * u < b.held ? row[j + 32u * u] : -1;
#pragma unroll
                for (int u = 0; u < kAhead; ++u)
                    if (id[u] >= 0 && int64_t(id[u]) < a.usedSize)
                        a.used[id[u]] = 0;
            }
        }
    }

    // what each request holds now; the last CTA counts those left short, over all of them where
    // each CTA has them all, else its share of them
    const bool last = blockIdx.x == gridDim.x - 1;
    uint32_t missed = 0;
    auto fits = [&](const Blocks& b, uint32_t r) {
        return b.need <= b.held || (b.need <= uint32_t(a.width) && upto[r] <= available);
    };
    for (uint32_t r = blockIdx.x * kThreads + threadIdx.x; r < a.requests; r += gridDim.x * kThreads) {
        const Blocks b = request(r);
        const bool ok = fits(b, r);
        a.blocks[r] = int32_t(!b.live ? 0u : (ok && b.need > b.held ? b.need : b.held));
        missed += !InBlock && !ok ? 1u : 0u;
    }
    if (InBlock && !last)
        return;
    if constexpr (InBlock)
        for (uint32_t r = threadIdx.x; r < a.requests; r += kThreads)
            missed += fits(request(r), r) ? 0u : 1u;
    missed = warpSum(missed);
    if (lane == 0 && missed != 0)
        atomicAdd(&sShort, missed);
    __syncthreads();
    if (threadIdx.x == 0) {
        if (last) {
            // the sums never fall, so the requests that fit with new blocks are the first ones,
            // up to the last sum within the pool
            const uint32_t fitting = requestOf(upto, a.requests, available);
            a.cells[0] = fitting == 0 ? 0u : upto[fitting - 1];
        }
        if (InBlock)
            a.cells[1] = sShort;
        else if (sShort != 0)  // zeroed by the scan
            atomicAdd(a.cells + 1, sShort);
    }
}

// ------------------------------------------------------------------ slots

/** kTokens neighbouring tokens a thread and step: four, stored as words, or one where that leaves
 *  SMs idle. ``Copied``: the scan is read from scratch into shared memory first (up to kScanAtOnce requests),
 *  where a search is a tenth of the time. ``Held``: entries past what a request holds are not read. */
template <class Len, class Slot, uint32_t kTokens, bool InBlock, bool Copied, bool Held>
__global__ __launch_bounds__(kThreads) void slotMapKernel(PagedArgs a)
{
    __shared__ uint32_t segment[InBlock ? kMaxSegments + 1 : 1];
    __shared__ int64_t starts[InBlock ? kScanInBlock : 1];
    __shared__ uint32_t sUpto[InBlock ? kScanInBlock : (Copied ? kScanAtOnce : 1)];
    const uint32_t* upto = InBlock || Copied ? sUpto : a.upto;
    letNextKernelStart();
    waitForKernelBefore();
    if constexpr (InBlock) {
        (void)scanBlock<kThreads, kItems, Tokens, Len>(a, 0, 0, sUpto, starts, segment);
    } else {
        if constexpr (Copied) {
#pragma unroll 8
            for (uint32_t i = threadIdx.x; i < a.requests; i += kThreads)
                sUpto[i] = __ldcg(a.upto + i);
            __syncthreads();
        }
    }
    const uint32_t lane = threadIdx.x & 31u, warp = blockIdx.x * kWarps + (threadIdx.x >> 5),
                   warps = gridDim.x * kWarps;
    for (uint64_t w0 = uint64_t(warp) * 32u * kTokens; w0 < a.capacity; w0 += uint64_t(warps) * 32u * kTokens) {
        // one search for the warp's tokens, which are mostly one request's
        uint32_t r = requestOf(upto, a.requests, uint32_t(w0));
        const bool one = r < a.requests && uint64_t(upto[r]) >= w0 + 32u * kTokens;
        const uint64_t q0 = w0 + lane * kTokens;
        Pack<Slot, kTokens> slot;
        Pack<Len, kTokens> position;
        Pack<int32_t, kTokens> request;
        int64_t id[kTokens];
        uint32_t within[kTokens];
#pragma unroll
        for (uint32_t k = 0; k < kTokens; ++k) {
            const uint32_t q = uint32_t(q0) + k;
            if (!one)
                r = requestFrom(upto, a.requests, q, r);
            position.e[k] = 0;
            request.e[k] = -1;
            id[k] = -1;
            within[k] = 0;
            if (r < a.requests) {
                const uint32_t before = r == 0 ? 0u : upto[r - 1];
                const int64_t start = InBlock ? starts[r] : lengthAt<Len>(a.start, r);
                const uint64_t p = uint64_t(start) + (q - before);
                position.e[k] = Len(p);
                request.e[k] = int32_t(r);
                if (p < uint64_t(a.room)) {
                    const uint32_t b = a.perBlock(uint32_t(p));
                    within[k] = uint32_t(p) - b * a.perBlock.d;
                    if (!Held || int64_t(b) < int64_t(a.held[r]))
                        id[k] = a.table[int64_t(r) * a.tableStride + b];
                }
            }
        }
#pragma unroll
        for (uint32_t k = 0; k < kTokens; ++k) {
            const int64_t at = id[k] * a.perBlock.d + within[k];
            slot.e[k] = id[k] >= 0 && int64_t(Slot(at)) == at ? Slot(at) : Slot(-1);
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

template <class What, class Len>
void launchScan(const PagedArgs& a, cudaStream_t s, const char* who)
{
    launchBehind(scanKernel<What, Len>, 1, kScanThreads, 0, s, a, who);
}

/** CTAs for ``threads`` threads' work, at most ``most`` an SM. */
unsigned gridFor(int64_t threads, int64_t most)
{
    return unsigned(std::max<int64_t>(1, std::min(most * smCount(), (threads + kThreads - 1) / kThreads)));
}

template <class Len, class Slot, uint32_t kTokens, bool Held>
void launchSlots(const PagedArgs& a, cudaStream_t s, const char* who)
{
    const int64_t threads = (int64_t(a.capacity) + kTokens - 1) / kTokens;
    if (a.requests <= kScanInBlock) {
        launchBehind(slotMapKernel<Len, Slot, kTokens, true, false, Held>, gridFor(threads, 4), kThreads, 0, s, a, who);
        return;
    }
    launchScan<Tokens, Len>(a, s, who);
    if (a.requests <= kScanAtOnce)
        launchBehind(slotMapKernel<Len, Slot, kTokens, false, true, Held>, gridFor(threads, 4), kThreads, 0, s, a, who);
    else
        launchBehind(slotMapKernel<Len, Slot, kTokens, false, false, Held>, gridFor(threads, 4), kThreads, 0, s, a,
            who);
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
        // a thread per four entries that the call can write, a warp per request at least
        const int64_t entries = std::min(d.pool_size + (d.used != 0 ? d.used_size : 0), d.requests * d.width);
        const int64_t threads = std::max(d.requests * 32, entries / 4);
        withIndex(d.length_type, [&](auto len) {
            using Len = decltype(len);
            if (d.requests <= int64_t(kScanInBlock)) {
                launchBehind(blockTablesKernel<Len, true>, gridFor(threads, 4), kThreads, 0, s, a, who);
            } else {
                launchScan<Blocks, Len>(a, s, who);
                launchBehind(blockTablesKernel<Len, false>, gridFor(threads, 4), kThreads, 0, s, a, who);
            }
        });
    });
}

EB_API eagle_backend_status eagle_backend_x_b200_slot_map(eagle_b200_paged_desc* desc)
{
    return guarded([&] {
        const char* who = "eagle_backend_x_b200_slot_map";
        const eagle_b200_paged_desc d = readDesc(desc, EAGLE_B200_SLOT_MAP_HELD, who);
        const bool held = (d.flags & EAGLE_B200_SLOT_MAP_HELD) != 0;
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
            if (held)
                requireAddress(d.held, 4, who, "held");
            if (d.width > 0)
                requireAddress(d.table, 4, who, "table");
        }
        requireDevice();
        DeviceScope scope(resolveDevice(d.device, d.offsets));
        a.start = reinterpret_cast<const void*>(d.start);
        a.fresh = reinterpret_cast<const void*>(d.fresh);
        a.held = reinterpret_cast<const int32_t*>(d.held);
        a.capacity = uint32_t(d.capacity);
        a.slots = reinterpret_cast<void*>(d.slots);
        a.positions = reinterpret_cast<void*>(d.positions);
        a.tokenRequests = reinterpret_cast<int32_t*>(d.token_requests);
        a.offsets = reinterpret_cast<int32_t*>(d.offsets);
        const cudaStream_t s = seamStream(d.stream);
        withIndex(d.length_type, [&](auto len) {
            withIndex(d.slot_type, [&](auto slot) {
                using Len = decltype(len);
                using Slot = decltype(slot);
                const bool few = d.capacity <= int64_t(smCount()) * kThreads;
                if (few && held)
                    launchSlots<Len, Slot, 1, true>(a, s, who);
                else if (few)
                    launchSlots<Len, Slot, 1, false>(a, s, who);
                else if (held)
                    launchSlots<Len, Slot, 4, true>(a, s, who);
                else
                    launchSlots<Len, Slot, 4, false>(a, s, who);
            });
        });
    });
}
