// The gradient of an embedding table:
//
//   table[v, :] = round(scale * sum over {t : token[t] = first + v} of values[t, :])
//
// A scatter-add, done without atomics on the values: the tokens are sorted by
// id (stable, so equal ids keep token order), the sorted order is cut into chunks of a length
// that the sizes fix, and every run of equal ids is summed in registers by the lanes that own
// its columns. A run inside one chunk, or across one boundary, goes straight to its row; a
// longer one leaves a 32-bit partial per chunk, joined in chunk order by a second kernel. A
// row is thus one sum in one order. Rows without a token are zeroed by CTAs that only store,
// beside the sort, the sums and the joins. 131072 tokens of 4096 bf16 into as many rows take
// 360 us, 6.0 TB/s of what has to move: 32 in the sort, 300 in the sums at 6.0 TB/s of DRAM
// traffic, 30 in the joins and the zeroing beside them.
//
// The sort is least-significant-digit radix over bits(rows) bits, at most 9 a pass: up to 131072
// tokens in one launch, by a CTA or a cluster that keeps the keys in shared memory; past that
// a kernel a pass, whose tiles add up one another's digit counts themselves (no wait on another
// CTA), from 129 tiles on after a kernel that scans them: the first counts come from a kernel of
// their own, each later pass's are gathered by the pass before, which knows where its keys land.
#include "sequences.cuh"

#include <cooperative_groups.h>

#include <algorithm>
#include <mutex>
#include <vector>

#define EB_API extern "C" __attribute__((visibility("default")))

namespace eb {
namespace {

// ------------------------------------------------------------------ the sort

constexpr uint32_t kMaxBins = 512;        // 9 bits a pass
constexpr int64_t kZeroUnit = 16384;      // bytes a CTA zeroes
constexpr int64_t kZeroByWarp = 2048;     // bytes of a row that one warp zeroes
constexpr uint32_t kWarpParts = 32;       // partials of a run that one warp joins
constexpr uint32_t kNoKey = 0xffffffffu;  // behind the last key: every digit of it is the highest

struct GradArgs {
    const void* tokens;
    const void* values;
    void* table;
    int64_t rows, first;
    int64_t tableStride;
    int64_t tokenBatch, tokenSeq;
    int64_t valueBatch, valueSeq, valueDim;
    FastDiv perBatch;  // by seq
    bool flatTokens, flatValues;
    bool tableAligned;  // every pack of the table's rows lies on its words
    bool accumulate;
    float scale;
    uint32_t n;
    uint32_t dim;
    // sort
    uint32_t bits, bins, digitBits;
    uint32_t tiles;
    uint32_t* present;   // a bit per row that has a token
    uint32_t* hist;      // this pass's digit counts, [tile][bin]
    uint32_t* nextHist;  // the next pass's, gathered by this one
    uint32_t* totals;    // the digits' counts over all tiles, hist then scanned over the tiles; or null
    const uint32_t* keyIn;
    const uint32_t* posIn;
    uint32_t* keyOut;
    uint32_t* posOut;
    uint32_t shift;
    // sums
    const uint32_t* keys;   // sorted; ``rows`` for a token without a row
    const uint32_t* order;  // the sorted keys' token positions
    uint32_t chunk, chunks;
    uint32_t group;      // lanes that share a row's pieces
    uint32_t slices;     // groups a row takes
    uint32_t pieces;     // packs (or columns) per row
    uint32_t sumBlocks;  // CTAs that sum; the others zero
    uint32_t polls;      // of a wait for rows, after which it gives up
    uint32_t asked;      // groups of rows asked for in the first chunk, at most
    uint32_t* lost;      // set to 1 where a wait gave up
    uint32_t* listCount; // {runs of up to kWarpParts partials, of more}
    uint32_t* list;      // the chunks they start in
    uint32_t* longList;
    float* head;         // [chunk][width]: the part of a long run that began in an earlier chunk
    float* tail;         // [chunk][width]: the part of a long run that goes on
    uint32_t width;      // dim rounded up to 8
    // zeroing
    int64_t rowBytes, strideBytes;
    uint32_t zeroRows;    // rows in a unit
    uint32_t zeroPieces;  // units in a row
    int64_t zeroed;       // rows [0, zeroed) are zeroed, with tokens or without, beside the sort
    int64_t zeroedBefore; // rows up to this are zeroed before the joins, the others beside them
    uint32_t joinBlocks;  // CTAs that join; the others zero
    uint32_t joinLanes;   // lanes that hold a row's columns, or 128 of them, four each
};

/** The keys of Items tokens, ``step`` apart from ``from`` on (kNoKey past the last). No branch
 *  stands between the loads, so all are in flight together. */
template <class Tok, int Items>
__device__ __forceinline__ void loadKeys(const GradArgs& a, uint32_t from, uint32_t step, uint32_t (&key)[Items])
{
    const Tok* tokens = reinterpret_cast<const Tok*>(a.tokens);
    Tok id[Items];
#pragma unroll
    for (int k = 0; k < Items; ++k) {
        const uint32_t i = min(from + uint32_t(k) * step, a.n - 1u);
        const uint32_t b = a.flatTokens ? 0u : a.perBatch(i);
        id[k] = tokens[int64_t(b) * a.tokenBatch + int64_t(i - b * a.perBatch.d) * a.tokenSeq];
    }
#pragma unroll
    for (int k = 0; k < Items; ++k) {
        const uint64_t r = uint64_t(int64_t(id[k])) - uint64_t(a.first);  // first >= 0: no wrap above it
        key[k] = int64_t(id[k]) >= a.first && r < uint64_t(a.rows) ? uint32_t(r) : uint32_t(a.rows);
        if (from + uint32_t(k) * step >= a.n)
            key[k] = kNoKey;
    }
}

/** Zero the bytes [from, to), both even, with threads ``at``, ``at + step``, ...: whole 16-byte
 *  words, and two bytes at a time before and after. */
__device__ __forceinline__ void zeroBytes(char* from, char* to, uint32_t at, uint32_t step)
{
    char* words = reinterpret_cast<char*>((reinterpret_cast<uint64_t>(from) + 15u) & ~uint64_t(15));
    char* rest = reinterpret_cast<char*>(reinterpret_cast<uint64_t>(to) & ~uint64_t(15));
    if (words > rest) {  // inside one word
        words = to;
        rest = to;
    }
    for (char* p = words + size_t(at) * 16u; p < rest; p += size_t(step) * 16u)
        *reinterpret_cast<uint4*>(p) = make_uint4(0u, 0u, 0u, 0u);
    for (char* p = from + size_t(at) * 2u; p < words; p += size_t(step) * 2u)
        *reinterpret_cast<uint16_t*>(p) = 0;
    for (char* p = rest + size_t(at) * 2u; p < to; p += size_t(step) * 2u)
        *reinterpret_cast<uint16_t*>(p) = 0;
}

/** Zero unit ``unit`` of the rows [row0, row1), of those whose bit in ``present`` is clear
 *  (all if it is null): a unit is ``zeroRows`` rows or, of longer ones, a piece of kZeroUnit
 *  bytes. CTAs that take neighbouring units one after the other write at 7.4 TB/s; a grid of as
 *  many CTAs as fit, striding over the plane, at 6.2, and beside the sums, a row a warp, at less:
 *  there the same work took 410 us instead of 312. */
__device__ __forceinline__ void zeroUnit(const GradArgs& a, const uint32_t* present, int64_t row0, int64_t row1,
    uint64_t unit)
{
    char* table = reinterpret_cast<char*>(a.table);
    const uint64_t which = unit / a.zeroPieces;
    const int64_t piece = int64_t(unit - which * a.zeroPieces) * kZeroUnit;
    const int64_t begin = row0 + int64_t(which) * a.zeroRows, end = min(begin + int64_t(a.zeroRows), row1);
    auto absent = [&](int64_t r) {
        return present == nullptr || ((present[r >> 5] >> (r & 31)) & 1u) == 0;
    };
    if (a.rowBytes <= kZeroByWarp) {
        for (int64_t r = begin + (threadIdx.x >> 5); r < end; r += blockDim.x >> 5)
            if (absent(r))
                zeroBytes(table + r * a.strideBytes, table + r * a.strideBytes + a.rowBytes, threadIdx.x & 31u, 32u);
    } else {
        for (int64_t r = begin; r < end; ++r)
            if (absent(r))
                zeroBytes(table + r * a.strideBytes + piece,
                    table + r * a.strideBytes + min(piece + kZeroUnit, a.rowBytes), threadIdx.x, blockDim.x);
    }
}

/** The keys of the same digit before each item among a CTA's: items are ranked warp by warp,
 *  among the 32 of a step by their lanes and between steps by the warp's running counts
 *  (item k of lane l is the warp's 32 k + l-th). The lanes of one digit find one another in a
 *  word of shared memory, each setting its own bit: match_any takes about 7 cycles per
 *  different value and warp (200 for random digits) and a ballot per bit 110, this 40.
 *  ``count`` and ``peers`` are [warp][bins] of shared memory, peers zero and left so; count is
 *  left scanned over the warps, and bin threadIdx.x's sum is returned. */
template <int Warps, int Items>
__device__ __forceinline__ uint32_t rankItems(const uint32_t (&key)[Items], uint32_t shift, uint32_t bits,
    uint32_t (&rank)[Items], uint16_t* count, uint32_t* peers)
{
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, bins = 1u << bits;
    __syncthreads();  // whoever still reads the counts of the pass before
    uint32_t* words = reinterpret_cast<uint32_t*>(count);
    for (uint32_t i = threadIdx.x; i < Warps * bins / 2; i += Warps * 32)
        words[i] = 0;
    __syncthreads();
    uint16_t* mine = count + warp * bins;
    uint32_t* same = peers + warp * bins;
#pragma unroll
    for (int k = 0; k < Items; ++k) {
        const uint32_t digit = (key[k] >> shift) & (bins - 1u);
        atomicOr(same + digit, 1u << lane);
        __syncwarp();
        const uint32_t lanes = same[digit], before = mine[digit];
        __syncwarp();
        if (lane == uint32_t(__ffs(lanes)) - 1u) {
            mine[digit] = uint16_t(before + __popc(lanes));
            same[digit] = 0;
        }
        __syncwarp();
        rank[k] = before + __popc(lanes & ((1u << lane) - 1u));
    }
    __syncthreads();
    uint32_t total = 0;
    if (threadIdx.x < bins) {
#pragma unroll
        for (int w = 0; w < Warps; ++w) {
            const uint32_t c = count[w * bins + threadIdx.x];
            count[w * bins + threadIdx.x] = uint16_t(total);
            total += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < Items; ++k)
        rank[k] += mine[(key[k] >> shift) & (bins - 1u)];
    return total;
}

// ---- up to kClusterKeys: one cluster, the keys in its distributed shared memory

constexpr int kClusterThreads = 512;  // a thread per bin; 1024, half the keys each, took 1.4 times as long
constexpr int kClusterWarps = kClusterThreads / 32;
constexpr int kClusterSize = 16;  // past the portable 8: asked for only where more than 8 are needed
constexpr int kClusterItems = 16;
constexpr uint32_t kClusterKeys = uint32_t(kClusterThreads) * kClusterSize * kClusterItems;  // 131072
constexpr uint32_t kPortableKeys = kClusterKeys / 2;
constexpr uint32_t kFewKeys = 8192;    // from here on 16 CTAs, where the device has such clusters, beat 8
// Up to here one CTA sorts: by eight, which exchange the keys, the gradient of 2500 to 4096 tokens
// takes 16.7 to 17.5 us instead of 18.2 to 19.5 where rows are narrow (64 bytes), and 25.1 instead of
// 24.6 where they are wide (2 KB), since fewer SMs are left to zero meanwhile.
constexpr uint32_t kAloneKeys = 4096;
static_assert(kClusterThreads >= int(kMaxBins), "a thread per bin");

/** Shared memory of the sort: the keys by place twice, the ranks' words and counts. */
constexpr size_t clusterShared(int items)
{
    return size_t(kClusterThreads) * items * 16 + size_t(kClusterWarps) * kMaxBins * 6;
}

/** Cluster 0 sorts: every CTA holds kClusterThreads * Items neighbouring keys in registers; a pass ranks
 *  them, puts them in digit order in the CTA's own shared memory, adds up the CTAs' digit
 *  counts over distributed shared memory and stores each key and position into the CTA that
 *  has its place, neighbours mostly to neighbours; two cluster barriers in all. The other
 *  clusters meanwhile zero the first ``zeroed`` rows. */
template <class Tok, int Items>
__global__ __launch_bounds__(kClusterThreads) void clusterSortKernel(GradArgs a)
{
    extern __shared__ __align__(16) unsigned char raw[];
    __shared__ uint32_t tileCount[kMaxBins], base[kMaxBins], scan[33];
    __shared__ uint32_t local[kMaxBins];
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t ctas = cluster.num_blocks(), cta = cluster.block_rank();
    letNextKernelStart();
    waitForKernelBefore();
    if (blockIdx.x >= ctas) {
        char* table = reinterpret_cast<char*>(a.table);
        const uint32_t at = blockIdx.x - ctas, others = gridDim.x - ctas;
        if (a.strideBytes == a.rowBytes) {  // one plane: every CTA 64 KB at a time
            constexpr int64_t kPiece = 65536;
            const int64_t bytes = a.zeroed * a.rowBytes;
            for (int64_t from = at * kPiece; from < bytes; from += others * kPiece)
                zeroBytes(table + from, table + min(from + kPiece, bytes), threadIdx.x, kClusterThreads);
        } else {
            for (int64_t r = int64_t(at) * kClusterWarps + (threadIdx.x >> 5); r < a.zeroed;
                 r += int64_t(others) * kClusterWarps)
                zeroBytes(table + r * a.strideBytes, table + r * a.strideBytes + a.rowBytes, threadIdx.x & 31u, 32u);
        }
        return;
    }
    constexpr uint32_t kTile = uint32_t(kClusterThreads) * Items;
    uint64_t* at = reinterpret_cast<uint64_t*>(raw);  // key and position by place in the order
    uint64_t* own = at + kTile;                       // by place among the CTA's
    uint32_t* peers = reinterpret_cast<uint32_t*>(own + kTile);
    uint16_t* count = reinterpret_cast<uint16_t*>(peers + kClusterWarps * kMaxBins);
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const uint32_t item0 = warp * (32u * Items) + lane;
    if (cta == 0 && threadIdx.x < 2)
        a.listCount[threadIdx.x] = 0;
    if (cta == 0 && threadIdx.x == 2)
        *a.lost = 0;
    if (a.present != nullptr)
        for (int64_t w = int64_t(cta) * kClusterThreads + threadIdx.x; w < (a.rows + 31) / 32;
             w += int64_t(ctas) * kClusterThreads)
            a.present[w] = 0;
    for (uint32_t i = threadIdx.x; i < kClusterWarps * kMaxBins; i += kClusterThreads)
        peers[i] = 0;
    uint32_t key[Items], pos[Items], rank[Items];
    loadKeys<Tok, Items>(a, cta * kTile + item0, 32u, key);
#pragma unroll
    for (int k = 0; k < Items; ++k)
        pos[k] = cta * kTile + item0 + 32u * k;
    for (uint32_t shift = 0; shift < a.bits; shift += a.digitBits) {
        const uint32_t mine = rankItems<kClusterWarps, Items>(key, shift, a.digitBits, rank, count, peers);
        uint32_t all = 0;
        const uint32_t first = blockExclusiveSum(mine, all, scan);
        if (threadIdx.x < a.bins) {
            tileCount[threadIdx.x] = mine;
            local[threadIdx.x] = first;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < Items; ++k)
            own[local[(key[k] >> shift) & (a.bins - 1u)] + rank[k]] = (uint64_t(pos[k]) << 32) | key[k];
        const uint64_t* from = own;
        if (ctas == 1) {
            __syncthreads();
        } else {
            cluster.sync();
            uint32_t before = 0, total = 0;
            if (threadIdx.x < a.bins) {
#pragma unroll 8
                for (uint32_t c = 0; c < ctas; ++c) {
                    const uint32_t v = cluster.map_shared_rank(tileCount, c)[threadIdx.x];
                    total += v;
                    before += c < cta ? v : 0u;
                }
            }
            const uint32_t lower = blockExclusiveSum(total, all, scan);
            if (threadIdx.x < a.bins)
                base[threadIdx.x] = lower + before - first;  // from a place among the CTA's to one in the order
            __syncthreads();
#pragma unroll
            for (int k = 0; k < Items; ++k) {
                const uint32_t j = uint32_t(k) * kClusterThreads + threadIdx.x;
                const uint64_t v = own[j];
                const uint32_t to = base[(uint32_t(v) >> shift) & (a.bins - 1u)] + j;
                cluster.map_shared_rank(at, to / kTile)[to % kTile] = v;
            }
            cluster.sync();
            from = at;
        }
#pragma unroll
        for (int k = 0; k < Items; ++k) {
            const uint64_t v = from[item0 + 32u * k];
            key[k] = uint32_t(v);
            pos[k] = uint32_t(v >> 32);
        }
    }
#pragma unroll
    for (int k = 0; k < Items; ++k) {
        const uint32_t i = cta * kTile + item0 + 32u * k;
        const uint32_t left = __shfl_up_sync(kFull, key[k], 1);
        if (i < a.n) {
            a.keyOut[i] = key[k];
            a.posOut[i] = pos[k];
            // cleared before the passes, whose barriers order that before this
            if (a.present != nullptr && key[k] < uint32_t(a.rows) && (lane == 0 || left != key[k]))
                atomicOr(a.present + (key[k] >> 5), 1u << (key[k] & 31u));
        }
    }
}

// ---- any number: a kernel a pass

constexpr int kSortThreads = 512;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortItems = 8;
constexpr uint32_t kSortTile = uint32_t(kSortThreads) * kSortItems;  // 4096 keys
constexpr uint32_t kTilesAdded = 128;  // adding up so many in every tile costs what the scan's launch does

/** A tile's digit counts of the first pass, and the rows that have a token. */
template <class Tok>
__global__ __launch_bounds__(kSortThreads) void histogramKernel(GradArgs a)
{
    __shared__ uint32_t count[kMaxBins];
    letNextKernelStart();
    if (threadIdx.x < a.bins)
        count[threadIdx.x] = 0;
    __syncthreads();
    uint32_t key[kSortItems], word[kSortItems];
    loadKeys<Tok, kSortItems>(a, blockIdx.x * kSortTile + threadIdx.x, kSortThreads, key);
#pragma unroll
    for (int k = 0; k < kSortItems; ++k)
        word[k] = a.present != nullptr && key[k] < uint32_t(a.rows) ? __ldcg(a.present + (key[k] >> 5)) : ~0u;
#pragma unroll
    for (int k = 0; k < kSortItems; ++k) {
        if (key[k] != kNoKey)
            atomicAdd(count + (key[k] & (a.bins - 1u)), 1u);
        const uint32_t bit = 1u << (key[k] & 31u);
        if ((word[k] & bit) == 0)  // a frequent id's bit is mostly seen set
            atomicOr(a.present + (key[k] >> 5), bit);
    }
    __syncthreads();
    if (threadIdx.x < a.bins)
        a.hist[size_t(blockIdx.x) * a.bins + threadIdx.x] = count[threadIdx.x];
}

/** The tiles' counts of each bin, scanned in place over the tiles, and their sums: a CTA takes 32
 *  bins and cuts the tiles into 32 stretches, added up, scanned and gone over again. */
__global__ __launch_bounds__(1024) void columnScanKernel(GradArgs a)
{
    __shared__ uint32_t sum[32][33];
    letNextKernelStart();
    waitForKernelBefore();
    const uint32_t column = threadIdx.x & 31u, stretch = threadIdx.x >> 5, bin = blockIdx.x * 32u + column;
    const uint32_t each = (a.tiles + 31u) / 32u, t0 = min(stretch * each, a.tiles), t1 = min(t0 + each, a.tiles);
    uint32_t mine = 0;
    if (bin < a.bins)
#pragma unroll 8
        for (uint32_t t = t0; t < t1; ++t)
            mine += __ldcg(a.hist + size_t(t) * a.bins + bin);
    sum[stretch][column] = mine;
    __syncthreads();
    uint32_t before = 0;
    for (uint32_t s = 0; s < stretch; ++s)
        before += sum[s][column];
    if (bin >= a.bins)
        return;
    if (stretch == 31)
        a.totals[bin] = before + mine;
    for (uint32_t t = t0; t < t1; ++t) {
        uint32_t* at = a.hist + size_t(t) * a.bins + bin;
        const uint32_t c = __ldcg(at);
        *at = before;
        before += c;
    }
}

/** One pass over one tile: a bin's first place is the keys of lower bins plus those of its
 *  own in earlier tiles, added up from every tile's counts by the bin's thread; past
 *  kTilesAdded tiles, where that would grow with their square, a scan has done it. */
template <bool First, class Tok>
__global__ __launch_bounds__(kSortThreads) void passKernel(GradArgs a)
{
    extern __shared__ __align__(16) unsigned char raw[];
    letNextKernelStart();
    waitForKernelBefore();
    uint32_t* peers = reinterpret_cast<uint32_t*>(raw);
    uint16_t* count = reinterpret_cast<uint16_t*>(peers + kSortWarps * kMaxBins);
    for (uint32_t i = threadIdx.x; i < kSortWarps * kMaxBins; i += kSortThreads)
        peers[i] = 0;
    __shared__ uint32_t base[kMaxBins], scan[33];
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const uint32_t item0 = blockIdx.x * kSortTile + warp * (32u * kSortItems) + lane;
    uint32_t key[kSortItems], pos[kSortItems], rank[kSortItems];
    if constexpr (First)
        loadKeys<Tok, kSortItems>(a, item0, 32u, key);
#pragma unroll
    for (int k = 0; k < kSortItems; ++k) {
        const uint32_t i = item0 + 32u * k;
        if constexpr (First) {
            pos[k] = i;
        } else {
            key[k] = i < a.n ? __ldcg(a.keyIn + i) : kNoKey;
            pos[k] = i < a.n ? __ldcg(a.posIn + i) : 0u;
        }
    }
    uint32_t before = 0, total = 0, all = 0;
    if (threadIdx.x < a.bins && a.totals != nullptr) {
        before = __ldcg(a.hist + size_t(blockIdx.x) * a.bins + threadIdx.x);
        total = __ldcg(a.totals + threadIdx.x);
    } else if (threadIdx.x < a.bins) {
        const uint32_t* column = a.hist + threadIdx.x;
#pragma unroll 16
        for (uint32_t t = 0; t < a.tiles; ++t) {
            const uint32_t c = __ldcg(column + size_t(t) * a.bins);
            total += c;
            before += t < blockIdx.x ? c : 0u;
        }
    }
    const uint32_t lower = blockExclusiveSum(total, all, scan);
    if (threadIdx.x < a.bins)
        base[threadIdx.x] = lower + before;
    (void)rankItems<kSortWarps, kSortItems>(key, a.shift, a.digitBits, rank, count, peers);  // its barriers publish base
#pragma unroll
    for (int k = 0; k < kSortItems; ++k) {
        const bool in = item0 + 32u * k < a.n;
        const uint32_t to = base[(key[k] >> a.shift) & (a.bins - 1u)] + rank[k];
        if (in) {
            a.keyOut[to] = key[k];
            a.posOut[to] = pos[k];
        }
        if (a.nextHist != nullptr) {
            // a frequent id's keys fall on one count: neighbours with the same one add together
            const uint32_t next =
                in ? (to / kSortTile) * a.bins + ((key[k] >> (a.shift + a.digitBits)) & (a.bins - 1u)) : kNoKey;
            const uint32_t lead = __shfl_sync(kFull, next, 0);
            const uint32_t equal = __ballot_sync(kFull, next == lead);
            if (in && (next != lead || lane == uint32_t(__ffs(equal)) - 1u))
                atomicAdd(a.nextHist + next, next == lead ? uint32_t(__popc(equal)) : 1u);
        }
    }
}

// ------------------------------------------------------------------ the sums

constexpr int kSumThreads = 256;
constexpr uint32_t kRowsInFlight = 8;

/** How a lane's N columns lie: neighbours read as one aligned 16-byte word; neighbours in a
 *  16-byte word of any alignment; or ``group`` apart, element by element, for values whose
 *  last stride is not 1. */
enum class Piece { Aligned, Shifted, Strided };

/** A row's value from its sum, and from what is there if that is added to: one rounding in 32 bits
 *  (written out, so that every path has the same bits) and the one to the row's type. */
template <class Out>
__device__ __forceinline__ Out scaled(const GradArgs& a, float sum, Out was)
{
    return fromFloat<Out>(a.accumulate ? __fmaf_rn(a.scale, sum, toFloat(was)) : __fmul_rn(a.scale, sum));
}

/** The columns ``col0``, ``col0 + apart``, ... of a row; ``apart`` is 1 but for Strided pieces. */
template <class In, class Out, Piece P, int N>
__device__ __forceinline__ void storeRow(const GradArgs& a, uint32_t row, uint32_t col0, uint32_t apart,
    const float (&acc)[N])
{
    Out* out = reinterpret_cast<Out*>(a.table) + int64_t(row) * a.tableStride;
    if (P == Piece::Aligned || (P == Piece::Shifted && a.tableAligned && col0 + N <= a.dim)) {
        Pack<Out, N>* at = reinterpret_cast<Pack<Out, N>*>(out + col0);
        Pack<Out, N> p{};
        if (a.accumulate)
            p = *at;
#pragma unroll
        for (int e = 0; e < N; ++e)
            p.e[e] = scaled<Out>(a, acc[e], p.e[e]);
        storePack(out + col0, p);
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const uint32_t col = col0 + uint32_t(e) * apart;
            if (col < a.dim)
                out[col] = scaled<Out>(a, acc[e], a.accumulate ? out[col] : Out());
        }
    }
}

/** A warp's 32 * N neighbouring columns from ``col0`` on, held N to a lane, through shared memory
 *  (``stage``, as many floats), so that rows that do not lie on words are written by neighbouring
 *  lanes all the same. The whole warp calls. */
template <class Out, int N>
__device__ __forceinline__ void storeStaged(const GradArgs& a, uint32_t row, uint32_t col0, const float (&acc)[N],
    float* stage)
{
    const uint32_t lane = threadIdx.x & 31u;
#pragma unroll
    for (int e = 0; e < N; ++e)
        stage[lane * N + e] = acc[e];
    __syncwarp();
    Out* out = reinterpret_cast<Out*>(a.table) + int64_t(row) * a.tableStride;
    Out was[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const uint32_t col = col0 + 32u * e + lane;
        was[e] = a.accumulate && col < a.dim ? out[col] : Out();
    }
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const uint32_t col = col0 + 32u * e + lane;
        if (col < a.dim)
            out[col] = scaled<Out>(a, stage[32 * e + lane], was[e]);
    }
    __syncwarp();
}

template <Piece P, int N>
__device__ __forceinline__ void storePartial(const GradArgs& a, float* to, uint32_t chunk, uint32_t col0,
    uint32_t apart, const float (&acc)[N])
{
    float* row = to + size_t(chunk) * a.width;
    if constexpr (P != Piece::Strided) {
        Pack<float, N> p;
#pragma unroll
        for (int e = 0; e < N; ++e)
            p.e[e] = acc[e];
        storePack(row + col0, p);
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const uint32_t col = col0 + uint32_t(e) * apart;
            if (col < a.dim)
                row[col] = acc[e];
        }
    }
}

/** Eight neighbours of an array of ``n`` from ``i`` (a multiple of 8) on; ``other`` past its end. */
__device__ __forceinline__ void loadEight(uint32_t (&v)[kRowsInFlight], const uint32_t* from, uint32_t i, uint32_t n,
    uint32_t other)
{
    if (i < n && n - i >= 8u) {
        const uint4 x = *reinterpret_cast<const uint4*>(from + i);
        const uint4 y = reinterpret_cast<const uint4*>(from + i)[1];
        v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
    } else {
#pragma unroll
        for (uint32_t u = 0; u < kRowsInFlight; ++u)
            v[u] = i < n && u < n - i ? from[i + u] : other;
    }
}

/** Element offset of token ``t``'s vector. */
__device__ __forceinline__ int64_t vectorOf(const GradArgs& a, uint32_t t)
{
    if (a.flatValues)
        return int64_t(t) * a.valueSeq;
    const uint32_t b = a.perBatch(t);
    return int64_t(b) * a.valueBatch + int64_t(t - b * a.perBatch.d) * a.valueSeq;
}

/** Chunk ``chunk``'s last run, of row ``key``, is one to join. In any order: each is joined on its own. */
__device__ __forceinline__ void listRun(const GradArgs& a, uint32_t chunk, uint32_t key)
{
    const uint64_t past = (uint64_t(chunk) + kWarpParts) * a.chunk;  // the first of one partial too many
    if (past < a.n && a.keys[past] == key)
        a.longList[atomicAdd(a.listCount + 1, 1u)] = chunk;
    else
        a.list[atomicAdd(a.listCount, 1u)] = chunk;
}

// The sorted order is cut into chunks. A run is long if two or more chunks begin inside it. A
// run that is not long is summed whole by the chunk it starts in, up to a chunk's length past
// its end, and skipped by the next. A long one leaves a partial in every chunk it touches.
// Which it is follows from the first keys of the neighbouring chunks, so both sides of a
// boundary agree.

// ---- wide contiguous rows: the copy engine brings them into shared memory

constexpr int kBulkLanes = 128;                   // threads that add, 16 bytes of a row each
constexpr int kBulkThreads = kBulkLanes + 32;     // and a warp that asks for the rows
constexpr uint32_t kBulkSlab = kBulkLanes * 16;   // bytes of a row per CTA
constexpr uint32_t kBulkSlot = kBulkSlab + 16;    // a piece of any alignment, in whole words
constexpr uint32_t kBulkRows = 4;                 // rows per barrier
constexpr uint32_t kBulkStages = 4;
constexpr uint32_t kMaxChunk = 64;
// bytes of an aligned row from which this is faster than loads into registers (65536 tokens of 512
// bytes: 67 us against 56; of 800: 74, 72); of one that is not, half of that (520: 91, 104)
constexpr int64_t kBulkLeast = 1024;
constexpr uint32_t kBulkWaits = 1u << 22;  // polls before a wait gives up
constexpr uint32_t kEvery = 0xffffffffu;

struct BulkShared {
    alignas(16) unsigned char row[kBulkStages][kBulkRows][kBulkSlot];
    uint64_t full[kBulkStages], empty[kBulkStages];
    uint32_t key[2 * kMaxChunk + 1], token[2 * kMaxChunk];
};

__device__ __forceinline__ void mbarArrive(uint64_t* bar)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(sharedAddr(bar)) : "memory");
}

__device__ __forceinline__ void mbarExpect(uint64_t* bar, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(sharedAddr(bar)), "r"(bytes)
                 : "memory");
}

__device__ __forceinline__ void bulkCopy(void* dst, const void* src, uint32_t bytes, uint64_t* bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                     sharedAddr(dst)),
        "l"(src), "r"(bytes), "r"(sharedAddr(bar))
        : "memory");
}

/** One CTA sums the runs that start in one chunk over 2 KB of the columns. A warp asks the copy
 *  engine for the rows, up to 16 ahead and each as the whole 16-byte words that hold it; four
 *  warps add them from shared memory. So the memory is kept busy whatever the adding
 *  threads wait for: six CTAs an SM, which is what the shared memory holds, with 24 adding warps
 *  and up to 32 KB asked for each. (Compiled for those six, 131072 tokens of 8 KB take 360 us;
 *  for no number, 377.) */
template <class In, class Out, bool Aligned>
__global__ __launch_bounds__(kBulkThreads, 6) void bulkSumKernel(GradArgs a)
{
    constexpr int N = 16 / int(sizeof(In));
    constexpr Piece P = Aligned ? Piece::Aligned : Piece::Shifted;
    extern __shared__ __align__(16) unsigned char raw[];
    letNextKernelStart();
    waitForKernelBefore();
    if (blockIdx.x >= a.sumBlocks) {
        zeroUnit(a, a.present, a.zeroed, a.zeroedBefore, blockIdx.x - a.sumBlocks);
        return;
    }
    BulkShared& s = *reinterpret_cast<BulkShared*>(raw);
    const uint32_t chunk = blockIdx.x / a.slices, slab = blockIdx.x - chunk * a.slices;
    const uint32_t begin = chunk * a.chunk, size = a.chunk, none = uint32_t(a.rows);
    const uint32_t len = min(size, a.n - begin);
    for (uint32_t i = threadIdx.x; i <= 2 * size; i += kBulkThreads) {
        const bool in = i < a.n - begin;
        s.key[i] = in ? a.keys[begin + i] : kNoKey;
        if (i < 2 * size)
            s.token[i] = in ? a.order[begin + i] : 0u;
    }
    const uint32_t left = begin > 0 ? a.keys[begin - 1] : kNoKey;
    const uint32_t before = begin > 0 ? a.keys[begin - size] : kNoKey;  // the chunk before's first
    if (threadIdx.x == 0) {
        for (uint32_t k = 0; k < kBulkStages; ++k) {
            mbarInit(&s.full[k], 1);
            mbarInit(&s.empty[k], kBulkLanes / 32);
        }
    }
    __syncthreads();
    const uint32_t i = threadIdx.x, first = s.key[0];
    if (first >= none)
        return;
    // the rows [r0, r1) of the chunk and the next that are summed here
    const bool continued = begin > 0 && left == first;
    const bool fromBefore = continued && (before == first || s.key[size] == first);
    const uint32_t leading = uint32_t(__syncthreads_count(i < len && s.key[i] == first));
    const uint32_t valid = uint32_t(__syncthreads_count(i < len && s.key[i] < none));
    const uint32_t r0 = continued && !fromBefore ? leading : 0u;
    if (r0 >= valid)
        return;
    const uint32_t last = s.key[valid - 1];
    const bool goesOn = valid == size && s.key[size] == last;
    const bool joined = goesOn && ((last == first && (!continued || fromBefore)) || s.key[2 * size] == last);
    const uint32_t extra = uint32_t(__syncthreads_count(i < size && s.key[size + i] == last));
    const uint32_t r1 = goesOn && !joined ? size + extra : valid;

    const In* values = reinterpret_cast<const In*>(a.values);
    const uint32_t slab0 = slab * (kBulkSlab / uint32_t(sizeof(In)));  // its first column
    const uint32_t bytes = min(kBulkSlab, (a.dim - slab0) * uint32_t(sizeof(In)));
    const uint32_t steps = (r1 - r0 + kBulkRows - 1) / kBulkRows;
    if (threadIdx.x >= kBulkLanes) {
        if (threadIdx.x == kBulkLanes) {
            const uint32_t most = chunk == 0 ? min(steps, a.asked) : steps;
            uint32_t j = 0;
            for (; j < most; ++j) {
                const uint32_t stage = j % kBulkStages;
                if (j >= kBulkStages && !mbarWait(&s.empty[stage], (j / kBulkStages - 1) & 1u, a.polls))
                    break;  // an adding warp gave up
                const uint32_t rows = min(kBulkRows, r1 - r0 - j * kBulkRows);
                const char* from[kBulkRows];
                uint32_t size_[kBulkRows], sum = 0;
#pragma unroll
                for (uint32_t u = 0; u < kBulkRows; ++u) {
                    if (u >= rows)
                        break;
                    const uint64_t p =
                        reinterpret_cast<uint64_t>(values + vectorOf(a, s.token[r0 + j * kBulkRows + u]) + slab0);
                    from[u] = reinterpret_cast<const char*>(p & ~uint64_t(15));
                    size_[u] = Aligned ? bytes : (uint32_t(p & 15u) + bytes + 15u) & ~15u;
                    sum += size_[u];
                }
                mbarExpect(&s.full[stage], sum);
#pragma unroll
                for (uint32_t u = 0; u < kBulkRows; ++u)
                    if (u < rows)
                        bulkCopy(s.row[stage][u], from[u], size_[u], &s.full[stage]);
            }
            // the shared memory stays until the last copies are there, whoever gave up
            for (uint32_t k = j > kBulkStages ? j - kBulkStages : 0u; k < j; ++k)
                (void)mbarWait(&s.full[k % kBulkStages], (k / kBulkStages) & 1u, a.polls);
        }
        return;
    }
    const uint32_t col0 = slab0 + threadIdx.x * N;
    const bool active = col0 < a.dim;
    float* stage = reinterpret_cast<float*>(raw + sizeof(BulkShared)) + (threadIdx.x & ~31u) * N;
    auto store = [&](uint32_t row, const float (&sum)[N]) {
        if constexpr (!Aligned)
            storeStaged<Out, N>(a, row, slab0 + (threadIdx.x & ~31u) * N, sum, stage);
        else if (active)
            storeRow<In, Out, P, N>(a, row, col0, 1u, sum);
    };
    float acc[N];
#pragma unroll
    for (int e = 0; e < N; ++e)
        acc[e] = 0.0f;
    uint32_t current = s.key[r0];
    bool partial = fromBefore;  // the run being summed began before: its sum is the chunk's head
    // the run of ``key`` from here on: what was summed goes where it belongs
    auto turnTo = [&](uint32_t key) {
        if (!partial)
            store(current, acc);
        else if (active)
            storePartial<P, N>(a, a.head, chunk, col0, 1u, acc);
        partial = false;
        current = key;
#pragma unroll
        for (int e = 0; e < N; ++e)
            acc[e] = 0.0f;
    };
    uint32_t j = 0;
    for (; j < steps; ++j) {
        const uint32_t stage = j % kBulkStages, parity = (j / kBulkStages) & 1u;
        if (!__all_sync(kFull, mbarWait(&s.full[stage], parity, a.polls)))
            break;
        const uint32_t rows = min(kBulkRows, r1 - r0 - j * kBulkRows);
#pragma unroll
        for (uint32_t u = 0; u < kBulkRows; ++u) {
            if (u >= rows)
                break;
            const uint32_t key = s.key[r0 + j * kBulkRows + u];
            if (key != current)
                turnTo(key);
            if (active) {
                uint4 w;
                if constexpr (Aligned) {
                    w = *reinterpret_cast<const uint4*>(s.row[stage][u] + threadIdx.x * 16);
                } else {
                    const uint64_t p =
                        reinterpret_cast<uint64_t>(values + vectorOf(a, s.token[r0 + j * kBulkRows + u]) + slab0);
                    const uint4* at = reinterpret_cast<const uint4*>(s.row[stage][u] + threadIdx.x * 16);
                    w = shiftWords(at[0], at[1], uint32_t(p) & 15u);
                }
                const Pack<In, N> v = *reinterpret_cast<const Pack<In, N>*>(&w);
#pragma unroll
                for (int e = 0; e < N; ++e)
                    acc[e] += toFloat(v.e[e]);
            }
        }
        __syncwarp();
        if ((threadIdx.x & 31u) == 0)
            mbarArrive(&s.empty[stage]);
    }
    if (j < steps) {
        // a wait gave up: the rows from there on count as NaN, unread, and the stage is not given
        // back, so that nothing more is asked for into it
        *a.lost = 1u;
#pragma unroll 1
        for (uint32_t r = r0 + j * kBulkRows; r < r1; ++r) {
            if (s.key[r] != current)
                turnTo(s.key[r]);
#pragma unroll
            for (int e = 0; e < N; ++e)
                acc[e] = __int_as_float(0x7fc00000);
        }
    }
    if (!partial && !joined) {
        store(current, acc);
    } else if (active) {
        storePartial<P, N>(a, partial ? a.head : a.tail, chunk, col0, 1u, acc);
        if (!partial && slab == 0 && threadIdx.x == 0)
            listRun(a, chunk, current);
    }
}

// ---- narrow or strided rows: loads into registers

/** A chunk by the lanes owning one slice of the columns; the next eight ids and positions are on
 *  their way while eight rows are. */
template <class In, class Out, Piece P, int N>
__global__ __launch_bounds__(kSumThreads) void sumKernel(GradArgs a)
{
    letNextKernelStart();
    waitForKernelBefore();
    if (blockIdx.x >= a.sumBlocks) {
        zeroUnit(a, a.present, a.zeroed, a.zeroedBefore, blockIdx.x - a.sumBlocks);
        return;
    }
    const uint64_t id = uint64_t(blockIdx.x) * kSumThreads + threadIdx.x;
    const uint32_t lane = uint32_t(id) & (a.group - 1u);
    const uint64_t which = id / a.group;  // a power of two
    const uint32_t chunk = uint32_t(which / a.slices), slice = uint32_t(which % a.slices);
    if (chunk >= a.chunks || (P != Piece::Strided && slice * a.group + lane >= a.pieces))
        return;
    const uint32_t begin = chunk * a.chunk, end = min(begin + a.chunk, a.n);
    const uint32_t none = uint32_t(a.rows);
    const In* values = reinterpret_cast<const In*>(a.values);
    const uint32_t apart = P == Piece::Strided ? a.group : 1u;
    const uint32_t col0 = P == Piece::Strided ? slice * N * a.group + lane : (slice * a.group + lane) * N;
    // the first key of the d-th chunk from this one
    auto firstKey = [&](int d) {
        const int64_t i = (int64_t(chunk) + d) * a.chunk;
        return i >= 0 && i < int64_t(a.n) ? a.keys[i] : kNoKey;
    };
    uint32_t key[kRowsInFlight], token[kRowsInFlight];
    loadEight(key, a.keys, begin, a.n, kNoKey);
    loadEight(token, a.order, begin, a.n, 0u);
    const uint32_t first = key[0];
    if (first >= none)
        return;
    uint32_t current = first, skipped = kNoKey;
    bool fromBefore = false;
    if (begin > 0 && a.keys[begin - 1] == first) {
        if (firstKey(-1) == first || firstKey(1) == first) {
            fromBefore = true;
        } else {
            skipped = first;
            current = kNoKey;  // no run yet
        }
    }
    float acc[N];
#pragma unroll
    for (int e = 0; e < N; ++e)
        acc[e] = 0.0f;
    uint32_t stop = end;
    bool extending = false, done = false;
    for (uint32_t i0 = begin; !done; i0 += kRowsInFlight) {
        if (i0 >= stop) {
            if (extending || current == kNoKey || end == a.n || a.keys[end] != current)
                break;
            if (fromBefore)
                break;
            if (first == current && skipped == kNoKey)  // it starts with the chunk: the second chunk to begin in it
                break;
            if (firstKey(2) == current)
                break;
            extending = true;
            stop = a.n - end < a.chunk ? a.n : end + a.chunk;
        }
        uint4 got[kRowsInFlight];
        float loose[kRowsInFlight][P == Piece::Strided ? N : 1];
#pragma unroll
        for (uint32_t u = 0; u < kRowsInFlight; ++u) {
            if (key[u] >= none || key[u] == skipped || (extending && key[u] != current))
                continue;
            const int64_t at = vectorOf(a, token[u]);
            if constexpr (P == Piece::Aligned)
                got[u] = *reinterpret_cast<const uint4*>(values + at + col0);
            else if constexpr (P == Piece::Shifted)
                got[u] = loadShifted(values + at + col0, min(uint32_t(N), a.dim - col0) * uint32_t(sizeof(In)));
            else {
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const uint32_t col = col0 + uint32_t(e) * apart;
                    loose[u][e] = col < a.dim ? toFloat(values[at + int64_t(col) * a.valueDim]) : 0.0f;
                }
            }
        }
        uint32_t nextKey[kRowsInFlight], nextToken[kRowsInFlight];
        loadEight(nextKey, a.keys, i0 + kRowsInFlight, a.n, kNoKey);
        loadEight(nextToken, a.order, i0 + kRowsInFlight, a.n, 0u);
#pragma unroll
        for (uint32_t u = 0; u < kRowsInFlight; ++u) {
            if (done || key[u] == skipped)
                continue;
            if (key[u] != current) {
                if (extending) {
                    done = true;
                    continue;
                }
                if (fromBefore)
                    storePartial<P, N>(a, a.head, chunk, col0, apart, acc);
                else if (current != kNoKey)
                    storeRow<In, Out, P, N>(a, current, col0, apart, acc);
                fromBefore = false;
                current = key[u];
                if (current >= none) {  // padding, or the end
                    current = kNoKey;
                    done = true;
                    continue;
                }
#pragma unroll
                for (int e = 0; e < N; ++e)
                    acc[e] = 0.0f;
            }
            if constexpr (P == Piece::Strided) {
#pragma unroll
                for (int e = 0; e < N; ++e)
                    acc[e] += loose[u][e];
            } else {
                const Pack<In, N> p = *reinterpret_cast<const Pack<In, N>*>(&got[u]);
#pragma unroll
                for (int e = 0; e < N; ++e)
                    acc[e] += toFloat(p.e[e]);
            }
        }
#pragma unroll
        for (uint32_t u = 0; u < kRowsInFlight; ++u) {
            key[u] = nextKey[u];
            token[u] = nextToken[u];
        }
    }
    if (current == kNoKey)
        return;
    if (fromBefore) {
        storePartial<P, N>(a, a.head, chunk, col0, apart, acc);
    } else if (!extending && end < a.n && a.keys[end] == current) {
        storePartial<P, N>(a, a.tail, chunk, col0, apart, acc);
        if (slice == 0 && lane == 0)
            listRun(a, chunk, current);
    } else {
        storeRow<In, Out, P, N>(a, current, col0, apart, acc);
    }
}

// ---- the rows of long runs

constexpr int kJoinThreads = 256;
constexpr int kJoinWarps = kJoinThreads / 32;
constexpr uint32_t kJoinColumns = 128;  // four per lane

/** The partials [p0, p1) of the run whose first is chunk ``chunk``'s tail, four columns from
 *  ``col`` on, Ahead of them in flight, added in order. */
template <int Ahead>
__device__ __forceinline__ float4 addPartials(const GradArgs& a, uint32_t chunk, uint32_t p0, uint32_t p1, uint32_t col)
{
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (uint32_t p = p0; p < p1; p += Ahead) {
        float4 v[Ahead];
#pragma unroll
        for (int u = 0; u < Ahead; ++u) {
            // past the last: the last again, not added
            const uint32_t q = min(p + uint32_t(u), p1 - 1u);
            v[u] = __ldcg(reinterpret_cast<const float4*>((q == 0 ? a.tail : a.head) + size_t(chunk + q) * a.width + col));
        }
#pragma unroll
        for (int u = 0; u < Ahead; ++u) {
            if (p + uint32_t(u) < p1) {
                sum.x += v[u].x;
                sum.y += v[u].y;
                sum.z += v[u].z;
                sum.w += v[u].w;
            }
        }
    }
    return sum;
}

template <class Out>
__device__ __forceinline__ void storeJoined(const GradArgs& a, uint32_t row, uint32_t col, float4 sum)
{
    Out* out = reinterpret_cast<Out*>(a.table) + int64_t(row) * a.tableStride;
    const float got[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (col + e < a.dim)
            out[col + e] = scaled<Out>(a, got[e], a.accumulate ? out[col + e] : Out());
}

/** Rows of up to kWarpParts partials: a warp adds 128 columns of one, in chunk order. Rows of
 *  more: a CTA's eight warps (of narrow rows up to 64 groups of lanes) add an eighth (a 64th) of
 *  its partials each, in chunk order, then those sums in order. (A frequent id of ordinary text has tens of partials and there are a
 *  few hundred of them: a CTA each, all columns in turn, took twice as long. A batch of one id
 *  has thousands.) */
template <class Out>
__global__ __launch_bounds__(kJoinThreads, 6) void joinKernel(GradArgs a)  // six an SM, for the zeroing ones
{
    __shared__ float4 part[kJoinThreads];
    letNextKernelStart();
    waitForKernelBefore();
    if (blockIdx.x >= a.joinBlocks) {
        zeroUnit(a, a.present, a.zeroedBefore, a.rows, blockIdx.x - a.joinBlocks);
        return;
    }
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const uint32_t blocks = (a.dim + kJoinColumns - 1) / kJoinColumns;
    // a long run's columns by groups of joinLanes lanes, its partials by the groups
    const uint32_t group = threadIdx.x / a.joinLanes, groups = kJoinThreads / a.joinLanes, at = threadIdx.x % a.joinLanes;
    const uint64_t longItems = uint64_t(a.listCount[1]) * blocks, items = uint64_t(a.listCount[0]) * blocks;
    for (uint64_t item = blockIdx.x; item < longItems; item += a.joinBlocks) {
        const uint32_t chunk = a.longList[item / blocks];
        const uint32_t col = uint32_t(item % blocks) * kJoinColumns + at * 4u;
        const uint32_t key = a.keys[(chunk + 1u) * a.chunk];
        uint32_t m = 1;  // chunks after this one that the run reaches: the keys are sorted, so they are counted
        for (uint32_t more = 4 * kJoinThreads; more == 4 * kJoinThreads;) {
            bool in[4];
#pragma unroll
            for (uint32_t u = 0; u < 4; ++u) {
                const uint64_t c = uint64_t(chunk) + 1u + m + u * kJoinThreads + threadIdx.x;
                in[u] = c < a.chunks && a.keys[c * a.chunk] == key;
            }
            more = 0;
#pragma unroll
            for (uint32_t u = 0; u < 4; ++u)
                more += uint32_t(__syncthreads_count(in[u]));
            m += more;
        }
        const uint32_t parts = m + 1u, each = (parts + groups - 1) / groups;
        const uint32_t p0 = group * each, p1 = min(p0 + each, parts);
        if (col < a.width && p0 < p1)
            part[threadIdx.x] = addPartials<16>(a, chunk, p0, p1, col);
        else
            part[threadIdx.x] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        __syncthreads();
        if (group == 0 && col < a.dim) {
            float4 sum = part[at];
#pragma unroll 8
            for (uint32_t g = 1; g < groups; ++g) {
                const float4 v = part[g * a.joinLanes + at];
                sum.x += v.x;
                sum.y += v.y;
                sum.z += v.z;
                sum.w += v.w;
            }
            storeJoined<Out>(a, key, col, sum);
        }
        __syncthreads();
    }
    for (uint64_t item = uint64_t(blockIdx.x) * kJoinWarps + warp; item < items;
         item += uint64_t(a.joinBlocks) * kJoinWarps) {
        const uint32_t chunk = a.list[item / blocks];
        const uint32_t col = uint32_t(item % blocks) * kJoinColumns + lane * 4u;
        const uint64_t next = uint64_t(chunk) + 1u + lane;
        const uint32_t first = next < a.chunks ? a.keys[next * a.chunk] : kNoKey;
        const uint32_t key = __shfl_sync(kFull, first, 0);
        const uint32_t parts = 1u + __popc(__ballot_sync(kFull, first == key));
        if (col < a.width)
            storeJoined<Out>(a, key, col, addPartials<8>(a, chunk, 0, parts, col));
    }
}

/** No tokens: every row is zero. */
__global__ __launch_bounds__(kSumThreads) void zeroRowsKernel(GradArgs a)
{
    zeroUnit(a, nullptr, 0, a.rows, blockIdx.x);
}

// ------------------------------------------------------------------ host side

uint64_t roundUp(uint64_t v, uint64_t to) { return (v + to - 1) / to * to; }

/** Whether the current device holds a cluster of kClusterSize CTAs of the sort (kept per device). */
bool largeClusters()
{
    static std::mutex mu;
    static std::vector<int> known;  // 0: not asked, 1: no, 2: yes
    int dev = 0;
    cudaCheck(cudaGetDevice(&dev), "cudaGetDevice");
    std::lock_guard<std::mutex> lock(mu);
    if (int(known.size()) <= dev)
        known.resize(size_t(dev) + 1, 0);
    if (known[size_t(dev)] == 0) {
        auto kernel = clusterSortKernel<int32_t, kClusterItems>;
        cudaLaunchAttribute attr{};
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim = {unsigned(kClusterSize), 1, 1};
        cudaLaunchConfig_t config{};
        config.gridDim = dim3(kClusterSize, 1, 1);
        config.blockDim = dim3(kClusterThreads, 1, 1);
        config.dynamicSmemBytes = clusterShared(kClusterItems);
        config.attrs = &attr;
        config.numAttrs = 1;
        int clusters = 0;
        const bool ok = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                            int(config.dynamicSmemBytes)) == cudaSuccess
            && cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess
            && cudaOccupancyMaxActiveClusters(&clusters, kernel, &config) == cudaSuccess && clusters > 0;
        (void)cudaGetLastError();
        known[size_t(dev)] = ok ? 2 : 1;
    }
    return known[size_t(dev)] == 2;
}

/** How the gradient's sort, sums and scratch are laid out. */
struct GradPlan {
    uint32_t n = 0, bits = 0, passes = 0, digitBits = 0, bins = 0, tiles = 0;
    Piece piece = Piece::Strided;
    uint32_t pieces = 0, group = 0, slices = 0, chunk = 0, chunks = 0, width = 0;
    bool bulk = false;
    uint64_t lost = 0, present = 0, listCount = 0, hist = 0, zeroed = 0;  // offsets; [0, zeroed) is cleared
    uint64_t firstHist = 0, totals = 0, key[2] = {0, 0}, pos[2] = {0, 0}, list = 0, longList = 0, head = 0, tail = 0, bytes = 0;
};

GradPlan planGrad(const eagle_b200_embedding_desc& d, const char* who)
{
    GradPlan p;
    p.n = uint32_t(d.batch * d.seq);
    const int inBytes = elementBytes(d.values_type, who), outBytes = elementBytes(d.table_type, who);
    // keys are 0 .. rows (rows: a token without a row)
    while (p.bits < 32 && (uint64_t(d.rows) >> p.bits) != 0)
        ++p.bits;
    p.passes = (p.bits + 8) / 9;
    p.digitBits = p.passes == 0 ? 0 : (p.bits + p.passes - 1) / p.passes;
    p.bins = 1u << p.digitBits;
    p.tiles = (p.n + kSortTile - 1) / kSortTile;
    // whole 16-byte words if every vector and every row of the table starts on them
    const int pack = 16 / inBytes;
    const int64_t outWord = pack * outBytes;
    if (d.value_strides[2] == 1 || d.dim <= 1)
        p.piece = d.dim % pack == 0 && d.values % 16 == 0 && d.table % uint64_t(outWord) == 0
                && d.value_strides[0] * inBytes % 16 == 0 && d.value_strides[1] * inBytes % 16 == 0
                && d.table_stride * outBytes % outWord == 0
            ? Piece::Aligned
            : Piece::Shifted;
    p.bulk = p.piece != Piece::Strided && d.dim * inBytes >= (p.piece == Piece::Aligned ? kBulkLeast : kBulkLeast / 2);
    const int64_t columns = p.piece == Piece::Strided ? 4 : pack;
    p.pieces = uint32_t((d.dim + columns - 1) / columns);
    p.group = 1;
    while (p.group < 32 && p.group < p.pieces)
        p.group *= 2;
    p.slices = (p.pieces + p.group - 1) / p.group;
    // the longest chunk that still leaves enough warps of 256 columns to hide the row loads: a
    // longer one leaves fewer partials of long runs. Of the sizes alone, not of types or
    // alignment: it fixes the order of the sums, and the scratch the query asks for. (Wanting
    // 2048 warps for wide rows too, 65536 tokens of 512 take 64 us instead of 59; wanting 4096
    // for narrow ones, 65536 of 128 take 42 instead of 38.)
    const uint64_t wanted = d.dim >= 512 ? 4096 : 2048;
    p.chunk = 8;
    while (p.chunk < 64 && uint64_t(p.n) * ((uint64_t(d.dim) + 7) / 8) / 32 / (p.chunk * 2) >= wanted)
        p.chunk *= 2;
    p.chunks = (p.n + p.chunk - 1) / p.chunk;
    p.width = uint32_t(roundUp(uint64_t(d.dim), 8));
    uint64_t at = 0;
    auto take = [&](uint64_t bytes) {
        const uint64_t was = at;
        at += roundUp(bytes, 256);
        return was;
    };
    p.lost = take(4);  // the scratch's first word: the caller may read it
    p.present = take((uint64_t(d.rows) + 31) / 32 * 4);
    p.listCount = take(8);
    const bool portable = p.n <= kPortableKeys;  // the query's answer does not depend on the device
    const uint64_t histBytes = portable ? 0 : uint64_t(p.tiles) * p.bins * 4;
    p.hist = take(p.passes > 1 ? histBytes * (p.passes - 1) : 0);
    p.zeroed = at;
    p.firstHist = take(histBytes);
    p.totals = take(portable ? 0 : p.bins * 4);
    for (int k = 0; k < (portable ? 1 : 2); ++k) {
        p.key[k] = take(uint64_t(p.n) * 4);
        p.pos[k] = take(uint64_t(p.n) * 4);
    }
    p.list = take(uint64_t(p.chunks) * 4);
    p.longList = take(uint64_t(p.chunks) * 4);
    p.head = take(uint64_t(p.chunks) * p.width * 4);
    p.tail = take(uint64_t(p.chunks) * p.width * 4);
    p.bytes = at;
    return p;
}

template <class In, class Out, Piece P>
void launchSum(const GradArgs& a, unsigned blocks, cudaStream_t s, const char* who)
{
    constexpr int N = P == Piece::Strided ? 4 : 16 / int(sizeof(In));
    launchBehind(sumKernel<In, Out, P, N>, blocks, kSumThreads, 0, s, a, who);
}

template <class In, class Out, bool Aligned>
void launchBulkSum(const GradArgs& a, unsigned blocks, cudaStream_t s, const char* who)
{
    auto kernel = bulkSumKernel<In, Out, Aligned>;
    const size_t shared = sizeof(BulkShared) + (Aligned ? 0 : kBulkLanes * 16 / sizeof(In) * sizeof(float));
    cudaCheck(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(shared)), who);
    launchBehind(kernel, blocks, kBulkThreads, shared, s, a, who);
}

template <class Tok, int Items>
void launchClusterSort(const GradArgs& a, unsigned ctas, unsigned blocks, cudaStream_t s, const char* who)
{
    auto kernel = clusterSortKernel<Tok, Items>;
    const size_t shared = clusterShared(Items);
    cudaCheck(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(shared)), who);
    if (ctas > 8)
        cudaCheck(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1), who);
    cudaLaunchAttribute attr[2]{};
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {ctas, 1, 1};
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(blocks, 1, 1);
    config.blockDim = dim3(kClusterThreads, 1, 1);
    config.dynamicSmemBytes = shared;
    config.stream = s;
    config.attrs = attr;
    config.numAttrs = 2;
    cudaCheck(cudaLaunchKernelEx(&config, kernel, a), who);
}

template <bool First, class Tok>
void launchPass(const GradArgs& a, unsigned tiles, cudaStream_t s, const char* who)
{
    auto kernel = passKernel<First, Tok>;
    const int shared = kSortWarps * int(kMaxBins) * 6;
    cudaCheck(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, shared), who);
    launchBehind(kernel, tiles, kSortThreads, shared, s, a, who);
}

/** Bytes of rows that the SMs without part in a cluster's sort zero meanwhile: what they write in
 *  about the sort's time (7 us with one key a thread, 14 with four, 30 with sixteen). */
constexpr int64_t zeroedBesideSort(unsigned perThread) { return (18ll + 6ll * perThread) << 20; }

/** And those that are left to the SMs without a join, whose 10 us of dependent reads they cover, ahead of
 *  what the sums' kernel zeroes (32 MB instead of 128: 94 us instead of 90 for 4096 tokens into 65536 rows of
 *  8 KB, 112 instead of 108 for 16384, 365 instead of 359 for 131072 into as many; all that is left: 377). */
constexpr int64_t kZeroedBesideJoin = 128ll << 20;

/** ``asked``: see GradArgs; anything below kEvery withholds rows, which the waits for them then miss. */
void enqueueGrad(const eagle_b200_embedding_desc& d, const GradPlan& p, const char* who, uint32_t polls = kBulkWaits,
    uint32_t asked = kEvery)
{
    const int inBytes = elementBytes(d.values_type, who), outBytes = elementBytes(d.table_type, who);
    requireAddress(d.table, uint64_t(outBytes), who, "table");
    const cudaStream_t s = seamStream(d.stream);
    const bool accumulate = (d.flags & EAGLE_B200_EMBEDDING_ACCUMULATE) != 0;
    GradArgs a{};
    a.table = reinterpret_cast<void*>(d.table);
    a.rows = d.rows;
    a.first = d.first;
    a.tableStride = d.table_stride;
    a.dim = uint32_t(d.dim);
    a.rowBytes = d.dim * outBytes;
    a.strideBytes = d.table_stride * outBytes;
    a.zeroRows = uint32_t(std::max<int64_t>(1, kZeroUnit / a.rowBytes));
    a.zeroPieces = uint32_t((a.rowBytes + kZeroUnit - 1) / kZeroUnit);
    auto unitsOf = [&](int64_t rows) { return (rows + a.zeroRows - 1) / a.zeroRows * a.zeroPieces; };
    const int64_t sms = smCount();
    if (p.n == 0) {
        if (!accumulate) {
            zeroRowsKernel<<<gridOf(unitsOf(d.rows), who), kSumThreads, 0, s>>>(a);
            launchCheck(who);
        }
        return;
    }
    requireAddress(d.tokens, uint64_t(indexBytes(d.token_type, who)), who, "tokens");
    requireAddress(d.values, uint64_t(inBytes), who, "values");
    requireAddress(d.scratch, 256, who, "scratch");
    char* scratch = reinterpret_cast<char*>(d.scratch);
    auto words = [&](uint64_t off) { return reinterpret_cast<uint32_t*>(scratch + off); };
    a.tokens = reinterpret_cast<const void*>(d.tokens);
    a.values = reinterpret_cast<const void*>(d.values);
    a.tokenBatch = d.token_strides[0];
    a.tokenSeq = d.token_strides[1];
    a.valueBatch = d.value_strides[0];
    a.valueSeq = d.value_strides[1];
    a.valueDim = d.value_strides[2];
    a.perBatch = FastDiv(uint32_t(d.seq));
    a.flatTokens = isFlat(d.batch, d.seq, a.tokenBatch, a.tokenSeq);
    a.flatValues = isFlat(d.batch, d.seq, a.valueBatch, a.valueSeq);
    const int64_t outWord = 16 / inBytes * outBytes;
    a.tableAligned = d.table % uint64_t(outWord) == 0 && a.strideBytes % outWord == 0;
    a.accumulate = accumulate;
    a.scale = float(d.scale);
    a.n = p.n;
    a.bits = p.bits;
    a.tiles = p.tiles;
    a.bins = p.bins;
    a.digitBits = p.digitBits;
    a.chunk = p.chunk;
    a.chunks = p.chunks;
    a.group = p.group;
    a.slices = p.slices;
    a.pieces = p.pieces;
    a.polls = polls;
    a.asked = asked;
    a.lost = words(p.lost);
    a.listCount = words(p.listCount);
    a.list = words(p.list);
    a.longList = words(p.longList);
    a.head = reinterpret_cast<float*>(scratch + p.head);
    a.tail = reinterpret_cast<float*>(scratch + p.tail);
    a.width = p.width;
    a.present = accumulate ? nullptr : words(p.present);
    if (p.n <= kPortableKeys || (p.n <= kClusterKeys && largeClusters())) {
        a.keyOut = words(p.key[0]);
        a.posOut = words(p.pos[0]);
        unsigned ctas = 1;
        if (p.n > kAloneKeys)
            ctas = p.n <= kFewKeys || !largeClusters() ? 8u : unsigned(kClusterSize);
        const unsigned perThread = (p.n + ctas * unsigned(kClusterThreads) - 1) / (ctas * unsigned(kClusterThreads));
        // the SMs beside the cluster, two CTAs each, in whole clusters
        unsigned blocks = ctas;
        if (!accumulate) {
            a.zeroed = std::min(d.rows, zeroedBesideSort(perThread) / a.rowBytes);
            const int64_t besides =
                std::min<int64_t>((a.zeroed * a.rowBytes / 65536 + ctas) / ctas, 2 * sms / ctas - 1);
            if (besides > 0)
                blocks += unsigned(besides) * ctas;
            else
                a.zeroed = 0;
        }
        withIndex(d.token_type, [&](auto tok) {
            using Tok = decltype(tok);
            if (perThread <= 1)
                launchClusterSort<Tok, 1>(a, ctas, blocks, s, who);
            else if (perThread <= 2)
                launchClusterSort<Tok, 2>(a, ctas, blocks, s, who);
            else if (perThread <= 4)
                launchClusterSort<Tok, 4>(a, ctas, blocks, s, who);
            else if (perThread <= 8)
                launchClusterSort<Tok, 8>(a, ctas, blocks, s, who);
            else
                launchClusterSort<Tok, kClusterItems>(a, ctas, blocks, s, who);
        });
        a.keys = a.keyOut;
        a.order = a.posOut;
    } else {
        cudaCheck(cudaMemsetAsync(scratch, 0, p.zeroed, s), who);
        a.hist = words(p.firstHist);
        withIndex(d.token_type, [&](auto tok) {
            using Tok = decltype(tok);
            histogramKernel<Tok><<<p.tiles, kSortThreads, 0, s>>>(a);
            launchCheck(who);
            for (uint32_t k = 0; k < p.passes; ++k) {
                GradArgs b = a;
                b.shift = k * p.digitBits;
                b.hist = k == 0 ? words(p.firstHist) : words(p.hist) + size_t(k - 1) * p.tiles * p.bins;
                b.nextHist = k + 1 < p.passes ? words(p.hist) + size_t(k) * p.tiles * p.bins : nullptr;
                b.keyIn = words(p.key[(k + 1) & 1]);
                b.posIn = words(p.pos[(k + 1) & 1]);
                b.keyOut = words(p.key[k & 1]);
                b.posOut = words(p.pos[k & 1]);
                if (p.tiles > kTilesAdded) {
                    b.totals = words(p.totals);
                    launchBehind(columnScanKernel, (p.bins + 31) / 32, 1024, 0, s, b, who);
                }
                if (k == 0)
                    launchPass<true, Tok>(b, p.tiles, s, who);
                else
                    launchPass<false, Tok>(b, p.tiles, s, who);
            }
        });
        a.keys = words(p.key[(p.passes + 1) & 1]);
        a.order = words(p.pos[(p.passes + 1) & 1]);
    }
    const uint64_t lanes = uint64_t(p.chunks) * p.slices * p.group;
    if (p.bulk) {
        a.slices = uint32_t((d.dim * inBytes + kBulkSlab - 1) / kBulkSlab);
        a.sumBlocks = gridOf(int64_t(p.chunks) * a.slices, who);
    } else {
        a.sumBlocks = gridOf(int64_t((lanes + kSumThreads - 1) / kSumThreads), who);
    }
    a.zeroedBefore = d.rows;
    if (a.present != nullptr && p.chunks > 1) {
        const int64_t left = (d.rows - a.zeroed) * a.rowBytes;
        a.zeroedBefore -= std::min(kZeroedBesideJoin, left) / a.rowBytes;
    }
    const int64_t zeroing = a.present == nullptr ? 0 : unitsOf(a.zeroedBefore - a.zeroed);
    const unsigned blocks = gridOf(int64_t(a.sumBlocks) + zeroing, who);
    withElement(d.values_type, [&](auto in) {
        withElement(d.table_type, [&](auto out) {
            using In = decltype(in);
            using Out = decltype(out);
            if (p.bulk && p.piece == Piece::Aligned)
                launchBulkSum<In, Out, true>(a, blocks, s, who);
            else if (p.bulk)
                launchBulkSum<In, Out, false>(a, blocks, s, who);
            else if (p.piece == Piece::Aligned)
                launchSum<In, Out, Piece::Aligned>(a, blocks, s, who);
            else if (p.piece == Piece::Shifted)
                launchSum<In, Out, Piece::Shifted>(a, blocks, s, who);
            else
                launchSum<In, Out, Piece::Strided>(a, blocks, s, who);
        });
    });
    if (p.chunks > 1) {
        const int64_t items = int64_t(p.chunks / 2) * ((d.dim + kJoinColumns - 1) / kJoinColumns);
        a.joinLanes = 4;
        while (a.joinLanes < 32 && a.joinLanes * 4 < a.dim)
            a.joinLanes *= 2;
        a.joinBlocks = unsigned(std::min<int64_t>(items, sms * 8));
        const unsigned all = gridOf(a.joinBlocks + (a.present == nullptr ? 0 : unitsOf(d.rows - a.zeroedBefore)), who);
        withElement(d.table_type,
            [&](auto out) { launchBehind(joinKernel<decltype(out)>, all, kJoinThreads, 0, s, a, who); });
    }
}

}  // namespace
}  // namespace eb

using namespace eb;

EB_API eagle_backend_status eagle_backend_x_b200_embedding_grad(eagle_b200_embedding_desc* desc)
{
    return guarded([&] {
        const char* who = "eagle_backend_x_b200_embedding_grad";
        const eagle_b200_embedding_desc d = readDesc(desc, EAGLE_B200_EMBEDDING_ACCUMULATE, who);
        if (desc->struct_size < sizeof d)
            invalid(std::string(who) + ": struct_size too small for the query's answer");
        checkEmbedding(d, who);
        const GradPlan p = planGrad(d, who);
        if (d.scratch == 0) {
            desc->scratch_bytes = int64_t(p.bytes);
            return;
        }
        if (d.rows == 0 || d.dim == 0)
            return;
        requireDevice();
        DeviceScope scope(resolveDevice(d.device, d.table));
        enqueueGrad(d, p, who);
    });
}

EB_API eagle_backend_status eagle_backend_x_b200_embedding_grad_wait_check(eagle_b200_embedding_desc* desc,
    uint32_t polls, uint32_t asked)
{
    return guarded([&] {
        const char* who = "eagle_backend_x_b200_embedding_grad_wait_check";
        const eagle_b200_embedding_desc d = readDesc(desc, EAGLE_B200_EMBEDDING_ACCUMULATE, who);
        checkEmbedding(d, who);
        const GradPlan p = planGrad(d, who);
        if (p.n == 0 || d.rows == 0 || d.dim == 0 || !p.bulk)
            invalid(std::string(who) + ": needs tokens, and rows long enough for the copy engine");
        if (polls == 0 || polls > kBulkWaits)
            invalid(std::string(who) + ": polls must lie in [1, 2^22]");
        if (d.scratch == 0)
            invalid(std::string(who) + ": needs embedding_grad's scratch (query it there)");
        requireDevice();
        DeviceScope scope(resolveDevice(d.device, d.table));
        enqueueGrad(d, p, who, polls, asked);
    });
}
