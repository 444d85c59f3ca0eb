// The embedding rows of a batch's tokens:
//
//   values[t, :] = round(scale * table[token[t] - first, :])
//
// A gather of rows in 16-byte pieces, several in flight per lane: HBM bounds it (65536 rows of
// 16 KB to bf16: 155 us, 5.6 TB/s of what it has to move, 6.0 of DRAM traffic), or the launch
// where there are few tokens (64: 3.4 us).
#include "sequences.cuh"

#define EB_API extern "C" __attribute__((visibility("default")))

namespace eb {
namespace {

// ------------------------------------------------------------------ lookup

struct LookupArgs {
    const void* table;
    const void* tokens;
    void* values;
    int64_t rows, first;
    int64_t tableStride;
    int64_t tokenBatch, tokenSeq;  // strides of the ids
    int64_t valueBatch, valueSeq;  // strides of the outputs
    int64_t n;                     // tokens
    uint32_t dim;
    uint32_t pieces;               // packs per row
    FastDiv perRow;                // by pieces
    FastDiv perBatch;              // by seq
    bool flat;                     // one stride serves batch and seq
    float scale;
};

constexpr int kLookupThreads = 256;

/** The row of token ``t``, or -1 where the table has none. */
template <class Tok>
__device__ __forceinline__ int64_t rowOfToken(const void* tokens, int64_t at, int64_t first, int64_t rows)
{
    const int64_t id = int64_t(reinterpret_cast<const Tok*>(tokens)[at]);
    if (id < first)
        return -1;
    const uint64_t r = uint64_t(id) - uint64_t(first);  // first >= 0, so the difference is exact
    return r < uint64_t(rows) ? int64_t(r) : -1;
}

/** Where a thread's packs read and write: token t's row (-1: none) and output vector. */
template <class Tok>
__device__ __forceinline__ void placeOf(const LookupArgs& a, int64_t t, int64_t& row, int64_t& to)
{
    const uint32_t b = a.flat ? 0u : a.perBatch(uint32_t(t));
    const int64_t s = t - int64_t(b) * a.perBatch.d;
    row = rowOfToken<Tok>(a.tokens, int64_t(b) * a.tokenBatch + s * a.tokenSeq, a.first, a.rows);
    to = int64_t(b) * a.valueBatch + s * a.valueSeq;
}

// Narrow rows: the packs of all of them in a row, so that no lane idles.

/** ``Unroll`` packs of N values per thread, a CTA's width apart: neighbouring threads hold
 *  neighbouring packs of the flattened (token, column) plane, so loads and stores are
 *  whole lines whatever the row length, and short rows leave no lane idle. */
template <class In, class Out, class Tok, int N, int Unroll>
__global__ __launch_bounds__(kLookupThreads) void lookupKernel(LookupArgs a)
{
    letNextKernelStart();
    waitForKernelBefore();
    const int64_t base = int64_t(blockIdx.x) * (kLookupThreads * Unroll);
    const int64_t row0 = base / a.pieces;
    const uint32_t col0 = uint32_t(base - row0 * a.pieces);
    const In* table = reinterpret_cast<const In*>(a.table);
    Out* values = reinterpret_cast<Out*>(a.values);
    int64_t from[Unroll], to[Unroll];
    bool inside[Unroll];
#pragma unroll
    for (int u = 0; u < Unroll; ++u) {
        const uint32_t k = col0 + uint32_t(u) * kLookupThreads + threadIdx.x;
        const uint32_t down = a.perRow(k);
        const uint32_t col = (k - down * a.pieces) * N;
        inside[u] = row0 + down < a.n;
        int64_t row;
        placeOf<Tok>(a, min(row0 + down, a.n - 1), row, to[u]);
        from[u] = row < 0 ? -1 : row * a.tableStride + col;
        to[u] += col;
    }
    Pack<In, N> got[Unroll];
#pragma unroll
    for (int u = 0; u < Unroll; ++u)
        if (from[u] >= 0)
            got[u] = *reinterpret_cast<const Pack<In, N>*>(table + from[u]);
#pragma unroll
    for (int u = 0; u < Unroll; ++u) {
        if (!inside[u])
            continue;
        Pack<Out, N> out;
#pragma unroll
        for (int e = 0; e < N; ++e)
            out.e[e] = fromFloat<Out>(from[u] >= 0 ? toFloat(got[u].e[e]) * a.scale : 0.0f);
        storePack(values + to[u], out);
    }
}

/** Rows of odd length or alignment: packs are cut where the output's 16-byte words begin, and the
 *  row is read from wherever that falls as aligned words shifted together (element by
 *  element, as the at most two incomplete packs of a row still are, took four times as long).
 *  A row of dim values has up to ceil(dim / N) + 1 packs, the first ending at its first word. */
template <class In, class Out, class Tok, int N, int Unroll>
__global__ __launch_bounds__(kLookupThreads) void lookupShiftedKernel(LookupArgs a)
{
    letNextKernelStart();
    waitForKernelBefore();
    const int64_t base = int64_t(blockIdx.x) * (kLookupThreads * Unroll);
    const int64_t row0 = base / a.pieces;
    const uint32_t col0 = uint32_t(base - row0 * a.pieces);
    const In* table = reinterpret_cast<const In*>(a.table);
    Out* values = reinterpret_cast<Out*>(a.values);
    const int dim = int(a.dim);
    const In* from[Unroll];
    Out* to[Unroll];
    int begin[Unroll];  // the pack's first column, of the row's dim
#pragma unroll
    for (int u = 0; u < Unroll; ++u) {
        const uint32_t k = col0 + uint32_t(u) * kLookupThreads + threadIdx.x;
        const uint32_t down = a.perRow(k);
        int64_t row, at;
        placeOf<Tok>(a, min(row0 + down, a.n - 1), row, at);
        to[u] = values + at;
        from[u] = row < 0 ? nullptr : table + row * a.tableStride;
        const int lead = int((0u - uint32_t(reinterpret_cast<uint64_t>(to[u]))) & 15u) / int(sizeof(Out));
        begin[u] = row0 + down < a.n ? lead + (int(k - down * a.pieces) - 1) * N : dim;
    }
    constexpr int kWords = N * int(sizeof(In)) / 16;
    uint4 got[Unroll][kWords];
#pragma unroll
    for (int u = 0; u < Unroll; ++u)
        if (from[u] != nullptr && begin[u] >= 0 && begin[u] + N <= dim)
#pragma unroll
            for (int w = 0; w < kWords; ++w)
                got[u][w] = loadShifted(from[u] + begin[u] + w * (N / kWords), 16u);
#pragma unroll
    for (int u = 0; u < Unroll; ++u) {
        if (begin[u] >= 0 && begin[u] + N <= dim) {
            const Pack<In, N>& in = *reinterpret_cast<const Pack<In, N>*>(&got[u]);
            Pack<Out, N> out;
#pragma unroll
            for (int e = 0; e < N; ++e)
                out.e[e] = fromFloat<Out>(from[u] != nullptr ? toFloat(in.e[e]) * a.scale : 0.0f);
            *reinterpret_cast<Pack<Out, N>*>(to[u] + begin[u]) = out;
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const int col = begin[u] + e;
                if (col >= 0 && col < dim)
                    to[u][col] = fromFloat<Out>(from[u] != nullptr ? toFloat(from[u][col]) * a.scale : 0.0f);
            }
        }
    }
}

// Wide rows (32 packs and more): a warp takes 32 * Unroll packs of one row, so that the row, its
// addresses and its alignment are worked out once for all of them. Worked out per pack, as
// for the narrow ones, that took more time than the bytes: 210 us against 155 at 65536 rows of
// 16 KB, and 20 against 8 at 10007 of 2002 bytes.

/** ``Shifted``: packs are cut where the output's words (of 16 bytes, or 32 if the table's type is the
 *  narrower) begin and read from wherever that falls in the table; the up to N - 1 values before the first and after the last are taken
 *  one to a lane. */
template <class In, class Out, class Tok, int N, int Unroll, bool Shifted>
__global__ __launch_bounds__(kLookupThreads) void lookupWideKernel(LookupArgs a)
{
    letNextKernelStart();
    waitForKernelBefore();
    const uint32_t lane = threadIdx.x & 31u;
    const uint32_t id = blockIdx.x * (kLookupThreads / 32) + (threadIdx.x >> 5);
    const int64_t t = a.perRow(id);  // pieces: warps to a row
    if (t >= a.n)
        return;
    const uint32_t segment = id - uint32_t(t) * a.pieces;
    int64_t row, at;
    placeOf<Tok>(a, t, row, at);
    const In* from = reinterpret_cast<const In*>(a.table) + (row < 0 ? 0 : row * a.tableStride);
    Out* to = reinterpret_cast<Out*>(a.values) + at;
    uint32_t lead = 0;
    if constexpr (Shifted)
        lead = min(((0u - uint32_t(reinterpret_cast<uint64_t>(to))) & (N * uint32_t(sizeof(Out)) - 1u))
                / uint32_t(sizeof(Out)),
            a.dim);
    const uint32_t whole = (a.dim - lead) / N;
    const uint32_t pack0 = segment * (32u * Unroll) + lane;
    constexpr int kWords = N * int(sizeof(In)) / 16;
    uint4 got[Unroll][kWords];
    if (row >= 0) {
#pragma unroll
        for (int u = 0; u < Unroll; ++u) {
            if (pack0 + 32u * u < whole) {
                const In* p = from + lead + (pack0 + 32u * u) * N;
#pragma unroll
                for (int w = 0; w < kWords; ++w) {
                    if constexpr (Shifted)
                        got[u][w] = loadShifted(p + w * (N / kWords), 16u);
                    else if constexpr (kWords == 1)
                        got[u][w] = *reinterpret_cast<const uint4*>(p);
                    else if (w == 0)
                        load32(p, got[u][0], got[u][kWords - 1]);
                }
            }
        }
    }
#pragma unroll
    for (int u = 0; u < Unroll; ++u) {
        if (pack0 + 32u * u < whole) {
            const Pack<In, N>& in = *reinterpret_cast<const Pack<In, N>*>(&got[u]);
            Pack<Out, N> out;
#pragma unroll
            for (int e = 0; e < N; ++e)
                out.e[e] = fromFloat<Out>(row >= 0 ? toFloat(in.e[e]) * a.scale : 0.0f);
            Out* p = to + lead + (pack0 + 32u * u) * N;
            if constexpr (sizeof(out) == 16)
                __stcs(reinterpret_cast<uint4*>(p), *reinterpret_cast<const uint4*>(&out));  // L2 is for the rows
            else
                storePack(p, out);
        }
    }
    if constexpr (Shifted) {
        const uint32_t col = lane < 16u ? lane : lead + whole * N + lane - 16u;
        if (segment == 0 && col < (lane < 16u ? lead : a.dim))
            to[col] = fromFloat<Out>(row >= 0 ? toFloat(from[col]) * a.scale : 0.0f);
    }
}

// ------------------------------------------------------------------ host side

template <class In, class Out, class Tok, int N, bool Shifted>
void launchLookup(LookupArgs a, cudaStream_t s, const char* who)
{
    const int64_t packs = a.dim / N;
    const int64_t sms = smCount();
    if (packs >= 32) {
        // four packs a lane keep the memory busy; a plane too small to give every SM a few CTAs
        // of those takes one each, so that more SMs share it
        const int unroll = a.n * packs >= sms * 2 * kLookupThreads * 4 ? 4 : 1;
        a.pieces = uint32_t((packs + 32 * unroll - 1) / (32 * unroll));
        a.perRow = FastDiv(a.pieces);
        const int64_t warps = a.n * a.pieces;
        if (warps > 0x7fffff00ll)
            unsupported(std::string(who) + ": the call is larger than one launch holds");
        const unsigned blocks = unsigned((warps + kLookupThreads / 32 - 1) / (kLookupThreads / 32));
        if (unroll == 1)
            launchBehind(lookupWideKernel<In, Out, Tok, N, 1, Shifted>, blocks, kLookupThreads, 0, s, a, who);
        else
            launchBehind(lookupWideKernel<In, Out, Tok, N, 4, Shifted>, blocks, kLookupThreads, 0, s, a, who);
    } else {
        a.pieces = Shifted ? (a.dim + N - 1) / N + 1 : a.dim / N;
        a.perRow = FastDiv(a.pieces);
        const int64_t all = a.n * int64_t(a.pieces);
        const int unroll = all >= sms * 2 * kLookupThreads * 4 ? 4 : 1;
        const unsigned blocks = gridOf((all + kLookupThreads * unroll - 1) / (kLookupThreads * unroll), who);
        if (Shifted && unroll == 1)
            launchBehind(lookupShiftedKernel<In, Out, Tok, N, 1>, blocks, kLookupThreads, 0, s, a, who);
        else if (Shifted)
            launchBehind(lookupShiftedKernel<In, Out, Tok, N, 4>, blocks, kLookupThreads, 0, s, a, who);
        else if (unroll == 1)
            launchBehind(lookupKernel<In, Out, Tok, N, 1>, blocks, kLookupThreads, 0, s, a, who);
        else
            launchBehind(lookupKernel<In, Out, Tok, N, 4>, blocks, kLookupThreads, 0, s, a, who);
    }
    launchCheck(who);
}

void enqueueLookup(const eagle_b200_embedding_desc& d, const char* who)
{
    const int inBytes = elementBytes(d.table_type, who), outBytes = elementBytes(d.values_type, who);
    requireAddress(d.tokens, uint64_t(indexBytes(d.token_type, who)), who, "tokens");
    requireAddress(d.values, uint64_t(outBytes), who, "values");
    if (d.rows > 0)
        requireAddress(d.table, uint64_t(inBytes), who, "table");
    if (d.dim > 1 && d.value_strides[2] != 1)
        invalid(std::string(who) + ": a vector's values must be contiguous");
    LookupArgs a{};
    a.table = reinterpret_cast<const void*>(d.table);
    a.tokens = reinterpret_cast<const void*>(d.tokens);
    a.values = reinterpret_cast<void*>(d.values);
    a.rows = d.rows;
    a.first = d.first;
    a.tableStride = d.table_stride;
    a.tokenBatch = d.token_strides[0];
    a.tokenSeq = d.token_strides[1];
    a.valueBatch = d.value_strides[0];
    a.valueSeq = d.value_strides[1];
    a.n = d.batch * d.seq;
    a.dim = uint32_t(d.dim);
    a.perBatch = FastDiv(uint32_t(d.seq));
    a.flat = isFlat(d.batch, d.seq, a.tokenBatch, a.tokenSeq) && isFlat(d.batch, d.seq, a.valueBatch, a.valueSeq);
    a.scale = float(d.scale);
    const cudaStream_t s = seamStream(d.stream);
    withElement(d.table_type, [&](auto in) {
        withElement(d.values_type, [&](auto out) {
            withIndex(d.token_type, [&](auto tok) {
                using In = decltype(in);
                using Out = decltype(out);
                using Tok = decltype(tok);
                // a pack is 16 bytes of the narrower type; every row has to start on its words
                constexpr int N = 16 / int(sizeof(In) < sizeof(Out) ? sizeof(In) : sizeof(Out));
                constexpr int64_t kInPack = N * int(sizeof(In)), kOutPack = N * int(sizeof(Out));
                const bool wide = d.dim % N == 0 && d.table % kInPack == 0 && d.values % kOutPack == 0
                    && d.table_stride * inBytes % kInPack == 0 && d.value_strides[0] * outBytes % kOutPack == 0
                    && d.value_strides[1] * outBytes % kOutPack == 0;
                if (wide)
                    launchLookup<In, Out, Tok, N, false>(a, s, who);
                else
                    launchLookup<In, Out, Tok, N, true>(a, s, who);
            });
        });
    });
}

}  // namespace
}  // namespace eb

using namespace eb;

EB_API eagle_backend_status eagle_backend_x_b200_embedding(const eagle_b200_embedding_desc* desc)
{
    return guarded([&] {
        const char* who = "eagle_backend_x_b200_embedding";
        const eagle_b200_embedding_desc d = readDesc(desc, 0u, who);
        checkEmbedding(d, who);
        if (d.batch * d.seq == 0 || d.dim == 0)
            return;
        requireDevice();
        DeviceScope scope(resolveDevice(d.device, d.values));
        enqueueLookup(d, who);
    });
}
