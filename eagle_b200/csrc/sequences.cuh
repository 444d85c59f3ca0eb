// Shared pieces of the token-sequence operators (embedding.cu, paged.cu): element
// conversions, division by a launch constant and the checks of their descs.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace eb {

// ------------------------------------------------------------- launch-constant division

/** Quotient by a divisor fixed at launch, for dividends below 2^31: with l = ceil(log2 d)
 *  and m = floor(2^32 (2^l - d) / d) + 1, n / d = (mulhi(n, m) + n) >> l (Granlund and
 *  Montgomery, "Division by invariant integers using multiplication", 1994). */
struct FastDiv {
    uint32_t d = 1, mul = 1, shift = 0;
    FastDiv() = default;
    explicit FastDiv(uint32_t div)
        : d(div)
    {
        while ((uint64_t(1) << shift) < div)
            ++shift;
        mul = uint32_t(((uint64_t(1) << 32) * ((uint64_t(1) << shift) - div)) / div + 1);
    }
    __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return (__umulhi(n, mul) + n) >> shift; }
};

// ------------------------------------------------------------- elements

template <class T>
__device__ __forceinline__ float toFloat(T v);
template <>
__device__ __forceinline__ float toFloat<float>(float v)
{
    return v;
}
template <>
__device__ __forceinline__ float toFloat<__nv_bfloat16>(__nv_bfloat16 v)
{
    return __bfloat162float(v);
}
template <>
__device__ __forceinline__ float toFloat<__half>(__half v)
{
    return __half2float(v);
}

/** The one rounding of a result, to nearest even. */
template <class T>
__device__ __forceinline__ T fromFloat(float v);
template <>
__device__ __forceinline__ float fromFloat<float>(float v)
{
    return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 fromFloat<__nv_bfloat16>(float v)
{
    return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half fromFloat<__half>(float v)
{
    return __float2half_rn(v);
}

/** N neighbouring elements, moved as words of up to 16 bytes. */
template <class T, int N>
struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Pack {
    T e[N];
};

/** 32 bytes in one load; ``p`` is 32-byte aligned. (Two of 16 touch every sector of a warp's twice.) */
__device__ __forceinline__ void load32(const void* p, uint4& lo, uint4& hi)
{
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(lo.x), "=r"(lo.y), "=r"(lo.z), "=r"(lo.w), "=r"(hi.x), "=r"(hi.y), "=r"(hi.z), "=r"(hi.w)
                 : "l"(p));
}

/** A pack of 8, 16 or 32 bytes in one store to an address aligned to as much. */
template <class T, int N>
__device__ __forceinline__ void storePack(T* to, const Pack<T, N>& p)
{
    if constexpr (sizeof(p) == 32) {
        const uint4* w = reinterpret_cast<const uint4*>(&p);
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(w[0].x), "r"(w[0].y),
                     "r"(w[0].z), "r"(w[0].w), "r"(w[1].x), "r"(w[1].y), "r"(w[1].z), "r"(w[1].w)
                     : "memory");
    } else {
        *reinterpret_cast<Pack<T, N>*>(to) = p;
    }
}

/** The 16 bytes ``skip`` into 32 neighbouring ones. */
__device__ __forceinline__ uint4 shiftWords(uint4 lo, uint4 hi, uint32_t skip)
{
    uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    if (skip & 8u) {
#pragma unroll
        for (int j = 0; j < 6; ++j)
            w[j] = w[j + 2];
    }
    if (skip & 4u) {
#pragma unroll
        for (int j = 0; j < 5; ++j)
            w[j] = w[j + 1];
    }
    const uint32_t shift = (skip & 3u) * 8u;
    return make_uint4(__funnelshift_r(w[0], w[1], shift), __funnelshift_r(w[1], w[2], shift),
        __funnelshift_r(w[2], w[3], shift), __funnelshift_r(w[3], w[4], shift));
}

/** 16 bytes from any address of whole elements, of which ``valid`` bytes are wanted: the one or
 *  two aligned words that hold them (each holds a wanted byte, so it lies in mapped memory),
 *  shifted together. What lies past ``valid`` is unspecified. */
__device__ __forceinline__ uint4 loadShifted(const void* p, uint32_t valid)
{
    const uint64_t at = reinterpret_cast<uint64_t>(p);
    const uint4* word = reinterpret_cast<const uint4*>(at & ~uint64_t(15));
    const uint32_t skip = uint32_t(at) & 15u;
    const uint4 lo = *word;
    const uint4 hi = skip + valid > 16u ? word[1] : make_uint4(0u, 0u, 0u, 0u);
    return shiftWords(lo, hi, skip);
}

// ------------------------------------------------------------- kernels in a row
//
// Kernels are launched while whatever runs before them, another of the call's or anything else on
// the stream, may still be running (programmatic dependent launch), so that their CTAs are in
// place when their turn comes. Such a kernel touches no memory before ``waitForKernelBefore``,
// which returns once every kernel before it has ended and its writes are visible; one of these
// lets the next start with ``letNextKernelStart``, early, which takes effect when all of its
// CTAs are running. Launched in plain order, and so without the wait: histogramKernel, behind a
// memset, and zeroRowsKernel.

// Since what such a kernel reads may be written while it waits, none of it is read through the
// non-coherent path (__ldg): plain loads, or past L1 (__ldcg).

__device__ __forceinline__ void waitForKernelBefore() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void letNextKernelStart() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

/** Launch ``kernel(args)``, which starts with waitForKernelBefore, behind whatever the stream has before it. */
template <class Args>
void launchBehind(void (*kernel)(Args), unsigned blocks, unsigned threads, size_t shared, cudaStream_t s,
    const Args& args, const char* who)
{
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(blocks, 1, 1);
    config.blockDim = dim3(threads, 1, 1);
    config.dynamicSmemBytes = shared;
    config.stream = s;
    config.attrs = &attr;
    config.numAttrs = 1;
    cudaCheck(cudaLaunchKernelEx(&config, kernel, args), who);
}

// ------------------------------------------------------------- host side

inline int elementBytes(uint32_t type, const char* who)
{
    switch (type) {
    case EAGLE_B200_TYPE_F32: return 4;
    case EAGLE_B200_TYPE_BF16:
    case EAGLE_B200_TYPE_F16: return 2;
    default: unsupported(std::string(who) + ": element type " + std::to_string(type) + " is not F32, BF16 or F16");
    }
}

inline int indexBytes(uint32_t type, const char* who)
{
    switch (type) {
    case EAGLE_B200_TYPE_I32: return 4;
    case EAGLE_B200_TYPE_I64: return 8;
    default: unsupported(std::string(who) + ": index type " + std::to_string(type) + " is not I32 or I64");
    }
}

/** ``p`` is an address whose elements of ``bytes`` are aligned. */
inline void requireAddress(uint64_t p, uint64_t bytes, const char* who, const char* what)
{
    if (p == 0 || p % bytes != 0)
        invalid(std::string(who) + ": " + what + " must be a device address aligned to " + std::to_string(bytes)
            + " bytes");
}

/** A grid of ``want`` blocks, refused where it passes the launch limit. */
inline unsigned gridOf(int64_t want, const char* who)
{
    if (want > 0x7fffffffll)
        unsupported(std::string(who) + ": the call is larger than one launch holds");
    return unsigned(want);
}

/** What the embedding's entries refuse. */
inline void checkEmbedding(const eagle_b200_embedding_desc& d, const char* who)
{
    const std::string w(who);
    (void)elementBytes(d.table_type, who);
    (void)elementBytes(d.values_type, who);
    (void)indexBytes(d.token_type, who);
    if (d.rows < 0 || d.rows > 0x7ffffffell)
        invalid(w + ": rows must lie in [0, 2^31 - 2]");
    if (d.dim < 0 || d.dim > (1ll << 24))
        invalid(w + ": dim must lie in [0, 2^24]");
    if (d.first < 0)
        invalid(w + ": first must not be negative");
    if (d.batch < 0 || d.seq < 0 || d.batch > 0x7fffffffll || d.seq > 0x7fffffffll || d.batch * d.seq > 0x7fffffffll)
        invalid(w + ": batch * seq must lie in [0, 2^31 - 1]");
    if (d.rows > 1 && d.table_stride < d.dim)
        invalid(w + ": the table's rows overlap (table_stride below dim)");
}

/** One stride serves both token axes. */
inline bool isFlat(int64_t batch, int64_t seq, int64_t outer, int64_t inner) { return batch <= 1 || outer == seq * inner; }

template <class F>
void withElement(uint32_t type, F&& f)
{
    if (type == EAGLE_B200_TYPE_F32)
        f(float{});
    else if (type == EAGLE_B200_TYPE_BF16)
        f(__nv_bfloat16{});
    else
        f(__half{});
}

template <class F>
void withIndex(uint32_t type, F&& f)
{
    if (type == EAGLE_B200_TYPE_I32)
        f(int32_t{});
    else
        f(int64_t{});
}

}  // namespace eb
