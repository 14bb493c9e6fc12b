// Four consecutive real values of a channel's row, as a lane of the operators around the spectral layer reads and writes them: 32-bit, bf16 or
// e4m3 in memory. Rows start at any multiple of a value's size and end anywhere.
#pragma once
#include "bf16_split.h"
#include "operators.h"

namespace tfno {

enum { kIn32 = 0, kIn16 = 1, kIn8 = 2 };                // 32-bit, bf16 and e4m3 values

template <int IN> struct Columns;
template <> struct Columns<kIn32> { typedef float4_v Raw; typedef float Value; };
template <> struct Columns<kIn16> { typedef uint2_v Raw; typedef unsigned short Value; };
template <> struct Columns<kIn8> { typedef unsigned Raw; typedef unsigned char Value; };
template <int IN> using RawOf = typename Columns<IN>::Raw;

// Rows start at any multiple of a value's size: the vector accesses say so
typedef float4_v float4_any __attribute__((aligned(4)));
typedef uint2_v uint2_any __attribute__((aligned(2)));
typedef unsigned uint_any __attribute__((aligned(1)));
typedef uint2_v uint2_bytes __attribute__((aligned(1)));
template <int IN> __device__ __forceinline__ RawOf<IN> load4(const void* row, long column)
{
    const auto* p = static_cast<const typename Columns<IN>::Value*>(row) + column;
    if constexpr (IN == kIn32) return *reinterpret_cast<const float4_any*>(p);
    else if constexpr (IN == kIn16) return *reinterpret_cast<const uint2_any*>(p);
    else return *reinterpret_cast<const uint_any*>(p);
}
// the same where the row may end inside: its last value stands for what lies beyond
template <int IN> __device__ __forceinline__ RawOf<IN> load4_ragged(const void* row, long column, long columns)
{
    const auto* p = static_cast<const typename Columns<IN>::Value*>(row);
    auto at = [&](int i) { return p[column + i < columns ? column + i : columns - 1]; };
    if constexpr (IN == kIn32) return (float4_v){ at(0), at(1), at(2), at(3) };
    else if constexpr (IN == kIn16) return (uint2_v){ at(0) | (unsigned)at(1) << 16, at(2) | (unsigned)at(3) << 16 };
    else return at(0) | (unsigned)at(1) << 8 | (unsigned)at(2) << 16 | (unsigned)at(3) << 24;
}
template <int IN> __device__ __forceinline__ float4_v to_float(RawOf<IN> v)
{
    if constexpr (IN == kIn32) return v;
    else return (float4_v){ __builtin_bit_cast(float, v[0] << 16), __builtin_bit_cast(float, v[0] & 0xffff0000u),
                            __builtin_bit_cast(float, v[1] << 16), __builtin_bit_cast(float, v[1] & 0xffff0000u) };
}
template <int IN> __device__ __forceinline__ RawOf<IN> from_float(float4_v v)
{
    if constexpr (IN == kIn32) return v;
    else return (uint2_v){ __builtin_bit_cast(unsigned, __builtin_convertvector((float2_v){ v[0], v[1] }, bf16x2_t)),
                           __builtin_bit_cast(unsigned, __builtin_convertvector((float2_v){ v[2], v[3] }, bf16x2_t)) };
}
template <int IN> __device__ __forceinline__ void store4(void* row, long column, RawOf<IN> v)
{
    auto* p = static_cast<typename Columns<IN>::Value*>(row) + column;
    if constexpr (IN == kIn32) *reinterpret_cast<float4_any*>(p) = v;
    else *reinterpret_cast<uint2_any*>(p) = v;
}
template <int IN> __device__ __forceinline__ void store4_ragged(void* row, long column, long columns, RawOf<IN> v)
{
    auto* p = static_cast<typename Columns<IN>::Value*>(row);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (column + i < columns) {
            if constexpr (IN == kIn32) p[column + i] = v[i];
            else if constexpr (IN == kIn16) p[column + i] = (unsigned short)(i & 1 ? v[i / 2] >> 16 : v[i / 2]);
            else p[column + i] = (unsigned char)(v >> 8 * i);
        }
}
// for results that are larger than the caches, or are not read again soon: they do not displace what is
template <int IN> __device__ __forceinline__ void store4_past_caches(void* row, long column, RawOf<IN> v)
{
    auto* p = static_cast<typename Columns<IN>::Value*>(row) + column;
    if constexpr (IN == kIn32) __builtin_nontemporal_store(v, reinterpret_cast<float4_any*>(p));
    else __builtin_nontemporal_store(v, reinterpret_cast<uint2_any*>(p));
}
template <int IN> __device__ __forceinline__ RawOf<IN> zero4()
{
    if constexpr (IN == kIn32) return (float4_v){ 0.f, 0.f, 0.f, 0.f };
    else if constexpr (IN == kIn16) return (uint2_v){ 0u, 0u };
    else return 0u;
}
// The same at an address of two parts: one for the whole wave, in scalar registers, and the lane's, of 32 bits. Kept apart from the compiler, which
// would add them per lane ahead of a loop and hold the 64-bit sums of every row in vector registers.
#define TFNO_GLOBAL __attribute__((address_space(1)))
typedef const TFNO_GLOBAL char* ScalarAddress;
__device__ __forceinline__ long scalar(long v)
{
    const unsigned lo = __builtin_amdgcn_readfirstlane((int)v), hi = __builtin_amdgcn_readfirstlane((int)(v >> 32));
    return (long)((unsigned long)hi << 32 | lo);
}
__device__ __forceinline__ ScalarAddress scalar(const void* base, long bytes) { return reinterpret_cast<ScalarAddress>(scalar(reinterpret_cast<long>(base) + bytes)); }
// a copy that the compiler does not know: what is made of it, its extension to 64 bits too, stays beside the access (which takes 32) instead of in
// registers of its own from ahead of a loop
__device__ __forceinline__ unsigned fresh(unsigned offset)
{
    asm volatile("" : "+v"(offset));
    return offset;
}
template <int IN> __device__ __forceinline__ RawOf<IN> near_load4(ScalarAddress base, unsigned offset)
{
    if constexpr (IN == kIn32) return *reinterpret_cast<const TFNO_GLOBAL float4_any*>(base + offset);
    else if constexpr (IN == kIn16) return *reinterpret_cast<const TFNO_GLOBAL uint2_any*>(base + offset);
    else return *reinterpret_cast<const TFNO_GLOBAL uint_any*>(base + offset);
}
template <int IN> __device__ __forceinline__ void near_store4(ScalarAddress base, unsigned offset, RawOf<IN> v)
{
    if constexpr (IN == kIn32) *(TFNO_GLOBAL float4_any*)(base + offset) = v;
    else if constexpr (IN == kIn16) *(TFNO_GLOBAL uint2_any*)(base + offset) = v;
    else *(TFNO_GLOBAL uint_any*)(base + offset) = v;
}
// Is one of the values below the range of the split (bf16_split.h), but not zero, in any lane: uniform. One minimum per two values; zeros are told
// apart where there are any
template <int COUNT> __device__ __forceinline__ bool below_split_range(const float4_v (&v)[COUNT])
{
    float low = 1.f;
#pragma unroll
    for (int j = 0; j < COUNT; ++j) low = smaller(smaller(low, v[j][0], v[j][1]), v[j][2], v[j][3]);
    if (__builtin_expect(!any_lane(low < kSplitSmallest), 1)) return false;
    unsigned bits = ~0u;
#pragma unroll
    for (int j = 0; j < COUNT; ++j) bits = lower(lower(bits, float2{ v[j][0], v[j][1] }), float2{ v[j][2], v[j][3] });
    return any_lane(bits < kSplitLow);
}
__device__ __forceinline__ float4_v mfma_fp32(float a, float b, float4_v c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

__device__ __forceinline__ float value_of(float v) { return v; }
__device__ __forceinline__ float value_of(unsigned short v) { return __builtin_bit_cast(float, (unsigned)v << 16); }

}  // namespace tfno
