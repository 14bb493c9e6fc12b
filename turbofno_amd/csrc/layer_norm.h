// What the layer norm and its gradient share.
#pragma once
#include "eight_bits.h"
#include "philox.h"
#include <algorithm>

namespace tfno {

// narrow strips up to here, as in the root-mean-square norm
constexpr long kFewColumns = 1L << 17;                  // real columns
constexpr long kNarrowColumns = 8192;                   // strips of 8 to 32 columns up to here
// a lane's part of an address in 32 bits: up to 31 channels, with 2 lanes side by side
inline bool far_apart(long ld) { return ld >= (1L << 30) / 32; }
constexpr int kChunk = 8;                               // channels of a lane whose loads overlap where not all are held

// with dropout, what a lane keeps of its columns
struct KeepAll { };
template <bool COMPLEX, bool DROP> __device__ __forceinline__ auto keep_of(const Drop& drop, long column)
{
    if constexpr (DROP) return Keep<COMPLEX>(drop, column);
    else return KeepAll();
}

// Rows of a strip, COUNT at a time: f(whole) loads them all, with Strip's accesses for whole strips (whole: a lane's four columns exist) or value by value. A lane's columns
// decide, once for all rows: a branch for each would wait for each. Lanes without columns load nothing.
template <bool FULL, typename F> __device__ __forceinline__ void for_lane(int lane_there, F f)
{
    if constexpr (FULL) f(std::true_type());
    else if (lane_there >= 4) f(std::true_type());
    else if (lane_there > 0) f(std::false_type());
}
template <int IN, bool FULL, typename S>
__device__ __forceinline__ void write_row(const S& strip, void* base, long ld, long column0, int there, int r, RawOf<IN> v)
{
    for_lane<FULL>(there - 4 * strip.lane, [&](auto whole) { strip.template write<IN, decltype(whole)::value>(base, ld, column0, there, r, v); });
}

}  // namespace tfno
