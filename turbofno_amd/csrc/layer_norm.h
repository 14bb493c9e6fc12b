// What the layer norm and its gradient share.
#pragma once
#include "eight_bits.h"
#include "philox.h"
#include <algorithm>

namespace tfno {

// narrow strips up to here, as in the root-mean-square norm
constexpr long kFewColumns = 1L << 17;                  // real columns
constexpr int kChunk = 8;                               // channels of a lane whose loads overlap where not all are held

// with dropout, what a lane keeps of its columns
struct KeepAll { };
template <bool COMPLEX, bool DROP> __device__ __forceinline__ auto keep_of(const Drop& drop, long column)
{
    if constexpr (DROP) return Keep<COMPLEX>(drop, column);
    else return KeepAll();
}

}  // namespace tfno
