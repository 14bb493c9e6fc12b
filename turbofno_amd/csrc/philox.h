// Dropout's random numbers: Philox 4x32 with ten rounds (J. K. Salmon, M. A. Moraes, R. O. Dror, D. E. Shaw: Parallel random numbers: as easy as 1, 2, 3;
// SC 2011), a function of a key and a counter, so that no mask is stored and the gradient forms the same one again:
//
//   key = seed (two words),  counter = (low word of q, channel + 2^16 high word of q, offset (two words)),  q = position / 4
//   element kept  <=>  word position % 4 of the result >= threshold, the whole number nearest to drop 2^32, at most 2^32 - 1
//
// q has at most 34 bits and a channel 16. A complex element is kept or dropped as a whole. The numbers depend on nothing else: not on strides, types or the
// kernel that asks. The key and the offset lie in memory of the GPU, so that a captured graph draws other numbers when its user has changed them.
#pragma once
#include "columns.h"

namespace tfno {

// four words. A round is two products of 32 by 32 bits, which the vector unit forms whole (v_mad_u64_u32)
__device__ __forceinline__ uint4_v philox(uint4_v c, unsigned k0, unsigned k1)
{
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const unsigned long a = 0xD2511F53ul * c[0], b = 0xCD9E8D57ul * c[2];
        c = (uint4_v){ (unsigned)(b >> 32) ^ c[1] ^ k0, (unsigned)b, (unsigned)(a >> 32) ^ c[3] ^ k1, (unsigned)a };
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return c;
}

// What a lane keeps of its four real columns (one quad of positions, or half of one): a bit per column that it has an element of
template <bool COMPLEX> struct Keep {
    const unsigned k0, k1, o0, o1, threshold;
    const unsigned q, high;                             // of the lane's quad
    const bool odd;                                     // complex: the lane has the last two positions of its quad
    __device__ __forceinline__ Keep(const Drop& d, long column) : k0(d.rng[0]), k1(d.rng[1]), o0(d.rng[2]), o1(d.rng[3]), threshold(d.threshold),
        q((unsigned)(column / (COMPLEX ? 8 : 4))), high((unsigned)(column / (COMPLEX ? 8 : 4) >> 32) << 16), odd(COMPLEX && (column & 4)) { }
    __device__ __forceinline__ unsigned quad(int channel) const
    {
        const uint4_v w = philox((uint4_v){ q, (unsigned)channel + high, o0, o1 }, k0, k1);
        return (w[0] >= threshold) | (w[1] >= threshold) << 1 | (w[2] >= threshold) << 2 | (w[3] >= threshold) << 3;
    }
    // of two channels. Complex: lanes 2 i and 2 i + 1 share a quad, so each forms one channel's and they exchange them; all lanes have to be here
    __device__ __forceinline__ void pair(int first, int second, unsigned& a, unsigned& b) const
    {
        if constexpr (!COMPLEX) {
            a = quad(first);
            b = quad(second);
        } else {
            const unsigned mine = quad(odd ? second : first), other = (unsigned)__builtin_amdgcn_update_dpp(0, (int)mine, 0xB1, 0xf, 0xf, true);
            a = odd ? other >> 2 : mine & 3u;
            b = odd ? mine >> 2 : other & 3u;
        }
    }
    // what is dropped becomes 0, whatever it was
    static __device__ __forceinline__ float4_v apply(float4_v v, unsigned bits, float lift)
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = bits >> (COMPLEX ? i / 2 : i) & 1u ? v[i] * lift : 0.f;
        return v;
    }
};

}  // namespace tfno
