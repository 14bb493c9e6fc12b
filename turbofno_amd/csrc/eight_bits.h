// Fields in 8 bits (e4m3) with a scale for each position and block of 128 channels, as strips of a field form them.
#pragma once
#include "strips.h"

namespace tfno {

constexpr long kFewStrips = 512;                        // strips of 256 columns that fill the GPU

// sums over the channels of a block of threads: over the lanes of a wave that share a column, then over the waves. `shared` holds COUNT x 8 x LANES values,
// which nothing else uses between two barriers
template <int LANES, int COUNT, typename F> __device__ __forceinline__ void over_waves(float4_v (&v)[COUNT], float4_v* shared, F join)
{
    constexpr int WAVES = kThreads / 64;
    const int lane = threadIdx.x % LANES, wave = threadIdx.x / 64;
#pragma unroll
    for (int d = LANES; d < 64; d *= 2)
#pragma unroll
        for (int c = 0; c < COUNT; ++c) {
            float4_v o;
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = __shfl_xor(v[c][i], d, 64);
            v[c] = join(v[c], o);
        }
    if (threadIdx.x % 64 < LANES)
#pragma unroll
        for (int c = 0; c < COUNT; ++c) shared[(c * WAVES + wave) * LANES + lane] = v[c];
    __syncthreads();
#pragma unroll
    for (int c = 0; c < COUNT; ++c) v[c] = shared[c * WAVES * LANES + lane];
    auto add = [&](int w) {
#pragma unroll
        for (int c = 0; c < COUNT; ++c) v[c] = join(v[c], shared[(c * WAVES + w) * LANES + lane]);
    };
    if constexpr (COUNT <= 2) {
#pragma unroll
        for (int w = 1; w < WAVES; ++w) add(w);
    } else                                              // few registers at a time
#pragma unroll 1
        for (int w = 1; w < WAVES; ++w) add(w);
}
// largest magnitudes per position, of COUNT blocks of channels
template <bool COMPLEX, int LANES, int COUNT> __device__ __forceinline__ void block_maxima(float4_v (&most)[COUNT], float4_v* shared)
{
#pragma unroll
    for (int c = 0; c < COUNT; ++c) most[c] = largest_per_position<COMPLEX>(most[c]);
    over_waves<LANES, COUNT>(most, shared, larger4);
}
// The scales of a block at the lane's positions; what its values are multiplied with. No normal number for a scale: a scale of 1 and zeros. A largest
// magnitude that is infinite or NaN: both NaN
template <bool COMPLEX, bool FULL> __device__ __forceinline__ float4_v write_scales(float* scale, long column, int there, bool writes, float4_v most)
{
    constexpr int PARTS = COMPLEX ? 2 : 1;
    float4_v factor, s;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float m = most[i] == __builtin_inff() ? __builtin_nanf("") : most[i];
        s[i] = m / 448.f;
        const bool none = s[i] < 0x1p-126f;
        factor[i] = none ? 0.f : 448.f / m;
        if (none) s[i] = 1.f;
    }
    if (writes)
#pragma unroll
        for (int i = 0; i < 4; i += PARTS)
            if (FULL || i < there) scale[(column + i) / PARTS] = s[i];
    return factor;
}
// four values in e4m3; the product may be a few roundings above 448: what is at most 464 becomes 448
__device__ __forceinline__ unsigned eight_bits(float4_v v, float4_v factor)
{
    v = v * factor;
    int bytes = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], bytes, true);
}

}  // namespace tfno
