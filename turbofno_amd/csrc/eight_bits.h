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
// Quotients by a scale s. A product with its reciprocal is off by up to two steps of fp32, and bf16 fields often hold values whose quotient lies exactly between two numbers of e4m3
// (three quarters of the block's largest, say), which that would tip: 5312 of 17160000 normal ones. So the reciprocal has two parts, r and d = r e with e = 1 - s r, which fp32 holds
// exactly: 1 / s = r / (1 - e) = r + d + ..., without terms of 2^-44, and v / s = v r + v d is rounded once. e is not negative, so that a zero keeps its sign. Against a product alone (inputs in
// the caches): bf16, 1024 channels at 65536 positions 31.7 us and 31.3; layer norm, 512 at 65536 with residual 60.9 and 60.4.
struct Divisor {
    float4_v r, d;
    __device__ __forceinline__ float4_v divide(float4_v v) const
    {
        float4_v q;
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] = __builtin_fmaf(v[i], r[i], v[i] * d[i]);
        return q;
    }
};
// The scales of a block at the lane's positions; what its values are divided by. No normal number for a scale: a scale of 1 and zeros. A largest
// magnitude that is infinite or NaN: both NaN
template <bool COMPLEX, bool FULL> __device__ __forceinline__ Divisor write_scales(float* scale, long column, int there, bool writes, float4_v most)
{
    constexpr int PARTS = COMPLEX ? 2 : 1;
    Divisor by;
    float4_v s;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float m = most[i] == __builtin_inff() ? __builtin_nanf("") : most[i];
        s[i] = m / 448.f;
        const bool none = s[i] < 0x1p-126f;
        float r = __builtin_amdgcn_rcpf(s[i]);
        if (__builtin_fmaf(-s[i], r, 1.f) < 0.f) r = __builtin_bit_cast(float, __builtin_bit_cast(unsigned, r) - 1);
        by.r[i] = none ? 0.f : r;
        by.d[i] = none ? 0.f : r * __builtin_fmaf(-s[i], r, 1.f);
        if (none) s[i] = 1.f;
    }
    if (writes)
#pragma unroll
        for (int i = 0; i < 4; i += PARTS)
            if (FULL || i < there) scale[(column + i) / PARTS] = s[i];
    return by;
}
// four quotients in e4m3; the largest may be a rounding above 448: what is at most 464 becomes 448
__device__ __forceinline__ unsigned eight_bits(float4_v v, const Divisor& by)
{
    v = by.divide(v);
    int bytes = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], bytes, true);
}

}  // namespace tfno
