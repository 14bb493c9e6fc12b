// Strips of the norms: a block takes 64 ... 256 real columns of a field and all of their channels. A lane has four consecutive columns of each of its
// channels; LANES lanes side by side make the strip, the groups of lanes that a block has take turns over the channels.
#pragma once
#include "columns.h"

namespace tfno {

constexpr int kThreads = 512;
constexpr long kFar = 1L << 28;                         // real values between channels

// Whether strips that lie side by side go to one XCD: where rows do not start at whole cache lines of 128 bytes, so that neighbours share lines, which the XCD's L2 cache then
// fetches once. bf16, layer norm of 300 channels at 65551 positions 57 us, 73 with strips dealt out to the XCDs in turns; its gradient, 128 channels at 200003 76 and 97 us; where
// rows start at whole lines the turns are ahead: complex64, 64 channels at 2^20 408 us and 422
inline bool run_together(long columns, int type, long strips) { return strips >= 64 && columns * (type == kIn16 ? 2 : 4) % 128; }
// columns a lane adds up belong to one position each (real) or two and two (complex)
template <bool COMPLEX> __device__ __forceinline__ float4_v per_position(float4_v v)
{
    if constexpr (!COMPLEX) return v;
    else { const float a = v[0] + v[1], b = v[2] + v[3]; return (float4_v){ a, a, b, b }; }
}
template <bool COMPLEX> __device__ __forceinline__ float4_v largest_per_position(float4_v v)
{
    if constexpr (!COMPLEX) return v;
    else { const float a = __builtin_elementwise_maximum(v[0], v[1]), b = __builtin_elementwise_maximum(v[2], v[3]); return (float4_v){ a, a, b, b }; }
}
__device__ __forceinline__ float4_v larger4(float4_v a, float4_v b)      // a NaN stays
{
    return __builtin_elementwise_maximum(a, b);
}
__device__ __forceinline__ float4_v magnitude(float4_v a)
{
    return (float4_v){ __builtin_fabsf(a[0]), __builtin_fabsf(a[1]), __builtin_fabsf(a[2]), __builtin_fabsf(a[3]) };
}

// Strip of a block: 4 LANES columns, and GROUPS channels of it side by side. Channel r GROUPS + group belongs to group `group`; a wave holds 64 / LANES
// groups, so a channel is a part common to the wave and the lane's.
template <int LANES> struct Strip {
    static constexpr int GROUPS = kThreads / LANES, OF_WAVE = 64 / LANES, COLUMNS = 4 * LANES;
    const int K, lane, sub, first;                      // first: the wave's first group
    __device__ __forceinline__ Strip(int channels) : K(channels), lane(threadIdx.x % LANES), sub(threadIdx.x % 64 / LANES),
        first(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * OF_WAVE) { }
    __device__ __forceinline__ int group() const { return first + sub; }
    // the r-th channel of a lane, or one that exists; its gain
    __device__ __forceinline__ int channel(int r) const { return has(r) ? r * GROUPS + first + sub : common(r); }
    __device__ __forceinline__ int common(int r) const { const int k = r * GROUPS + first; return k < K ? k : K - 1; }
    __device__ __forceinline__ bool has(int r) const { return r * GROUPS + first + sub < K; }
    // four columns of that channel. FULL: all columns of the strip exist, otherwise `there` of them
    template <int IN, bool FULL> __device__ __forceinline__ RawOf<IN> read(const void* base, long ld, long column0, int there, int r) const
    {
        typedef typename Columns<IN>::Value Value;
        const unsigned lane_row = has(r) ? sub : 0;
        if constexpr (FULL) return near_load4<IN>(scalar(base, (common(r) * ld + column0) * (long)sizeof(Value)), fresh((lane_row * (unsigned)ld + 4 * lane) * (unsigned)sizeof(Value)));
        else return load4_ragged<IN>(static_cast<const Value*>(base) + (common(r) + lane_row) * ld + column0, 4 * lane, there);
    }
    template <int IN, bool FULL> __device__ __forceinline__ void write(void* base, long ld, long column0, int there, int r, RawOf<IN> v) const
    {
        typedef typename Columns<IN>::Value Value;
        if constexpr (FULL) near_store4<IN>(scalar(base, (common(r) * ld + column0) * (long)sizeof(Value)), fresh((sub * (unsigned)ld + 4 * lane) * (unsigned)sizeof(Value)), v);
        else store4_ragged<IN>(static_cast<Value*>(base) + (common(r) + sub) * ld + column0, 4 * lane, there, v);
    }
    // over the groups of a block; `shared` holds GROUPS x LANES values. TIGHT: in a loop, four at a time, where the registers are taken
    template <bool TIGHT, typename F> __device__ __forceinline__ float4_v over_channels(float4_v v, float4_v* shared, F join) const
    {
        shared[threadIdx.x] = v;
        __syncthreads();
        v = shared[lane];
        if constexpr (TIGHT) {
#pragma unroll
            for (int g = 1; g < 4; ++g) v = join(v, shared[g * LANES + lane]);
#pragma unroll 1
            for (int g = 4; g < GROUPS; g += 4) {
                const float4_v a = shared[g * LANES + lane], b = shared[(g + 1) * LANES + lane], c = shared[(g + 2) * LANES + lane], d = shared[(g + 3) * LANES + lane];
                v = join(join(join(join(v, a), b), c), d);
            }
        } else
#pragma unroll 7
            for (int g = 1; g < GROUPS; ++g) v = join(v, shared[g * LANES + lane]);
        return v;
    }
};
__device__ __forceinline__ float4_v four(const float (&v)[4]) { return (float4_v){ v[0], v[1], v[2], v[3] }; }
__device__ __forceinline__ float4_v sum4(float4_v a, float4_v b) { return a + b; }
template <int PARTS> __device__ __forceinline__ float4_v per_column(const float* values, long column, int there)    // of the lane's columns; 0 beyond
{
    float4_v v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < there ? values[(column + i) / PARTS] : 0.f;
    return v;
}

// 1 / sqrt(v). The instruction takes numbers below 2^-126 for zeros
__device__ __forceinline__ float reciprocal_root(float v)
{
    const bool small = v < 0x1p-100f;
    const float r = __builtin_amdgcn_rsqf(small ? v * 0x1p48f : v);
    return small ? r * 0x1p24f : r;
}

}  // namespace tfno
