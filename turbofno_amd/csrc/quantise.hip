// A field in 8 bits with a scale for each position and block of 128 channels (turbofno_quantise_8bit):
//
//   scale[b][p] = max over the channels k of block b of |x[k][p]| / 448 (real and imaginary parts),  q[k][p] = e4m3(x[k][p] / scale[k / 128][p])
//
// A block of threads takes a strip of columns and one block of channels, which it holds in registers between the maximum and its use: every byte moves once.
// bf16, 1024 channels at 65536 positions 38.5 us, 5.3 TB/s: the stream. float32, 200 at 10007 5.5 us: one round of 314 blocks behind the launch.
#include "eight_bits.h"

namespace tfno {

namespace {

template <int IN, bool COMPLEX, int LANES, bool FULL>
__device__ __forceinline__ void quantise_strip(const QuantiseParams& q, int block, float4_v* shared, long column0, int there)
{
    typedef Strip<LANES> S;
    constexpr int HELD = kScaleBlock / S::GROUPS;
    const int first = block * kScaleBlock;
    const S strip(q.K - first < kScaleBlock ? q.K - first : kScaleBlock);
    const auto* x = static_cast<const typename Columns<IN>::Value*>(q.x) + first * q.ldx;
    unsigned char* to = static_cast<unsigned char*>(q.q) + first * q.ldq;
    RawOf<IN> raw[HELD];
#pragma unroll
    for (int r = 0; r < HELD; ++r) raw[r] = strip.template read<IN, FULL>(x, q.ldx, column0, there, r);
    float4_v most[1] = {};
#pragma unroll
    for (int r = 0; r < HELD; ++r)
        if (strip.has(r)) most[0] = larger4(most[0], magnitude(to_float<IN>(raw[r])));
    block_maxima<COMPLEX, LANES>(most, shared);
    const Divisor by = write_scales<COMPLEX, FULL>(q.scale + block * q.positions, column0 + 4 * strip.lane, there - 4 * strip.lane, strip.group() == 0, most[0]);
#pragma unroll
    for (int r = 0; r < HELD; ++r)
        if (strip.has(r)) strip.template write<kIn8, FULL>(to, q.ldq, column0, there, r, eight_bits(to_float<IN>(raw[r]), by));
}
template <int IN, bool COMPLEX, int LANES> __global__ __launch_bounds__(kThreads, 4) void quantise_kernel(const QuantiseParams q, long strips, long run)
{
    __shared__ float4_v shared[kThreads / 64 * LANES];
    const long id = block_index(), block = id / strips, place = id - block * strips, column0 = (run ? side_by_side(place, run) : place) * (4 * LANES);
    if (block * kScaleBlock >= q.K || column0 >= q.columns) return;
    if (column0 + 4 * LANES <= q.columns) quantise_strip<IN, COMPLEX, LANES, true>(q, (int)block, shared, column0, 4 * LANES);
    else quantise_strip<IN, COMPLEX, LANES, false>(q, (int)block, shared, column0, (int)(q.columns - column0));
}
template <int IN, bool COMPLEX, int LANES> hipError_t launch_as(const QuantiseParams& q, hipStream_t stream)
{
    const long all = (q.columns + 4 * LANES - 1) / (4 * LANES), blocks = (q.K + kScaleBlock - 1) / kScaleBlock;
    // bf16, 256 channels at 50021 positions 9.8 us side by side, 15.3 in turns; float32, 200 at 10007 5.4 and 4.7, 1000 at 10007 11.0 and 14.1
    const long run = all * blocks >= 512 && run_together(q.columns, IN, all) ? (all + 7) / 8 : 0, strips = run ? 8 * run : all;
    hipLaunchKernelGGL((quantise_kernel<IN, COMPLEX, LANES>), grid_of(strips * blocks), dim3(kThreads), 0, stream, q, strips, run);
    return hipGetLastError();
}
template <int IN, bool COMPLEX> hipError_t launch(const QuantiseParams& q, hipStream_t stream)
{
    // narrow strips where wide ones would leave most of the GPU idle; a lane's part of an address, up to three channels, in 32 bits
    const bool far = q.ldx >= kFar || q.ldq >= kFar;
    const long wide = (q.columns + 255) / 256 * ((q.K + kScaleBlock - 1) / kScaleBlock);
    if (wide < kFewStrips && !far) return launch_as<IN, COMPLEX, 16>(q, stream);
    return launch_as<IN, COMPLEX, 64>(q, stream);
}

}  // namespace

hipError_t launch_quantise_8bit(const QuantiseParams& q, int type, hipStream_t stream)
{
    if (q.columns == 0) return hipSuccess;
    switch (type) {
    case kC64: return launch<kIn32, true>(q, stream);
    case kF32: return launch<kIn32, false>(q, stream);
    default: return launch<kIn16, false>(q, stream);
    }
}

}  // namespace tfno
