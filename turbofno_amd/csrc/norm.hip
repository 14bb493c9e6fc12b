// Root-mean-square norm over channels with the residual's addition (turbofno_rms_norm), with its result in 8 bits (turbofno_rms_norm_8bit), and its
// gradient (turbofno_rms_norm_backward). Per position p, sums over the K channels:
//
//   s = x + residual,  rstd = 1 / sqrt(mean_k |s_k|^2 + eps),  y_k = gain_k rstd s_k
//   8 bit     scale = max_k |y_k| / 448 (real and imaginary parts), q_k = e4m3(y_k / scale)
//   gradient  d = mean_k gain_k Re(conj(s_k) gy_k),  gx_k = rstd gain_k gy_k - rstd^3 d s_k + gs_k,  ggain_k = sum_p rstd Re(conj(s_k) gy_k)
//
// Channels are the outermost axis, so a block takes a strip of positions and all of their channels, keeps them in registers between the sum and
// its use, and moves every byte once: nothing but memory traffic bounds it. A lane has four consecutive real columns of each of its channels;
// 16 or 64 lanes side by side make a strip of 64 or 256 columns (16: four channels per wave and access), the waves of a block take turns over the
// channels. Sums over channels are formed per lane, then over the lanes and waves that share a column through LDS, in fp32. Where the channels do
// not fit into registers the strip is read a second time. Measured, with residual: complex64, 64 channels, 2^20 positions 405 us (5.3 TB/s), its gradient
// 426 us (5.0 TB/s); bf16 to 8 bits, 256 channels, 262144 positions 97 us (4.8 TB/s); a large copy reaches 5.15 TB/s.
#include "strips.h"
#include <algorithm>

namespace tfno {

namespace {

// Up to here, narrow strips: 512 blocks run at a time, each loads all of its channels, then stores them, and fewer wide strips than that do both once, one after the
// other. bf16, 128 channels, residual: 10000 columns 7.2 us (wide strips 12), 60000 15.4 (20.7), 120000 27.1 (43.5); above, wide strips read longer
// pieces of a row: 500000 columns 117 us (narrow 122), 8 bits at 262144 50 us (narrow 62).
constexpr long kFewColumns = 1L << 17;                  // real columns

// HELD: channels per lane kept in registers; 0: read again. At most 16: 32 lanes side by side for 256 channels, 16 for 512 (bf16 to 8 bits, 256 channels at 262144
// positions: 97 us, with 64 lanes and so 32 channels in a lane, which spill, 467; float32 210 and 219)
template <int IN, bool COMPLEX, bool EIGHT, int LANES, int HELD, bool FULL>
__device__ __forceinline__ void norm_strip(const NormParams& q, float4_v* shared, const float* gains, long column0, int there)
{
    constexpr int PARTS = COMPLEX ? 2 : 1;
    const Strip<LANES> strip(q.K);
    auto gain = [&](int r) { return HELD ? gains[r * strip.GROUPS + strip.group()] : q.gain[strip.channel(r)]; };
    const int lane_there = there - 4 * strip.lane;
    const long column = column0 + 4 * strip.lane;
    auto value = [&](int r) {
        float4_v v = to_float<IN>(strip.template read<IN, FULL>(q.x, q.ldx, column0, there, r));
        if (q.residual) v += to_float<IN>(strip.template read<IN, FULL>(q.residual, q.ldr, column0, there, r));
        return v;
    };
    const int rounds = (q.K + strip.GROUPS - 1) / strip.GROUPS;
    float held[HELD ? HELD : 1][4];                     // one by one: quadruples would need four registers in a row each
    float4_v sum = {}, most = {};
    auto add = [&](int r, float4_v v) {
        sum += v * v;
        if constexpr (EIGHT) most = larger4(most, magnitude(v * gain(r)));
    };
    if constexpr (HELD > 0) {
        // all loads first: channels beyond the last read another one
        RawOf<IN> x[HELD], residual[HELD];
#pragma unroll
        for (int r = 0; r < HELD; ++r) x[r] = strip.template read<IN, FULL>(q.x, q.ldx, column0, there, r);
        if (q.residual)
#pragma unroll
            for (int r = 0; r < HELD; ++r) residual[r] = strip.template read<IN, FULL>(q.residual, q.ldr, column0, there, r);
        __syncthreads();                                // gains
#pragma unroll
        for (int r = 0; r < HELD; ++r) {
            float4_v v = to_float<IN>(x[r]);
            if (q.residual) v += to_float<IN>(residual[r]);
            if (strip.has(r)) sum += v * v;
#pragma unroll
            for (int i = 0; i < 4; ++i) held[r][i] = v[i];
        }
        if constexpr (EIGHT)
#pragma unroll
            for (int r = 0; r < HELD; ++r)
                if (strip.has(r)) most = larger4(most, magnitude(four(held[r]) * gain(r)));
    } else
        for (int r = 0; r < rounds; ++r)
            if (strip.has(r)) add(r, value(r));
    sum = strip.template over_channels<true>(per_position<COMPLEX>(sum), shared, sum4);
    if constexpr (EIGHT) most = strip.template over_channels<true>(largest_per_position<COMPLEX>(most), shared + kThreads, larger4);
    float4_v rstd, factor, lift = { 1.f, 1.f, 1.f, 1.f };
#pragma unroll
    for (int i = 0; i < 4; ++i) factor[i] = rstd[i] = reciprocal_root(sum[i] / (float)q.K + q.eps);
    if constexpr (EIGHT)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            // y / scale = s gain (448 / max |s gain|), which is at most 448 and a few roundings: e4m3 takes up to 464 to 448. The product s gain comes first: 448 / max
            // alone times a gain may be infinite. Where max is small, both are lifted so that 448 / max is finite
            if (most[i] < 0x1p-96f) lift[i] = 0x1p64f;
            factor[i] = 448.f / (most[i] * lift[i]);
            rstd[i] /= factor[i];
            if (most[i] < 0x1p-96f) rstd[i] *= 0x1p-64f;
            // nothing but zeros, or no normal number for a scale: a scale of 1, which leaves zeros of what is below 2^-117
            if (most[i] == 0.f || rstd[i] < 0x1p-126f) {
                rstd[i] = 1.f;
                factor[i] = 0.f;
            }
        }
    if (strip.group() == 0 && q.rstd)
#pragma unroll
        for (int i = 0; i < 4; i += PARTS)
            if (FULL || i < lane_there) q.rstd[(column + i) / PARTS] = rstd[i];
    auto store_sum = [&](int r, float4_v v) { strip.template write<IN, FULL>(q.s, q.lds, column0, there, r, from_float<IN>(v)); };
    auto finish = [&](int r, float4_v v) {
        if constexpr (EIGHT) {
            v = v * gain(r) * lift * factor;
            int bytes = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
            bytes = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], bytes, true);
            strip.template write<kIn8, FULL>(q.y, q.ldy, column0, there, r, (unsigned)bytes);
        } else strip.template write<IN, FULL>(q.y, q.ldy, column0, there, r, from_float<IN>(v * (factor * gain(r))));
    };
    auto both = [&](int r, float4_v v) {                // v is there before either result is written: they may take its operands' place
        if (q.s) store_sum(r, v);
        finish(r, v);
    };
    if constexpr (HELD > 0) {
#pragma unroll
        for (int r = 0; r < HELD; ++r)
            if (strip.has(r)) both(r, four(held[r]));
    } else
        for (int r = 0; r < rounds; ++r)
            if (strip.has(r)) both(r, value(r));
}
// 16-bit values: 128 registers and so 16 waves on a CU, which load and store in turn
template <int IN, bool COMPLEX, bool EIGHT, int LANES, int HELD> __global__ __launch_bounds__(kThreads, IN == kIn16 ? 4 : 2) void norm_kernel(const NormParams q)
{
    typedef Strip<LANES> S;
    const long column0 = block_index() * S::COLUMNS;
    if (column0 >= q.columns) return;
    __shared__ float4_v shared[(EIGHT ? 2 : 1) * kThreads];
    __shared__ float gains[HELD ? HELD * S::GROUPS : 1];
    if constexpr (HELD > 0)
        for (int k = threadIdx.x; k < HELD * S::GROUPS; k += kThreads) gains[k] = q.gain[k < q.K ? k : q.K - 1];
    if (column0 + S::COLUMNS <= q.columns) norm_strip<IN, COMPLEX, EIGHT, LANES, HELD, true>(q, shared, gains, column0, S::COLUMNS);
    else norm_strip<IN, COMPLEX, EIGHT, LANES, HELD, false>(q, shared, gains, column0, (int)(q.columns - column0));
}

template <int IN, bool COMPLEX, int LANES, int HELD, bool FULL>
__device__ __forceinline__ void norm_grad_strip(const NormGradParams& q, float4_v* shared, const float* gains, long column0, int there, float (&ggain)[HELD])
{
    const Strip<LANES> strip(q.K);
    auto gain = [&](int r) { return gains[r * strip.GROUPS + strip.group()]; };
    RawOf<IN> gy[HELD], s[HELD];
#pragma unroll
    for (int r = 0; r < HELD; ++r) {
        gy[r] = strip.template read<IN, FULL>(q.gy, q.ldgy, column0, there, r);
        s[r] = strip.template read<IN, FULL>(q.s, q.lds, column0, there, r);
    }
    const int lane_there = there - 4 * strip.lane;
    const float4_v rstd = per_column<COMPLEX ? 2 : 1>(q.rstd, column0 + 4 * strip.lane, FULL ? 4 : lane_there);
    float4_v along = {};
#pragma unroll
    for (int r = 0; r < HELD; ++r)
        if (strip.has(r)) {
            const float4_v d = to_float<IN>(gy[r]) * to_float<IN>(s[r]);
            along += d * gain(r);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (FULL || i < lane_there) ggain[r] = __builtin_fmaf(d[i], rstd[i], ggain[r]);
        }
    along = strip.template over_channels<false>(per_position<COMPLEX>(along), shared, sum4);
    const float4_v shrink = along * rstd * rstd * (1.f / (float)q.K);        // times s rstd: the cube of rstd may be infinite
#pragma unroll
    for (int r = 0; r < HELD; ++r)
        if (strip.has(r)) {
            if constexpr (IN == kIn16) asm volatile("" : "+v"(gy[r]), "+v"(s[r]));       // widened again, not held in twice the registers
            float4_v v = to_float<IN>(gy[r]) * (rstd * gain(r)) - to_float<IN>(s[r]) * rstd * shrink;
            if (q.gs) v += to_float<IN>(strip.template read<IN, FULL>(q.gs, q.ldgs, column0, there, r));
            strip.template write<IN, FULL>(q.gx, q.ldgx, column0, there, r, from_float<IN>(v));
        }
}
// Persistent over strips, so that the sums of ggain stay in registers
template <int IN, bool COMPLEX, int LANES, int HELD> __global__ __launch_bounds__(kThreads, HELD < 32 ? 4 : 2) void norm_grad_kernel(const NormGradParams q, long strips)
{
    __shared__ float4_v shared[2][kThreads];
    __shared__ float gains[HELD * Strip<LANES>::GROUPS];
    for (int k = threadIdx.x; k < HELD * Strip<LANES>::GROUPS; k += kThreads) gains[k] = q.gain[k < q.K ? k : q.K - 1];
    __syncthreads();
    float ggain[HELD] = {};
    // two buffers: a strip's sums are read while the next strip's are written by the waves that are ahead, never two strips ahead
    int turn = 0;
    for (long b = blockIdx.x; b < strips; b += gridDim.x, turn ^= 1) {
        const long column0 = b * Strip<LANES>::COLUMNS;
        if (column0 + Strip<LANES>::COLUMNS <= q.columns) norm_grad_strip<IN, COMPLEX, LANES, HELD, true>(q, shared[turn], gains, column0, Strip<LANES>::COLUMNS, ggain);
        else norm_grad_strip<IN, COMPLEX, LANES, HELD, false>(q, shared[turn], gains, column0, (int)(q.columns - column0), ggain);
    }
    const Strip<LANES> strip(q.K);
#pragma unroll
    for (int r = 0; r < HELD; ++r) {
        float v = ggain[r];
#pragma unroll
        for (int d = 1; d < LANES; d *= 2) v += __shfl_xor(v, d, LANES);
        if (strip.lane == 0 && strip.has(r)) q.sums[(long)blockIdx.x * q.K + strip.channel(r)] = v;
    }
}

// More channels than registers hold: one strip per block, read twice
template <int IN, bool COMPLEX, int LANES, bool FULL>
__device__ __forceinline__ void norm_grad_long_strip(const NormGradParams& q, float4_v* shared, long column0, int there)
{
    const Strip<LANES> strip(q.K);
    const int lane_there = there - 4 * strip.lane, rounds = (q.K + strip.GROUPS - 1) / strip.GROUPS;
    const float4_v rstd = per_column<COMPLEX ? 2 : 1>(q.rstd, column0 + 4 * strip.lane, FULL ? 4 : lane_there);
    auto value = [&](const void* p, long ld, int r) { return to_float<IN>(strip.template read<IN, FULL>(p, ld, column0, there, r)); };
    float4_v along = {};
    for (int r = 0; r < rounds; ++r)
        if (strip.has(r)) along += value(q.gy, q.ldgy, r) * value(q.s, q.lds, r) * q.gain[strip.channel(r)];
    along = strip.template over_channels<false>(per_position<COMPLEX>(along), shared, sum4);
    const float4_v shrink = along * rstd * rstd * (1.f / (float)q.K);
    for (int r = 0; r < rounds; ++r) {
        if (!strip.has(r)) continue;                    // the lanes of a group together
        const float4_v gy = value(q.gy, q.ldgy, r), s = value(q.s, q.lds, r);
        float4_v v = gy * (rstd * q.gain[strip.channel(r)]) - s * rstd * shrink;
        if (q.gs) v += value(q.gs, q.ldgs, r);
        strip.template write<IN, FULL>(q.gx, q.ldgx, column0, there, r, from_float<IN>(v));
        const float4_v d = gy * s;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (FULL || i < lane_there) sum = __builtin_fmaf(d[i], rstd[i], sum);
#pragma unroll
        for (int e = 1; e < LANES; e *= 2) sum += __shfl_xor(sum, e, LANES);
        if (strip.lane == 0) q.sums[block_index() * q.K + strip.channel(r)] = sum;
    }
}
template <int IN, bool COMPLEX, int LANES> __global__ __launch_bounds__(kThreads) void norm_grad_long_kernel(const NormGradParams q)
{
    __shared__ float4_v shared[kThreads];
    constexpr int COLUMNS = Strip<LANES>::COLUMNS;
    const long column0 = block_index() * COLUMNS;
    if (column0 >= q.columns) return;
    if (column0 + COLUMNS <= q.columns) norm_grad_long_strip<IN, COMPLEX, LANES, true>(q, shared, column0, COLUMNS);
    else norm_grad_long_strip<IN, COMPLEX, LANES, false>(q, shared, column0, (int)(q.columns - column0));
}

// ggain: the blocks' sums, one channel per block, always in the same order
__global__ __launch_bounds__(256) void add_gain_kernel(const float* __restrict__ sums, long blocks, int K, float* __restrict__ ggain)
{
    __shared__ float part[4];
    float v = 0.f;
    for (long b = threadIdx.x; b < blocks; b += 256) v += sums[b * K + blockIdx.x];
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d, 64);
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = v;
    __syncthreads();
    if (threadIdx.x == 0) ggain[blockIdx.x] = (part[0] + part[1]) + (part[2] + part[3]);
}

template <int IN, bool COMPLEX, bool EIGHT, int LANES, int HELD> hipError_t launch_norm_as(const NormParams& q, hipStream_t stream)
{
    hipLaunchKernelGGL((norm_kernel<IN, COMPLEX, EIGHT, LANES, HELD>), grid_of((q.columns + 4 * LANES - 1) / (4 * LANES)), dim3(kThreads), 0, stream, q);
    return hipGetLastError();
}
template <int IN, bool COMPLEX, bool EIGHT> hipError_t launch_norm(const NormParams& q, hipStream_t stream)
{
    // a lane's part of an address, up to three channels, in 32 bits; with 64 lanes side by side it has no channel in it
    const bool far = std::max(std::max(q.ldx, q.ldr), std::max(q.lds, q.ldy)) >= kFar;
    // strips of 64 columns instead of 256 where those would leave most of the GPU idle
    if (q.columns < kFewColumns && !far) {
        if (q.K <= 64) return launch_norm_as<IN, COMPLEX, EIGHT, 16, 2>(q, stream);
        if (q.K <= 128) return launch_norm_as<IN, COMPLEX, EIGHT, 16, 4>(q, stream);
        if (q.K <= 256) return launch_norm_as<IN, COMPLEX, EIGHT, 16, 8>(q, stream);
    }
    if (q.K <= 32) return launch_norm_as<IN, COMPLEX, EIGHT, 64, 4>(q, stream);
    if (q.K <= 64) return launch_norm_as<IN, COMPLEX, EIGHT, 64, 8>(q, stream);
    if (q.K <= 128) return launch_norm_as<IN, COMPLEX, EIGHT, 64, 16>(q, stream);
    if (far) return launch_norm_as<IN, COMPLEX, EIGHT, 64, 0>(q, stream);
    if (q.K <= 256) return launch_norm_as<IN, COMPLEX, EIGHT, 32, 16>(q, stream);
    if (q.K <= 512) return launch_norm_as<IN, COMPLEX, EIGHT, 16, 16>(q, stream);
    return launch_norm_as<IN, COMPLEX, EIGHT, 16, 0>(q, stream);
}

constexpr int kGradHeldChannels = 256;                  // 8 per lane, 32 side by side
// persistent blocks, two per CU (bf16, 128 channels at 262144 positions: 65 us, twice as many 69; complex64, 64 channels at 2^20: 427 and 423)
constexpr long kGradBlocks = 512;

// lanes side by side: by the channels that registers hold, fewer where wide strips would leave most of the GPU idle (bf16, 128 channels at 262144 positions: 65 us
// with 32, 70 with 16; float32 108 and 112)
int grad_lanes(int K, long columns) { return columns < kFewColumns ? 16 : K <= 64 ? 64 : K <= 128 ? 32 : 16; }
long grad_strips(int K, long columns) { return (columns + 4 * grad_lanes(K, columns) - 1) / (4 * grad_lanes(K, columns)); }
long grad_blocks(int K, long columns)
{
    const long strips = grad_strips(K, columns);
    return K > kGradHeldChannels || strips < kGradBlocks ? strips : kGradBlocks;
}

template <int IN, bool COMPLEX> hipError_t launch_grad(const NormGradParams& q, hipStream_t stream)
{
    const long strips = grad_strips(q.K, q.columns), wide = (q.columns + 255) / 256;
    const bool far = std::max(std::max(q.ldgy, q.lds), std::max(q.ldgs, q.ldgx)) >= kFar;
    const long blocks = far && q.K > kGradHeldChannels ? wide : grad_blocks(q.K, q.columns);
    const dim3 grid = grid_of(blocks);                  // one row of them where they are persistent
#define TFNO_NORM_GRAD(LANES, HELD, STRIPS) hipLaunchKernelGGL((norm_grad_kernel<IN, COMPLEX, LANES, HELD>), grid, dim3(kThreads), 0, stream, q, STRIPS)
    if (blocks) {
        if (q.K > kGradHeldChannels) {
            if (far) hipLaunchKernelGGL((norm_grad_long_kernel<IN, COMPLEX, 64>), grid, dim3(kThreads), 0, stream, q);
            else hipLaunchKernelGGL((norm_grad_long_kernel<IN, COMPLEX, 16>), grid, dim3(kThreads), 0, stream, q);
        } else if (far) {
            if (q.K <= 64) TFNO_NORM_GRAD(64, 8, wide);
            else TFNO_NORM_GRAD(64, 32, wide);
        } else if (grad_lanes(q.K, q.columns) == 64) {
            if (q.K <= 32) TFNO_NORM_GRAD(64, 4, strips);
            else TFNO_NORM_GRAD(64, 8, strips);
        } else if (grad_lanes(q.K, q.columns) == 32) TFNO_NORM_GRAD(32, 8, strips);
        else if (q.K <= 64) TFNO_NORM_GRAD(16, 2, strips);
        else if (q.K <= 128) TFNO_NORM_GRAD(16, 4, strips);
        else TFNO_NORM_GRAD(16, 8, strips);
        if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
#undef TFNO_NORM_GRAD
    hipLaunchKernelGGL(add_gain_kernel, dim3((unsigned)q.K), dim3(256), 0, stream, q.sums, blocks, q.K, q.ggain);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_rms_norm(const NormParams& q, int type, bool eight_bits, hipStream_t stream)
{
    if (q.columns == 0) return hipSuccess;
    switch (type) {
    case kC64: return eight_bits ? launch_norm<kIn32, true, true>(q, stream) : launch_norm<kIn32, true, false>(q, stream);
    case kF32: return eight_bits ? launch_norm<kIn32, false, true>(q, stream) : launch_norm<kIn32, false, false>(q, stream);
    default: return eight_bits ? launch_norm<kIn16, false, true>(q, stream) : launch_norm<kIn16, false, false>(q, stream);
    }
}

size_t rms_norm_backward_workspace(int type, long P, int K)
{
    const long blocks = grad_blocks(K, P * values_of(type));
    return (size_t)(blocks ? blocks : 1) * K * sizeof(float);
}

hipError_t launch_rms_norm_backward(const NormGradParams& q, int type, hipStream_t stream)
{
    switch (type) {
    case kC64: return launch_grad<kIn32, true>(q, stream);
    case kF32: return launch_grad<kIn32, false>(q, stream);
    default: return launch_grad<kIn16, false>(q, stream);
    }
}

}  // namespace tfno
