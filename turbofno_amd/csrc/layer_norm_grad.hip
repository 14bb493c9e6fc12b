// Gradient of the layer norm (turbofno_layer_norm_backward). Per position p, over the K channels, with h_k = rstd (s_k - m):
//
//   g_k = gain_k gy_k,  gr_k = rstd (g_k - mean g - h_k mean Re(conj(h) g)) + gs_k,  gx_k = keep gr_k / (1 - drop)
//   ggain_k = sum_p Re(conj(h_k) gy_k),  gbias_k = sum_p gy_k
//
// Strips of positions with all of their channels, as in the norm; the blocks are persistent and hold their sums over positions in registers, a last kernel adds
// them up in a fixed order. Where the channels do not fit into registers the strip is read twice and the sums lie in the workspace.
//
// complex64, 64 channels at 2^20 positions with residual stream and dropout 528 us, 5.1 TB/s: the stream, and 5 us of the last kernel. bf16 takes as long per value for half the
// bytes, 256 channels at 131072 without either 55 us, 3.7 TB/s. From 257 channels on a compute unit has one block, whose loads nothing covers while its sums are joined and its
// results written: bf16, 512 at 65536 71 us, 2.9 TB/s, with both 99. 200 channels at 30011 positions, bf16, 19.2 us: 469 strips are one round, in which loads, sums, joins and stores follow one another
// (16.0 us at 30016, where rows start at whole cache lines), and 4 us of the last kernel.
#include "layer_norm.h"

namespace tfno {

namespace {

// what the rows of a strip share: rstd and, of the sums over channels, rstd times the mean of g and of Re(conj(h) g)
struct Shares {
    float4_v mean, rstd, level, slope;
};
template <bool COMPLEX, bool FULL> __device__ __forceinline__ void read_shares(const LayerNormGradParams& q, long column, int there, Shares& f)
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {                       // 0 beyond the last column
        f.mean[i] = FULL || i < there ? q.mean[column + i] : 0.f;
        f.rstd[i] = FULL || i < there ? q.rstd[(column + i) / (COMPLEX ? 2 : 1)] : 0.f;
    }
}
template <bool COMPLEX, int LANES> __device__ __forceinline__ void join_shares(float4_v (&sums)[2], float4_v* shared, int K, Shares& f)
{
    sums[1] = per_position<COMPLEX>(sums[1]);
    over_waves<LANES, 2>(sums, shared, sum4);
    f.level = sums[0] * (1.f / (float)K);
    f.slope = sums[1] * (1.f / (float)K);
}
// sums over positions of a channel: of its gain, and of its bias (real and imaginary parts)
template <bool COMPLEX> struct ChannelSums {
    float gain = 0.f, bias[COMPLEX ? 2 : 1] = {};
    template <bool FULL> __device__ __forceinline__ void add(float4_v gy, float4_v h, int there)
    {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (FULL || i < there) {
                gain = __builtin_fmaf(gy[i], h[i], gain);
                bias[COMPLEX ? i & 1 : 0] += gy[i];
            }
    }
    // over the lanes side by side
    template <int LANES> __device__ __forceinline__ void join()
    {
#pragma unroll
        for (int d = 1; d < LANES; d *= 2) {
            gain += __shfl_xor(gain, d, LANES);
#pragma unroll
            for (int i = 0; i < (COMPLEX ? 2 : 1); ++i) bias[i] += __shfl_xor(bias[i], d, LANES);
        }
    }
};
// one channel of a lane: gr and, with dropout, gx
template <int IN, bool COMPLEX, bool DROP, bool FULL, typename S>
__device__ __forceinline__ void write_gradients(const LayerNormGradParams& q, const S& strip, const Shares& f, long column0, int there, int r, float4_v g, float4_v h, RawOf<IN> gs,
                                                unsigned bits)
{
    float4_v v = f.rstd * (g - f.level - h * f.slope);
    if (q.gs) v += to_float<IN>(gs);
    if constexpr (DROP) {
        write_row<IN, FULL>(strip, q.gr, q.ldgr, column0, there, r, from_float<IN>(v));
        v = Keep<COMPLEX>::apply(v, bits, q.drop.lift);
    }
    write_row<IN, FULL>(strip, q.gx, q.ldgx, column0, there, r, from_float<IN>(v));
}

template <int IN, bool COMPLEX, bool DROP, int LANES, int HELD, bool FULL>
__device__ __forceinline__ void layer_norm_grad_strip(const LayerNormGradParams& q, float4_v* shared, const float* gains, long column0, int there, ChannelSums<COMPLEX> (&sums)[HELD])
{
    const Strip<LANES> strip(q.K);
    auto gain = [&](int r) { return gains[r * strip.GROUPS + strip.group()]; };
    RawOf<IN> gy[HELD], s[HELD], gs[HELD];
    const int lane_there = there - 4 * strip.lane;
    if constexpr (!FULL)
#pragma unroll
        for (int r = 0; r < HELD; ++r) gy[r] = s[r] = gs[r] = zero4<IN>();
    for_lane<FULL>(lane_there, [&](auto whole) {
#pragma unroll
        for (int r = 0; r < HELD; ++r) {
            gy[r] = strip.template read<IN, decltype(whole)::value>(q.gy, q.ldgy, column0, there, r);
            s[r] = strip.template read<IN, decltype(whole)::value>(q.s, q.lds, column0, there, r);
        }
    });
    const long column = column0 + 4 * strip.lane;
    Shares f;
    read_shares<COMPLEX, FULL>(q, column, lane_there, f);
    unsigned bits[HELD] = {};
    if constexpr (DROP) {
        const auto keep = keep_of<COMPLEX, DROP>(q.drop, column);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int r = 0; r < HELD; r += 2) keep.pair(strip.channel(r), strip.channel(r + 1), bits[r], bits[r + 1]);
    }
    float4_v joint[2] = {};
#pragma unroll
    for (int r = 0; r < HELD; ++r)
        if (strip.has(r)) {
            const float4_v v = to_float<IN>(gy[r]), h = (to_float<IN>(s[r]) - f.mean) * f.rstd, g = v * gain(r);
            joint[0] += g;
            joint[1] += g * h;
            sums[r].template add<FULL>(v, h, lane_there);
        }
    if (q.gs)
        for_lane<FULL>(lane_there, [&](auto whole) {
#pragma unroll
            for (int r = 0; r < HELD; ++r) gs[r] = strip.template read<IN, decltype(whole)::value>(q.gs, q.ldgs, column0, there, r);
        });
    join_shares<COMPLEX, LANES>(joint, shared, q.K, f);
#pragma unroll
    for (int r = 0; r < HELD; ++r)
        if (strip.has(r)) {
            if constexpr (IN == kIn16) asm volatile("" : "+v"(gy[r]), "+v"(s[r]));       // widened again, not held in twice the registers
            write_gradients<IN, COMPLEX, DROP, FULL>(q, strip, f, column0, there, r, to_float<IN>(gy[r]) * gain(r), (to_float<IN>(s[r]) - f.mean) * f.rstd, gs[r], bits[r]);
        }
}
// a block's sums of all channels: K of the gain, then K or 2 K of the bias
template <bool COMPLEX> __device__ __forceinline__ void put_sums(float* sums, int K, int k, const ChannelSums<COMPLEX>& v)
{
    sums[k] = v.gain;
#pragma unroll
    for (int i = 0; i < (COMPLEX ? 2 : 1); ++i) sums[K + (COMPLEX ? 2 : 1) * k + i] = v.bias[i];
}
// Persistent over strips, so that the sums of the channels stay in registers
template <int IN, bool COMPLEX, bool DROP, int LANES, int HELD> __global__ __launch_bounds__(kThreads, 2) void layer_norm_grad_kernel(const LayerNormGradParams q, const StripTurns turns)
{
    // two buffers: a strip's sums are read while the next strip's are written by the waves that are ahead, never two strips ahead
    __shared__ float4_v shared[2][2 * (kThreads / 64) * LANES];
    __shared__ float gains[HELD * Strip<LANES>::GROUPS];
    for (int k = threadIdx.x; k < HELD * Strip<LANES>::GROUPS; k += kThreads) gains[k] = q.gain[k < q.K ? k : q.K - 1];
    __syncthreads();
    ChannelSums<COMPLEX> sums[HELD];
    int turn = 0;
    const long last = turns.last(blockIdx.x);
    for (long b = turns.first(blockIdx.x); b < last; b += turns.step, turn ^= 1) {
        const long column0 = b * Strip<LANES>::COLUMNS;
        if (column0 + Strip<LANES>::COLUMNS <= q.columns)
            layer_norm_grad_strip<IN, COMPLEX, DROP, LANES, HELD, true>(q, shared[turn], gains, column0, Strip<LANES>::COLUMNS, sums);
        else layer_norm_grad_strip<IN, COMPLEX, DROP, LANES, HELD, false>(q, shared[turn], gains, column0, (int)(q.columns - column0), sums);
    }
    const Strip<LANES> strip(q.K);
    float* to = q.sums + (long)blockIdx.x * q.K * (COMPLEX ? 3 : 2);
#pragma unroll
    for (int r = 0; r < HELD; ++r) {
        sums[r].template join<LANES>();
        if (strip.lane == 0 && strip.has(r)) put_sums(to, q.K, strip.channel(r), sums[r]);
    }
}

// More channels than registers hold: the strip is read twice. The block's sums are added up in its part of the workspace, each channel's by one lane
template <int IN, bool COMPLEX, bool DROP, int LANES, bool FULL>
__device__ __forceinline__ void layer_norm_grad_long_strip(const LayerNormGradParams& q, float4_v* shared, long column0, int there, float* sums, bool first)
{
    const Strip<LANES> strip(q.K);
    const int lane_there = there - 4 * strip.lane, rounds = (q.K + strip.GROUPS - 1) / strip.GROUPS;
    const long column = column0 + 4 * strip.lane;
    Shares f;
    read_shares<COMPLEX, FULL>(q, column, lane_there, f);
    float4_v joint[2] = {};
    for (int r0 = 0; r0 < rounds; r0 += kChunk) {
        RawOf<IN> gy[kChunk], s[kChunk];
        if constexpr (!FULL)
#pragma unroll
            for (int r = 0; r < kChunk; ++r) gy[r] = s[r] = zero4<IN>();
        for_lane<FULL>(lane_there, [&](auto whole) {
#pragma unroll
            for (int r = 0; r < kChunk; ++r) {
                gy[r] = strip.template read<IN, decltype(whole)::value>(q.gy, q.ldgy, column0, there, r0 + r);
                s[r] = strip.template read<IN, decltype(whole)::value>(q.s, q.lds, column0, there, r0 + r);
            }
        });
#pragma unroll
        for (int r = 0; r < kChunk; ++r)
            if (strip.has(r0 + r)) {
                const float4_v g = to_float<IN>(gy[r]) * q.gain[strip.channel(r0 + r)];
                joint[0] += g;
                joint[1] += g * ((to_float<IN>(s[r]) - f.mean) * f.rstd);
            }
    }
    join_shares<COMPLEX, LANES>(joint, shared, q.K, f);
    const auto keep = keep_of<COMPLEX, DROP>(q.drop, column);
    constexpr int PART = 4;
    for (int r0 = 0; r0 < rounds; r0 += PART) {
        RawOf<IN> gy[PART], s[PART], gs[PART];
        unsigned bits[PART] = {};
        if constexpr (!FULL)
#pragma unroll
            for (int r = 0; r < PART; ++r) gy[r] = s[r] = gs[r] = zero4<IN>();
        for_lane<FULL>(lane_there, [&](auto whole) {
#pragma unroll
            for (int r = 0; r < PART; ++r) {
                gy[r] = strip.template read<IN, decltype(whole)::value>(q.gy, q.ldgy, column0, there, r0 + r);
                s[r] = strip.template read<IN, decltype(whole)::value>(q.s, q.lds, column0, there, r0 + r);
                if (q.gs) gs[r] = strip.template read<IN, decltype(whole)::value>(q.gs, q.ldgs, column0, there, r0 + r);
            }
        });
        if constexpr (DROP)
#pragma unroll
            for (int r = 0; r < PART; r += 2) keep.pair(strip.channel(r0 + r), strip.channel(r0 + r + 1), bits[r], bits[r + 1]);
#pragma unroll
        for (int r = 0; r < PART; ++r) {
            if (!strip.has(r0 + r)) continue;           // the lanes of a group together
            const int k = strip.channel(r0 + r);
            const float4_v v = to_float<IN>(gy[r]), h = (to_float<IN>(s[r]) - f.mean) * f.rstd;
            write_gradients<IN, COMPLEX, DROP, FULL>(q, strip, f, column0, there, r0 + r, v * q.gain[k], h, gs[r], bits[r]);
            ChannelSums<COMPLEX> sum;
            sum.template add<FULL>(v, h, lane_there);
            sum.template join<LANES>();
            if (strip.lane == 0) {
                if (!first) {
                    sum.gain += sums[k];
#pragma unroll
                    for (int i = 0; i < (COMPLEX ? 2 : 1); ++i) sum.bias[i] += sums[q.K + (COMPLEX ? 2 : 1) * k + i];
                }
                put_sums(sums, q.K, k, sum);
            }
        }
    }
}
template <int IN, bool COMPLEX, bool DROP, int LANES> __global__ __launch_bounds__(kThreads, 2) void layer_norm_grad_long_kernel(const LayerNormGradParams q, const StripTurns turns)
{
    __shared__ float4_v shared[2][2 * (kThreads / 64) * LANES];
    constexpr int COLUMNS = Strip<LANES>::COLUMNS;
    float* to = q.sums + (long)blockIdx.x * q.K * (COMPLEX ? 3 : 2);
    int turn = 0;
    const long start = turns.first(blockIdx.x), last = turns.last(blockIdx.x);
    if (start >= last)                                  // no strip: its sums are added up all the same
        for (int k = threadIdx.x; k < q.K * (COMPLEX ? 3 : 2); k += kThreads) to[k] = 0.f;
    for (long b = start; b < last; b += turns.step, turn ^= 1) {
        const long column0 = b * COLUMNS;
        const bool first = b == start;
        if (column0 + COLUMNS <= q.columns) layer_norm_grad_long_strip<IN, COMPLEX, DROP, LANES, true>(q, shared[turn], column0, COLUMNS, to, first);
        else layer_norm_grad_long_strip<IN, COMPLEX, DROP, LANES, false>(q, shared[turn], column0, (int)(q.columns - column0), to, first);
    }
}

// The blocks' sums, 16 values per block, always in the same order; those of the bias may not be asked for
__global__ __launch_bounds__(1024) void add_sums_kernel(const float* __restrict__ sums, long blocks, int K, int count, float* __restrict__ ggain, float* __restrict__ gbias)
{
    __shared__ float part[16][17];
    const int c = threadIdx.x % 16, r = threadIdx.x / 16, value = blockIdx.x * 16 + c;
    float v = 0.f;
    if (value < count)
#pragma unroll 8
        for (long b = r; b < blocks; b += 64) v += sums[b * count + value];
    v += __shfl_xor(v, 16, 64);                         // four rows of a wave
    v += __shfl_xor(v, 32, 64);
    if (threadIdx.x % 64 < 16) part[r / 4][c] = v;
    __syncthreads();
    if (r || value >= count) return;
#pragma unroll
    for (int i = 1; i < 16; ++i) v += part[i][c];
    if (value < K) ggain[value] = v;
    else if (gbias) gbias[value - K] = v;
}

// Lanes side by side and channels held per lane (0: read twice)
template <int IN, bool COMPLEX, bool DROP, int LANES, int HELD> hipError_t launch_as(const LayerNormGradParams& q, hipStream_t stream)
{
    const long strips = (q.columns + 4 * LANES - 1) / (4 * LANES), each = strips_of_launch(strips);
    const int count = q.K * (COMPLEX ? 3 : 2);
    long blocks = 0;
    for (long base = 0; base < strips; base += each) {
        const long these = std::min(each, strips - base);
        const StripTurns turns(base, these, LANES >= 4 && run_together(q.columns, IN, these));
        LayerNormGradParams part = q;
        part.sums += blocks * count;
        blocks += turns.blocks();
        const dim3 grid((unsigned)turns.blocks()), block(kThreads);
        if constexpr (HELD > 0) hipLaunchKernelGGL((layer_norm_grad_kernel<IN, COMPLEX, DROP, LANES, HELD>), grid, block, 0, stream, part, turns);
        else hipLaunchKernelGGL((layer_norm_grad_long_kernel<IN, COMPLEX, DROP, LANES>), grid, block, 0, stream, part, turns);
        if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(add_sums_kernel, dim3((unsigned)((count + 15) / 16)), dim3(1024), 0, stream, q.sums, blocks, q.K, count, q.ggain, q.gbias);
    return hipGetLastError();
}
template <int IN, bool COMPLEX, bool DROP> hipError_t launch_grad(const LayerNormGradParams& q, hipStream_t stream)
{
    if (far_apart(std::max(std::max(q.ldgy, q.lds), std::max(std::max(q.ldgs, q.ldgr), q.ldgx))))      // with 64 lanes side by side a lane's part of an address has no channel in it
        return q.K <= 64 ? launch_as<IN, COMPLEX, DROP, 64, 8>(q, stream) : launch_as<IN, COMPLEX, DROP, 64, 0>(q, stream);
    if (q.K <= 64 && q.columns >= kFewColumns) return q.K <= 32 ? launch_as<IN, COMPLEX, DROP, 64, 4>(q, stream) : launch_as<IN, COMPLEX, DROP, 64, 8>(q, stream);
    if (q.K <= 64) return launch_as<IN, COMPLEX, DROP, 16, 2>(q, stream);
    // all with residual stream and dropout: bf16, 128 channels at 262144 columns 84 us, 90 with 32 lanes
    if (q.K <= 128) return launch_as<IN, COMPLEX, DROP, 16, 4>(q, stream);
    if (q.K <= 256) return launch_as<IN, COMPLEX, DROP, 16, 8>(q, stream);
    const bool few = q.columns < kNarrowColumns;
    // bf16, 512 channels at 65536 columns 99 us (8 lanes 131, read twice 132), 300 at 4000 18.6 us (8 lanes 12.3); 32 bits spill with 16 channels
    if (q.K <= 512) {
        if constexpr (IN == kIn16)
            if (!few) return launch_as<IN, COMPLEX, DROP, 16, 16>(q, stream);
        return launch_as<IN, COMPLEX, DROP, 8, 8>(q, stream);
    }
    // float32, 1024 channels at 4000 columns 28.6 us, 53 where the strip is read twice, at 16384 113 and 100; bf16, 2048 at 2000 44 and 95
    if (q.K <= 1024 && few) return launch_as<IN, COMPLEX, DROP, 4, 8>(q, stream);
    if (q.K <= 2048 && q.columns < kNarrowColumns / 2) return launch_as<IN, COMPLEX, DROP, 2, 8>(q, stream);
    return few ? launch_as<IN, COMPLEX, DROP, 4, 0>(q, stream) : launch_as<IN, COMPLEX, DROP, 16, 0>(q, stream);
}
template <int IN, bool COMPLEX> hipError_t launch_grad(const LayerNormGradParams& q, hipStream_t stream)
{
    return q.drop.rng ? launch_grad<IN, COMPLEX, true>(q, stream) : launch_grad<IN, COMPLEX, false>(q, stream);
}

}  // namespace

size_t layer_norm_backward_workspace(int type, long P, int K)
{
    return (size_t)grad_rows(P * values_of(type)) * K * (1 + values_of(type)) * sizeof(float);
}

hipError_t launch_layer_norm_backward(const LayerNormGradParams& q, int type, hipStream_t stream)
{
    switch (type) {
    case kC64: return launch_grad<kIn32, true>(q, stream);
    case kF32: return launch_grad<kIn32, false>(q, stream);
    default: return launch_grad<kIn16, false>(q, stream);
    }
}

}  // namespace tfno
