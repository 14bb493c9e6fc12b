// Layer norm over channels with the addition of a residual and dropout (turbofno_layer_norm), with its result in 8 bits (turbofno_layer_norm_8bit): the kernel and its
// variants, of which layer_norm.hip, layer_norm_dropout.hip and layer_norm_8bit.hip each build one form. Per position p, over the K channels:
//
//   s = residual + keep x / (1 - drop),  m = mean_k s_k,  rstd = 1 / sqrt(mean_k |s_k - m|^2 + eps),  y_k = gain_k rstd (s_k - m) + bias_k
//   8 bit     per block of 128 channels: scale = max |y_k| / 448, q_k = e4m3(y_k / scale)
//
// As in the root-mean-square norm a block takes a strip of positions with all of their channels and keeps them in registers: every byte moves once. The deviations
// are squared after the mean is known, which two joins over the waves cost: a sum of squares less the square of the sum loses what a mean far from zero takes.
// Where the channels do not fit into registers the strip is read twice, and the squares are taken of what is left over the mean of the first channels.
//
// The stream bounds it where a compute unit has two blocks, whose loads and sums overlap: complex64, 64 channels at 2^20 positions with residual and dropout 405 us, 5.3 TB/s (a
// copy: 5.1); bf16, 128 channels at 262144 60 us, 4.5 TB/s. From 257 channels on registers leave room for one: bf16, 512 channels at 65536 with residual 64 us, 4.2 TB/s, into 8 bits
// 75 us, 3.1 TB/s, with a third join. Small calls: 64 channels at 128 positions 5.5 us, of which the kernel is 3.
#pragma once
#include "layer_norm.h"

namespace tfno {

// One channel's gain and bias
template <bool COMPLEX> struct Affine {
    float gain, bias[COMPLEX ? 2 : 1];
    __device__ __forceinline__ float4_v biases() const { return (float4_v){ bias[0], bias[COMPLEX], bias[0], bias[COMPLEX] }; }
};
template <bool COMPLEX> __device__ __forceinline__ Affine<COMPLEX> affine_of(const float* gain, const float* bias, int k)
{
    Affine<COMPLEX> a;
    a.gain = gain[k];
#pragma unroll
    for (int i = 0; i < (COMPLEX ? 2 : 1); ++i) a.bias[i] = bias ? bias[(COMPLEX ? 2 : 1) * (long)k + i] : 0.f;
    return a;
}

// HELD: channels per lane kept in registers (an even number); 0: read again
template <int IN, bool COMPLEX, bool DROP, bool EIGHT, int LANES, int HELD, bool FULL>
__device__ __forceinline__ void layer_norm_strip(const LayerNormParams& q, float4_v* shared, const Affine<COMPLEX>* affines, long column0, int there)
{
    typedef Strip<LANES> S;
    constexpr int PARTS = COMPLEX ? 2 : 1, ROWS = HELD ? HELD : kChunk, OF_BLOCK = kScaleBlock / S::GROUPS, AREA = kThreads / 64 * LANES;
    const S strip(q.K);
    const int lane_there = there - 4 * strip.lane;
    const long column = column0 + 4 * strip.lane;
    const float per_channel = 1.f / (float)q.K;
    const auto keep = keep_of<COMPLEX, DROP>(q.drop, column);
    // channels first ... first + COUNT - 1 of the lane
    auto fetch = [&](int first, auto& v) {
        constexpr int COUNT = sizeof(v) / sizeof(v[0]);
        RawOf<IN> x[COUNT], residual[COUNT];            // all loads first: channels beyond the last read another one
        if constexpr (!FULL)
#pragma unroll
            for (int r = 0; r < COUNT; ++r) x[r] = residual[r] = zero4<IN>();
        for_lane<FULL>(lane_there, [&](auto whole) {
            constexpr bool WHOLE = decltype(whole)::value;
#pragma unroll
            for (int r = 0; r < COUNT; ++r) x[r] = strip.template read<IN, WHOLE>(q.x, q.ldx, column0, there, first + r);
            if (q.residual)
#pragma unroll
                for (int r = 0; r < COUNT; ++r) residual[r] = strip.template read<IN, WHOLE>(q.residual, q.ldr, column0, there, first + r);
        });
        unsigned bits[COUNT];
        if constexpr (DROP) {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int r = 0; r < COUNT; r += 2) keep.pair(strip.channel(first + r), strip.channel(first + r + 1), bits[r], bits[r + 1]);
        }
#pragma unroll
        for (int r = 0; r < COUNT; ++r) {
            float4_v f = to_float<IN>(x[r]);
            if constexpr (DROP) f = Keep<COMPLEX>::apply(f, bits[r], q.drop.lift);
            if (q.residual) f += to_float<IN>(residual[r]);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[r][i] = f[i];
        }
    };
    float held[ROWS][4];
    fetch(0, held);
    if constexpr (HELD > 0) __syncthreads();            // gains and biases
    float4_v sum[1] = {};
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
        if (strip.has(r)) sum[0] += four(held[r]);
    over_waves<LANES, 1>(sum, shared, sum4);
    const int counted = HELD || q.K < ROWS * S::GROUPS ? q.K : ROWS * S::GROUPS;
    float4_v mean = HELD ? sum[0] * per_channel : sum[0] * (1.f / (float)counted);      // of the first channels, if not all are held
    float4_v rest[2] = {};                              // squares, sum over the mean
    auto deviate = [&](int first, auto& v) {
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
            if (strip.has(first + r)) {
                const float4_v d = four(v[r]) - mean;
                rest[0] += d * d;
                if constexpr (HELD == 0) rest[1] += d;
            }
    };
    deviate(0, held);
    const int rounds = (q.K + S::GROUPS - 1) / S::GROUPS;
    if constexpr (HELD == 0)
        for (int first = ROWS; first < rounds; first += ROWS) {
            fetch(first, held);
            deviate(first, held);
        }
    rest[0] = per_position<COMPLEX>(rest[0]);
    over_waves<LANES, HELD ? 1 : 2>(reinterpret_cast<float4_v (&)[HELD ? 1 : 2]>(rest), shared + AREA, sum4);
    float4_v variance = rest[0] * per_channel, rstd;
    if constexpr (HELD == 0) {
        const float4_v shift = rest[1] * per_channel, less = per_position<COMPLEX>(shift * shift);
        mean += shift;
#pragma unroll
        for (int i = 0; i < 4; ++i) variance[i] = __builtin_elementwise_maximum(variance[i] - less[i], 0.f);        // a NaN stays
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) rstd[i] = reciprocal_root(variance[i] + q.eps);
    if constexpr (!EIGHT)
        if (strip.group() == 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (FULL || i < lane_there) {
                    if (q.mean) q.mean[column + i] = mean[i];
                    if (q.rstd && i % PARTS == 0) q.rstd[(column + i) / PARTS] = rstd[i];
                }
        }
    auto result = [&](int r, float4_v v) {
        const Affine<COMPLEX> a = HELD ? affines[r * S::GROUPS + strip.group()] : affine_of<COMPLEX>(q.gain, q.bias, strip.channel(r));
        const float4_v h = (v - mean) * rstd, b = a.biases();
        float4_v y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = __builtin_fmaf(h[i], a.gain, b[i]);
        return y;
    };
    if constexpr (!EIGHT) {
        auto finish = [&](int first, auto& v) {         // v is there before either result is written: they may take its operands' place
#pragma unroll
            for (int r = 0; r < ROWS; ++r)
                if (strip.has(first + r)) {
                    if (q.s) write_row<IN, FULL>(strip, q.s, q.lds, column0, there, first + r, from_float<IN>(four(v[r])));
                    write_row<IN, FULL>(strip, q.y, q.ldy, column0, there, first + r, from_float<IN>(result(first + r, four(v[r]))));
                }
        };
        if constexpr (HELD > 0) finish(0, held);
        else
            for (int first = 0; first < rounds; first += ROWS) {
                fetch(first, held);
                finish(first, held);
            }
    } else {
        // COUNT blocks of 128 channels, in v from its first row on
        auto finish = [&](int block, auto& v) {
            constexpr int COUNT_ROWS = sizeof(v) / sizeof(v[0]), COUNT = (COUNT_ROWS + OF_BLOCK - 1) / OF_BLOCK;
            const int first = block * OF_BLOCK;
            float4_v most[COUNT] = {};
#pragma unroll
            for (int r = 0; r < COUNT_ROWS; ++r)
                if (strip.has(first + r)) {
                    if (q.s) write_row<IN, FULL>(strip, q.s, q.lds, column0, there, first + r, from_float<IN>(four(v[r])));
                    const float4_v y = result(first + r, four(v[r]));
                    most[r / OF_BLOCK] = larger4(most[r / OF_BLOCK], magnitude(y));
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[r][i] = y[i];
                }
            // HELD = 0: two areas in turns, so that a block's maxima are read before another wave's next but one are written
            block_maxima<COMPLEX, LANES>(most, shared + (HELD ? 2 : 2 + (block & 1)) * AREA + (HELD ? 0 : AREA));
#pragma unroll
            for (int c = 0; c < COUNT; ++c) {
                if ((block + c) * kScaleBlock >= q.K) break;
                const Divisor by = write_scales<COMPLEX, FULL>(q.rstd + (block + c) * q.positions, column, lane_there, strip.group() == 0, most[c]);
#pragma unroll
                for (int r = c * OF_BLOCK; r < (c + 1) * OF_BLOCK && r < COUNT_ROWS; ++r)
                    if (strip.has(first + r)) write_row<kIn8, FULL>(strip, q.y, q.ldy, column0, there, first + r, eight_bits(four(v[r]), by));
            }
        };
        if constexpr (HELD > 0) finish(0, held);
        else {
            float rows[OF_BLOCK][4];
            for (int block = 0; block * kScaleBlock < q.K; ++block) {
                fetch(block * OF_BLOCK, rows);
                finish(block, rows);
            }
        }
    }
}
// areas of LDS for joins: the mean's, the squares' (two values where channels are read again), and the maxima of blocks of 128 channels
template <bool EIGHT, int LANES, int HELD> constexpr int kAreas = (HELD ? 2 : 3) + (!EIGHT ? 0 : HELD ? (HELD * (kThreads / LANES) + kScaleBlock - 1) / kScaleBlock : 2);
template <int IN, bool COMPLEX, bool DROP, bool EIGHT, int LANES, int HELD>
__global__ __launch_bounds__(kThreads, (IN == kIn16 && HELD < 16 && !(EIGHT && LANES < 16) ? 4 : 2)) void layer_norm_kernel(const LayerNormParams q, long run)
{
    typedef Strip<LANES> S;
    const long id = block_index(), column0 = (run ? side_by_side(id, run) : id) * S::COLUMNS;
    if (column0 >= q.columns) return;
    __shared__ float4_v shared[kAreas<EIGHT, LANES, HELD> * (kThreads / 64) * LANES];
    __shared__ Affine<COMPLEX> affines[HELD ? HELD * S::GROUPS : 1];
    if constexpr (HELD > 0)
        for (int k = threadIdx.x; k < HELD * S::GROUPS; k += kThreads) affines[k] = affine_of<COMPLEX>(q.gain, q.bias, k < q.K ? k : q.K - 1);
    if (column0 + S::COLUMNS <= q.columns) layer_norm_strip<IN, COMPLEX, DROP, EIGHT, LANES, HELD, true>(q, shared, affines, column0, S::COLUMNS);
    else layer_norm_strip<IN, COMPLEX, DROP, EIGHT, LANES, HELD, false>(q, shared, affines, column0, (int)(q.columns - column0));
}

template <int IN, bool COMPLEX, bool DROP, bool EIGHT, int LANES, int HELD> hipError_t launch_as(const LayerNormParams& q, hipStream_t stream)
{
    const long strips = (q.columns + 4 * LANES - 1) / (4 * LANES), run = run_together(q.columns, IN, strips) ? (strips + 7) / 8 : 0;
    hipLaunchKernelGGL((layer_norm_kernel<IN, COMPLEX, DROP, EIGHT, LANES, HELD>), grid_of(run ? 8 * run : strips), dim3(kThreads), 0, stream, q, run);
    return hipGetLastError();
}
// Lanes side by side and channels held: wide strips read long pieces of a row, narrow ones give the GPU more blocks, and hold more channels
template <int IN, bool COMPLEX, bool DROP, bool EIGHT> hipError_t launch(const LayerNormParams& q, hipStream_t stream)
{
    if (far_apart(std::max(std::max(q.ldx, q.ldr), std::max(q.lds, q.ldy)))) {         // with 64 lanes side by side a lane's part of an address has no channel in it
        if (q.K <= 32) return launch_as<IN, COMPLEX, DROP, EIGHT, 64, 4>(q, stream);
        if (q.K <= 64) return launch_as<IN, COMPLEX, DROP, EIGHT, 64, 8>(q, stream);
        return launch_as<IN, COMPLEX, DROP, EIGHT, 64, 0>(q, stream);
    }
    if (q.K <= 64 && q.columns >= kFewColumns) return q.K <= 32 ? launch_as<IN, COMPLEX, DROP, EIGHT, 64, 4>(q, stream) : launch_as<IN, COMPLEX, DROP, EIGHT, 64, 8>(q, stream);
    if (q.K <= 256 && q.columns < kFewColumns / (q.K <= 64 ? 1 : 2)) {
        if (q.K <= 64) return launch_as<IN, COMPLEX, DROP, EIGHT, 16, 2>(q, stream);
        if (q.K <= 128) return launch_as<IN, COMPLEX, DROP, EIGHT, 16, 4>(q, stream);
        return launch_as<IN, COMPLEX, DROP, EIGHT, 16, 8>(q, stream);
    }
    // all with residual: bf16, 128 channels at 262144 columns 60 us, 65 with 64 lanes; float32, 256 at 65536 53 us, 58 with 16
    if (q.K <= 128) return launch_as<IN, COMPLEX, DROP, EIGHT, 32, 8>(q, stream);
    if (q.K <= 256) return launch_as<IN, COMPLEX, DROP, EIGHT, 32, 16>(q, stream);
    // float32, 512 channels at 4000 columns 8.7 us, 11.2 with 16 lanes; at 16000 24.1 and 23.0
    if (q.K <= 512) return q.columns < kNarrowColumns ? launch_as<IN, COMPLEX, DROP, EIGHT, 8, 8>(q, stream) : launch_as<IN, COMPLEX, DROP, EIGHT, 16, 16>(q, stream);
    // bf16, 1024 channels, strips read once with 4 or 8 lanes, and twice with 16: at 1000 columns 10.3, 11.3 and 25 us, at 4000 18, 13 and 27, at 16000 60, 42 and 38;
    // float32 at 16000 86, 64 and 75 us, at 32000 178, 127 and 158
    if (q.K <= 1024) {
        if (q.columns <= 1024) return launch_as<IN, COMPLEX, DROP, EIGHT, 4, 8>(q, stream);
        if (q.columns < kNarrowColumns || (IN == kIn32 && !EIGHT)) return launch_as<IN, COMPLEX, DROP, EIGHT, 8, 16>(q, stream);
    }
    // bf16, 2048 channels at 1000 columns 16 us, 50 with 16 lanes; at 16000 157 and 87
    if (q.columns < kNarrowColumns) return q.K <= 2048 ? launch_as<IN, COMPLEX, DROP, EIGHT, 4, 16>(q, stream) : launch_as<IN, COMPLEX, DROP, EIGHT, 4, 0>(q, stream);
    return launch_as<IN, COMPLEX, DROP, EIGHT, 16, 0>(q, stream);
}
template <bool DROP, bool EIGHT> hipError_t launch(const LayerNormParams& q, int type, hipStream_t stream)
{
    switch (type) {
    case kC64: return launch<kIn32, true, DROP, EIGHT>(q, stream);
    case kF32: return launch<kIn32, false, DROP, EIGHT>(q, stream);
    default: return launch<kIn16, false, DROP, EIGHT>(q, stream);
    }
}

}  // namespace tfno
