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
// not fit into registers the strip is read a second time.
#include "columns.h"

namespace tfno {

namespace {

constexpr int kWaves = 8, kThreads = 64 * kWaves;

// columns a lane adds up belong to one position each (real) or two and two (complex)
template <bool COMPLEX> __device__ __forceinline__ float4_v per_position(float4_v v)
{
    if constexpr (!COMPLEX) return v;
    else { const float a = v[0] + v[1], b = v[2] + v[3]; return (float4_v){ a, a, b, b }; }
}
template <bool COMPLEX> __device__ __forceinline__ float4_v largest_per_position(float4_v v)
{
    if constexpr (!COMPLEX) return v;
    else { const float a = __builtin_fmaxf(v[0], v[1]), b = __builtin_fmaxf(v[2], v[3]); return (float4_v){ a, a, b, b }; }
}
__device__ __forceinline__ float4_v larger4(float4_v a, float4_v b)
{
    return (float4_v){ __builtin_fmaxf(a[0], b[0]), __builtin_fmaxf(a[1], b[1]), __builtin_fmaxf(a[2], b[2]), __builtin_fmaxf(a[3], b[3]) };
}
__device__ __forceinline__ float4_v magnitude(float4_v a)
{
    return (float4_v){ __builtin_fabsf(a[0]), __builtin_fabsf(a[1]), __builtin_fabsf(a[2]), __builtin_fabsf(a[3]) };
}

// Strip of a block: lane -> column and first channel, and sums over all channels of a column
template <int LANES> struct Strip {
    static constexpr int GROUPS = kThreads / LANES;     // channels side by side
    static constexpr int COLUMNS = 4 * LANES;
    const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
    // the r-th channel of a lane, or the last one
    __device__ __forceinline__ int channel(int r, int K) const { const int k = r * GROUPS + group; return k < K ? k : K - 1; }
    __device__ __forceinline__ bool has(int r, int K) const { return r * GROUPS + group < K; }
    // over the groups of a block; `shared` holds GROUPS x LANES values
    template <typename F> __device__ __forceinline__ float4_v over_channels(float4_v v, float4_v* shared, F join) const
    {
        shared[threadIdx.x] = v;
        __syncthreads();
        v = shared[lane];
#pragma unroll
        for (int g = 1; g < GROUPS; ++g) v = join(v, shared[g * LANES + lane]);
        return v;
    }
};

template <int IN> __device__ __forceinline__ RawOf<IN> read4(const void* base, long row, long ld, long column, long columns, bool full)
{
    const void* p = static_cast<const typename Columns<IN>::Value*>(base) + row * ld;
    return full ? load4<IN>(p, column) : load4_ragged<IN>(p, column, columns);
}
template <int IN> __device__ __forceinline__ void write4(void* base, long row, long ld, long column, long columns, bool full, RawOf<IN> v)
{
    void* p = static_cast<typename Columns<IN>::Value*>(base) + row * ld;
    if (full) store4<IN>(p, column, v);
    else store4_ragged<IN>(p, column, columns, v);
}

// HELD: channels per lane kept in registers; 0: read again
template <int IN, bool COMPLEX, bool EIGHT, int LANES, int HELD> __global__ __launch_bounds__(kThreads) void norm_kernel(const NormParams q)
{
    __shared__ float4_v shared[(EIGHT ? 2 : 1) * kThreads];
    const Strip<LANES> strip;
    const long column0 = (long)blockIdx.x * strip.COLUMNS, column = column0 + 4 * strip.lane;
    const bool full = column0 + strip.COLUMNS <= q.columns;
    auto value = [&](int k) {
        float4_v v = to_float<IN>(read4<IN>(q.x, k, q.ldx, column, q.columns, full));
        if (q.residual) v += to_float<IN>(read4<IN>(q.residual, k, q.ldr, column, q.columns, full));
        return v;
    };
    float4_v held[HELD ? HELD : 1];
    float4_v sum = {}, most = {};
    auto add = [&](int k, float4_v v) {
        sum += v * v;
        if constexpr (EIGHT) most = larger4(most, magnitude(v * q.gain[k]));
    };
    if constexpr (HELD) {
        // all loads first: channels beyond the last read the last one again
        RawOf<IN> x[HELD], residual[HELD];
#pragma unroll
        for (int r = 0; r < HELD; ++r) x[r] = read4<IN>(q.x, strip.channel(r, q.K), q.ldx, column, q.columns, full);
        if (q.residual)
#pragma unroll
            for (int r = 0; r < HELD; ++r) residual[r] = read4<IN>(q.residual, strip.channel(r, q.K), q.ldr, column, q.columns, full);
#pragma unroll
        for (int r = 0; r < HELD; ++r) {
            held[r] = to_float<IN>(x[r]);
            if (q.residual) held[r] += to_float<IN>(residual[r]);
            if (strip.has(r, q.K)) add(strip.channel(r, q.K), held[r]);
        }
    } else
        for (int k = strip.group; k < q.K; k += strip.GROUPS) add(k, value(k));
    sum = strip.over_channels(per_position<COMPLEX>(sum), shared, [](float4_v a, float4_v b) { return a + b; });
    if constexpr (EIGHT) most = strip.over_channels(largest_per_position<COMPLEX>(most), shared + kThreads, larger4);
    float4_v rstd, factor, inverse;
#pragma unroll
    for (int i = 0; i < 4; ++i) factor[i] = rstd[i] = __builtin_amdgcn_rsqf(sum[i] / (float)q.K + q.eps);
    if constexpr (EIGHT)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float scale = most[i] * rstd[i] * (1.f / 448.f);
            if (scale < 0x1p-126f) scale = 1.f;         // nothing but zeros, or values whose scale would be no normal number: q = 0
            inverse[i] = 1.f / scale;                   // apart from rstd: their product may leave the range of floats
            rstd[i] = scale;
        }
    if (strip.group == 0)
#pragma unroll
        for (int i = 0; i < 4; i += COMPLEX ? 2 : 1)
            if (q.rstd && column + i < q.columns) q.rstd[(column + i) / (COMPLEX ? 2 : 1)] = rstd[i];
    auto finish = [&](int k, float4_v v) {
        if (q.s) write4<IN>(q.s, k, q.lds, column, q.columns, full, from_float<IN>(v));
        v *= factor * q.gain[k];
        if constexpr (EIGHT) {
            v *= inverse;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = __builtin_amdgcn_fmed3f(v[i], -448.f, 448.f) + (v[i] - v[i]);      // a NaN stays
            int bytes = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
            bytes = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], bytes, true);
            unsigned char* p = static_cast<unsigned char*>(q.y) + k * q.ldy;
            if (full) *reinterpret_cast<uint_any*>(p + column) = (unsigned)bytes;
            else
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (column + i < q.columns) p[column + i] = (unsigned char)(bytes >> 8 * i);
        } else write4<IN>(q.y, k, q.ldy, column, q.columns, full, from_float<IN>(v));
    };
    if constexpr (HELD) {
#pragma unroll
        for (int r = 0; r < HELD; ++r)
            if (strip.has(r, q.K)) finish(strip.channel(r, q.K), held[r]);
    } else
        for (int k = strip.group; k < q.K; k += strip.GROUPS) finish(k, value(k));
}

// Persistent over strips, so that the sums of ggain stay in registers
template <int IN, bool COMPLEX, int LANES, int HELD> __global__ __launch_bounds__(kThreads) void norm_grad_kernel(const NormGradParams q, long strips)
{
    __shared__ float4_v shared[2][kThreads];
    const Strip<LANES> strip;
    float gains[HELD], ggain[HELD];
#pragma unroll
    for (int r = 0; r < HELD; ++r) {
        gains[r] = q.gain[strip.channel(r, q.K)];
        ggain[r] = 0.f;
    }
    int turn = 0;
    for (long b = blockIdx.x; b < strips; b += gridDim.x, turn ^= 1) {
        const long column0 = b * strip.COLUMNS, column = column0 + 4 * strip.lane;
        const bool full = column0 + strip.COLUMNS <= q.columns;
        RawOf<IN> gy[HELD], s[HELD];
#pragma unroll
        for (int r = 0; r < HELD; ++r) {
            gy[r] = read4<IN>(q.gy, strip.channel(r, q.K), q.ldgy, column, q.columns, full);
            s[r] = read4<IN>(q.s, strip.channel(r, q.K), q.lds, column, q.columns, full);
        }
        float4_v rstd;
#pragma unroll
        for (int i = 0; i < 4; ++i) rstd[i] = column + i < q.columns ? q.rstd[(column + i) / (COMPLEX ? 2 : 1)] : 0.f;
        float4_v along = {};
#pragma unroll
        for (int r = 0; r < HELD; ++r) {
            if (strip.has(r, q.K)) {
                const float4_v d = to_float<IN>(gy[r]) * to_float<IN>(s[r]);
                along += d * gains[r];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (column + i < q.columns) ggain[r] = __builtin_fmaf(d[i], rstd[i], ggain[r]);
            }
        }
        // two buffers: a strip's sums are read while the next strip's are written by the waves that are ahead, never two strips ahead
        along = strip.over_channels(per_position<COMPLEX>(along), shared[turn], [](float4_v a, float4_v b) { return a + b; });
        const float4_v shrink = along * rstd * rstd * rstd * (1.f / (float)q.K);
#pragma unroll
        for (int r = 0; r < HELD; ++r) {
            if (strip.has(r, q.K)) {
                const int k = strip.channel(r, q.K);
                float4_v v = to_float<IN>(gy[r]) * (rstd * gains[r]) - to_float<IN>(s[r]) * shrink;
                if (q.gs) v += to_float<IN>(read4<IN>(q.gs, k, q.ldgs, column, q.columns, full));
                write4<IN>(q.gx, k, q.ldgx, column, q.columns, full, from_float<IN>(v));
            }
        }
    }
#pragma unroll
    for (int r = 0; r < HELD; ++r) {
        float v = ggain[r];
#pragma unroll
        for (int d = 1; d < LANES; d *= 2) v += __shfl_xor(v, d, LANES);
        if (strip.lane == 0 && strip.has(r, q.K)) q.sums[(long)blockIdx.x * q.K + strip.channel(r, q.K)] = v;
    }
}

// More channels than registers hold: one strip per block, read twice
template <int IN, bool COMPLEX> __global__ __launch_bounds__(kThreads) void norm_grad_long_kernel(const NormGradParams q)
{
    constexpr int LANES = 16;
    __shared__ float4_v shared[kThreads];
    const Strip<LANES> strip;
    const long column0 = (long)blockIdx.x * strip.COLUMNS, column = column0 + 4 * strip.lane;
    const bool full = column0 + strip.COLUMNS <= q.columns;
    float4_v rstd;
#pragma unroll
    for (int i = 0; i < 4; ++i) rstd[i] = column + i < q.columns ? q.rstd[(column + i) / (COMPLEX ? 2 : 1)] : 0.f;
    float4_v along = {};
    for (int k = strip.group; k < q.K; k += strip.GROUPS) {
        const float4_v d = to_float<IN>(read4<IN>(q.gy, k, q.ldgy, column, q.columns, full)) * to_float<IN>(read4<IN>(q.s, k, q.lds, column, q.columns, full));
        along += d * q.gain[k];
    }
    along = strip.over_channels(per_position<COMPLEX>(along), shared, [](float4_v a, float4_v b) { return a + b; });
    const float4_v shrink = along * rstd * rstd * rstd * (1.f / (float)q.K);
    for (int k = strip.group; k < q.K; k += strip.GROUPS) {
        const float4_v gy = to_float<IN>(read4<IN>(q.gy, k, q.ldgy, column, q.columns, full)), s = to_float<IN>(read4<IN>(q.s, k, q.lds, column, q.columns, full));
        float4_v v = gy * (rstd * q.gain[k]) - s * shrink;
        if (q.gs) v += to_float<IN>(read4<IN>(q.gs, k, q.ldgs, column, q.columns, full));
        write4<IN>(q.gx, k, q.ldgx, column, q.columns, full, from_float<IN>(v));
        const float4_v d = gy * s;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (column + i < q.columns) sum = __builtin_fmaf(d[i], rstd[i], sum);
#pragma unroll
        for (int e = 1; e < LANES; e *= 2) sum += __shfl_xor(sum, e, LANES);
        if (strip.lane == 0) q.sums[(long)blockIdx.x * q.K + k] = sum;
    }
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

template <int IN, bool COMPLEX, bool EIGHT> hipError_t launch_norm(const NormParams& q, hipStream_t stream)
{
    const long wide = (q.columns + 255) / 256, narrow = (q.columns + 63) / 64;
    if (q.K <= 32) hipLaunchKernelGGL((norm_kernel<IN, COMPLEX, EIGHT, 64, 4>), dim3((unsigned)wide), dim3(kThreads), 0, stream, q);
    else if (q.K <= 64) hipLaunchKernelGGL((norm_kernel<IN, COMPLEX, EIGHT, 64, 8>), dim3((unsigned)wide), dim3(kThreads), 0, stream, q);
    else if (q.K <= 128) hipLaunchKernelGGL((norm_kernel<IN, COMPLEX, EIGHT, 64, 16>), dim3((unsigned)wide), dim3(kThreads), 0, stream, q);
    else if (q.K <= 256) hipLaunchKernelGGL((norm_kernel<IN, COMPLEX, EIGHT, 32, 16>), dim3((unsigned)((q.columns + 127) / 128)), dim3(kThreads), 0, stream, q);
    else if (q.K <= 512) hipLaunchKernelGGL((norm_kernel<IN, COMPLEX, EIGHT, 16, 16>), dim3((unsigned)narrow), dim3(kThreads), 0, stream, q);
    else hipLaunchKernelGGL((norm_kernel<IN, COMPLEX, EIGHT, 16, 0>), dim3((unsigned)narrow), dim3(kThreads), 0, stream, q);
    return hipGetLastError();
}

constexpr int kGradHeldChannels = 256;                  // 8 per lane, 32 side by side
constexpr long kGradBlocks = 512;                       // persistent blocks: two per CU

int grad_lanes(int K) { return K <= 64 ? 64 : 16; }
long grad_strips(int K, long columns) { return (columns + 4 * grad_lanes(K) - 1) / (4 * grad_lanes(K)); }
long grad_blocks(int K, long columns)
{
    const long strips = grad_strips(K, columns);
    return K > kGradHeldChannels || strips < kGradBlocks ? strips : kGradBlocks;
}

template <int IN, bool COMPLEX> hipError_t launch_grad(const NormGradParams& q, hipStream_t stream)
{
    const long strips = grad_strips(q.K, q.columns), blocks = grad_blocks(q.K, q.columns);
    const dim3 grid((unsigned)blocks);
    if (blocks) {
        if (q.K <= 32) hipLaunchKernelGGL((norm_grad_kernel<IN, COMPLEX, 64, 4>), grid, dim3(kThreads), 0, stream, q, strips);
        else if (q.K <= 64) hipLaunchKernelGGL((norm_grad_kernel<IN, COMPLEX, 64, 8>), grid, dim3(kThreads), 0, stream, q, strips);
        else if (q.K <= 128) hipLaunchKernelGGL((norm_grad_kernel<IN, COMPLEX, 16, 4>), grid, dim3(kThreads), 0, stream, q, strips);
        else if (q.K <= 256) hipLaunchKernelGGL((norm_grad_kernel<IN, COMPLEX, 16, 8>), grid, dim3(kThreads), 0, stream, q, strips);
        else hipLaunchKernelGGL((norm_grad_long_kernel<IN, COMPLEX>), grid, dim3(kThreads), 0, stream, q);
        if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
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
