// Channel product of 8-bit operands with a scale for each block of 128 channels (turbofno_mix_8bit_blocks):
//
//   z[n][p] = sum_b xscale[b][p] wscale[n / 128][b] (sum over the channels k of block b of Wq[n][k] xq[k][p]) + bias[n] + residual[n][p],   y = act(z)
//
// A thread takes one position and eight channels of the result, in fp32.
#include "mix_kernel.h"

namespace tfno {

namespace {

constexpr int kRows = 8;
__device__ __forceinline__ float from_e4m3(unsigned char v) { return __builtin_amdgcn_cvt_f32_fp8((int)v, 0); }

template <int OUT, bool COMPLEX> __global__ __launch_bounds__(256) void mix_blocks_kernel(const MixBlocksParams q, long tiles)
{
    typedef typename Columns<OUT>::Value Value;
    constexpr int V = COMPLEX ? 2 : 1;
    const long id = block_index(), p = id % tiles * 256 + threadIdx.x;
    const int row0 = (int)(id / tiles) * kRows;
    if (row0 >= q.rows || p >= q.positions) return;
    const auto *x = static_cast<const unsigned char*>(q.x) + p * V, *W = static_cast<const unsigned char*>(q.W);
    float total[kRows][V] = {};
    const int blocks = (q.contraction + kScaleBlock - 1) / kScaleBlock;
    for (int b = 0; b < blocks; ++b) {
        float part[kRows][V] = {};
        const int end = q.contraction < (b + 1) * kScaleBlock ? q.contraction : (b + 1) * kScaleBlock;
        for (int k = b * kScaleBlock; k < end; ++k) {
            float v[V], w[V];
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = from_e4m3(x[k * q.ldx + i]);
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                const long at = ((long)(row0 + r < q.rows ? row0 + r : q.rows - 1) * q.contraction + k) * V;
#pragma unroll
                for (int i = 0; i < V; ++i) w[i] = from_e4m3(W[at + i]);
                part[r][0] = __builtin_fmaf(w[0], v[0], part[r][0]);
                if constexpr (COMPLEX) {
                    part[r][0] = __builtin_fmaf(-w[1], v[1], part[r][0]);
                    part[r][1] = __builtin_fmaf(w[0], v[1], __builtin_fmaf(w[1], v[0], part[r][1]));
                }
            }
        }
        const float xs = q.xscale[b * q.positions + p];
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const float ws = q.wscale[(long)((row0 + r < q.rows ? row0 + r : q.rows - 1) / kScaleBlock) * blocks + b];
#pragma unroll
            for (int i = 0; i < V; ++i) total[r][i] = __builtin_fmaf(part[r][i] * ws, xs, total[r][i]);
        }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        const int row = row0 + r;
        if (row >= q.rows) break;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float z = total[r][i];
            if (q.bias) z += value_of(static_cast<const Value*>(q.bias)[row * V + i]);
            if (q.residual) z += value_of(static_cast<const Value*>(q.residual)[row * q.ldr + p * V + i]);
            z = activate(q.act, z);
            Value* y = static_cast<Value*>(q.y) + row * q.ldy + p * V + i;
            if constexpr (OUT == kIn32) *y = z;
            else *reinterpret_cast<__bf16*>(y) = (__bf16)z;
        }
    }
}
template <int OUT, bool COMPLEX> hipError_t launch(const MixBlocksParams& q, hipStream_t stream)
{
    const long tiles = (q.positions + 255) / 256;
    hipLaunchKernelGGL((mix_blocks_kernel<OUT, COMPLEX>), grid_of(tiles * ((q.rows + kRows - 1) / kRows)), dim3(256), 0, stream, q, tiles);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_mix_8bit_blocks(const MixBlocksParams& q, int type, hipStream_t stream)
{
    if (q.columns == 0) return hipSuccess;
    switch (type) {
    case kC64: return launch<kIn32, true>(q, stream);
    case kF32: return launch<kIn32, false>(q, stream);
    default: return launch<kIn16, false>(q, stream);
    }
}

}  // namespace tfno
