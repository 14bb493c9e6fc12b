// The operators around the spectral layer, as their translation units and the C ABI share them. Types and activations are numbered as in
// include/turbofno.h.
#pragma once
#include "block_order.h"
#include <hip/hip_runtime.h>
#include <cstddef>

namespace tfno {

enum { kC64 = 0, kF32 = 1, kBF16 = 2 };
enum { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGeluTanh = 3 };
inline int values_of(int type) { return type == kC64 ? 2 : 1; }         // real values of an element
inline size_t size_of(int type) { return type == kC64 ? 8 : type == kF32 ? 4 : 2; }

// a grid of any number of blocks
inline dim3 grid_of(long blocks) { return grid_rows(blocks) == 1 ? dim3((unsigned)blocks) : dim3((unsigned)kGridRow, (unsigned)grid_rows(blocks)); }
__device__ __forceinline__ long block_index() { return blockIdx.y * kGridRow + blockIdx.x; }

typedef unsigned uint2_v __attribute__((ext_vector_type(2)));

struct MixParams;
// Strides and columns of the parameters are in real values already
hipError_t launch_mix_c64(const MixParams& q, bool grad, hipStream_t stream);
hipError_t launch_mix_f32(const MixParams& q, bool grad, hipStream_t stream);
hipError_t launch_mix_bf16(const MixParams& q, bool grad, hipStream_t stream);
hipError_t launch_mix_8bit(const MixParams& q, int type, hipStream_t stream);

// Gradient of the weights and of the bias: strides in elements; either result may be null
size_t mix_weight_grad_workspace(int type, long P, int N, int K);
hipError_t launch_mix_weight_grad(int type, long P, int N, int K, const void* gz, long ldgz, const void* x, long ldx, void* gW, void* gbias, void* workspace,
                                  hipStream_t stream);

// Root-mean-square norm over channels, strides in real values. 8 bits: y is q, rstd is scale.
struct NormParams {
    const void *x, *residual;
    const float* gain;
    void *s, *y;
    float* rstd;
    long columns, ldx, ldr, lds, ldy;
    int K;
    float eps;
};
hipError_t launch_rms_norm(const NormParams& q, int type, bool eight_bits, hipStream_t stream);
struct NormGradParams {
    const void *gy, *s, *gs;
    const float *gain, *rstd;
    void* gx;
    float *ggain, *sums;
    long columns, ldgy, lds, ldgs, ldgx;
    int K;
};
size_t rms_norm_backward_workspace(int type, long P, int K);
hipError_t launch_rms_norm_backward(const NormGradParams& q, int type, hipStream_t stream);

// Layer norm over channels, strides in real values. bias: K values, pairs where the fields are complex, or null. 8 bits: y is q, rstd the scales of blocks of 128
// channels, which are `positions` apart; mean is not used. drop.rng: null without dropout.
struct Drop {
    const unsigned* rng;                                // seed and offset, low words first
    unsigned threshold;                                 // elements whose word is below it are dropped
    float lift;                                         // 1 / (1 - drop)
};
struct LayerNormParams {
    const void *x, *residual;
    const float *gain, *bias;
    void *s, *y;
    float *mean, *rstd;
    long columns, positions, ldx, ldr, lds, ldy;
    int K;
    float eps;
    Drop drop;
};
hipError_t launch_layer_norm(const LayerNormParams& q, int type, bool eight_bits, hipStream_t stream);
hipError_t launch_layer_norm_dropout(const LayerNormParams& q, int type, hipStream_t stream);
hipError_t launch_layer_norm_8bit(const LayerNormParams& q, int type, hipStream_t stream);
struct LayerNormGradParams {
    const void *gy, *s, *gs;
    const float *gain, *mean, *rstd;
    void *gr, *gx;                                      // gradients of s and, with dropout, of x; without, gr is null
    float *ggain, *gbias, *sums;                        // gbias: null, or K values or pairs
    long columns, ldgy, lds, ldgs, ldgr, ldgx;
    int K;
    Drop drop;
};
size_t layer_norm_backward_workspace(int type, long P, int K);
hipError_t launch_layer_norm_backward(const LayerNormGradParams& q, int type, hipStream_t stream);

// y = residual + dropout(x), strides in real values
struct DropoutParams {
    const void *x, *residual;
    void* y;
    long columns, ldx, ldr, ldy;
    int K;
    Drop drop;
};
hipError_t launch_dropout(const DropoutParams& q, int type, hipStream_t stream);

// A field in 8 bits with a scale per position and block of 128 channels, strides in real values
constexpr int kScaleShift = 7, kScaleBlock = 1 << kScaleShift;         // channels of a scale
struct QuantiseParams {
    const void* x;
    void* q;
    float* scale;
    long columns, positions, ldx, ldq;
    int K;
};
hipError_t launch_quantise_8bit(const QuantiseParams& q, int type, hipStream_t stream);

// Channel product of 8-bit operands with scales by blocks of 128 channels, strides in real values; type of the result
struct MixBlocksParams {
    const void *x, *W, *bias, *residual;
    const float *xscale, *wscale;                       // [K / 128][positions], [N / 128][K / 128]
    void* y;
    long columns, positions, ldx, ldr, ldy;
    int rows, contraction, act;
};
hipError_t launch_mix_8bit_blocks(const MixBlocksParams& q, int type, hipStream_t stream);

// Norm over many tensors and clipping. sizes in elements; `out` may name the gradients themselves.
size_t clip_workspace(int count);
hipError_t launch_clip(int count, const void* const* grads, void* const* out, const long* sizes, const int* types, float max_norm, float* norm, void* workspace,
                       hipStream_t stream);

}  // namespace tfno
