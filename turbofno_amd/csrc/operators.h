// The operators around the spectral layer, as their translation units and the C ABI share them. Types and activations are numbered as in
// include/turbofno.h.
#pragma once
#include <hip/hip_runtime.h>
#include <cstddef>

namespace tfno {

enum { kC64 = 0, kF32 = 1, kBF16 = 2 };
enum { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGeluTanh = 3 };
inline int values_of(int type) { return type == kC64 ? 2 : 1; }         // real values of an element
inline size_t size_of(int type) { return type == kC64 ? 8 : type == kF32 ? 4 : 2; }

// A grid of any number of blocks: a dimension of a launch holds fewer than 2^32 threads, so from 2^22 blocks (of up to 512) on there are several rows of
// them, whose last blocks may have nothing to do
constexpr long kGridRow = 1L << 22;
inline dim3 grid_of(long blocks) { return blocks <= kGridRow ? dim3((unsigned)blocks) : dim3((unsigned)kGridRow, (unsigned)((blocks + kGridRow - 1) / kGridRow)); }
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

// Norm over many tensors and clipping. sizes in elements; `out` may name the gradients themselves.
size_t clip_workspace(int count);
hipError_t launch_clip(int count, const void* const* grads, void* const* out, const long* sizes, const int* types, float max_norm, float* norm, void* workspace,
                       hipStream_t stream);

}  // namespace tfno
