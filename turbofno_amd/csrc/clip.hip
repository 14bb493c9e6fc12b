// Global norm of the gradients of many tensors, and clipping (turbofno_clip_grad_norm):
//
//   norm = sqrt(sum over all values |g|^2),   out = g min(1, max_norm / (norm + 1e-6))
//
// Two kernels whatever the number of tensors up to 96 (their addresses travel in the kernel's arguments; more take one launch of each for every 96):
// the first adds squares, the second adds the first's block sums - every block for itself, they are few - and scales. Squares are added in
// 64 bits, which costs nothing beside the memory traffic: no overflow, and the same order in every call. The work is cut into units of 4096 values of one tensor that
// the blocks take turns over; the second kernel walks them backwards, because the last ones read are the ones that the Infinity Cache still holds,
// and stores past the caches (100 million fp32 values: 232 -> 199 us, 4.0 TB/s of what is read and written once: 68 us for the squares, 5.9 TB/s, and
// 132 us for reading again and scaling, 6.1 TB/s). Small lists are two launches: 60 tensors of 250000 values 12.6 us, 0.5 of them
// the check on the host that no two results overlap.
// Where nothing is to be scaled and the results are the gradients themselves, the second kernel writes nothing.
#include "columns.h"
#include "kernels.h"

namespace tfno {

namespace {

constexpr int kTensors = 96, kUnit = 4096, kBlocks = 2048;

struct ClipParams {
    const void* grads[kTensors];
    void* out[kTensors];
    long sizes[kTensors];                               // real values
    unsigned first[kTensors + 1];                       // units before the tensor's
    unsigned char wide[kTensors];                       // 32-bit values
    int count;
    double* sums;                                       // of this launch's blocks; of all launches in the second kernel
    int blocks;                                         // in all launches
    float max_norm;
    float* norm;                                        // written by the launch that has it
};
static_assert(sizeof(ClipParams) <= 4096, "kernel arguments");

// unit -> tensor
__device__ __forceinline__ int tensor_of(const ClipParams& q, unsigned unit)
{
    int low = 0, high = q.count;                        // first[low] <= unit < first[high]
    while (high - low > 1) {
        const int mid = (low + high) / 2;
        if (q.first[mid] <= unit) low = mid;
        else high = mid;
    }
    return low;
}
__device__ __forceinline__ double over_block(double v, double* shared)
{
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d, 64);
    if (threadIdx.x % 64 == 0) shared[threadIdx.x / 64] = v;
    __syncthreads();
    return (shared[0] + shared[1]) + (shared[2] + shared[3]);
}
template <int IN> __device__ __forceinline__ double squares(const void* g, long at, long size)
{
    double sum = 0.;
    if (at + kUnit <= size) {
        RawOf<IN> v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = load4<IN>(g, at + 1024 * j + 4 * threadIdx.x);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float4_v f = to_float<IN>(v[j]);
#pragma unroll
            for (int i = 0; i < 4; ++i) sum += (double)f[i] * (double)f[i];
        }
    } else
        for (long e = at + threadIdx.x; e < size; e += 256) {
            const double f = value_of(static_cast<const typename Columns<IN>::Value*>(g)[e]);
            sum += f * f;
        }
    return sum;
}
template <int IN> __device__ __forceinline__ void scale(const void* g, void* out, long at, long size, float factor)
{
    if (at + kUnit <= size) {
        RawOf<IN> v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = load4<IN>(g, at + 1024 * j + 4 * threadIdx.x);
#pragma unroll
        for (int j = 0; j < 4; ++j) store4_past_caches<IN>(out, at + 1024 * j + 4 * threadIdx.x, from_float<IN>(to_float<IN>(v[j]) * factor));
    } else
        for (long e = at + threadIdx.x; e < size; e += 256) {
            const float f = value_of(static_cast<const typename Columns<IN>::Value*>(g)[e]) * factor;
            if constexpr (IN == kIn32) static_cast<float*>(out)[e] = f;
            else static_cast<__bf16*>(out)[e] = (__bf16)f;
        }
}

__global__ __launch_bounds__(256) void squares_kernel(const ClipParams q)
{
    __shared__ double shared[4];
    double sum = 0.;
    for (unsigned u = blockIdx.x; u < q.first[q.count]; u += gridDim.x) {
        const int t = tensor_of(q, u);
        const long at = (long)(u - q.first[t]) * kUnit;
        sum += q.wide[t] ? squares<kIn32>(q.grads[t], at, q.sizes[t]) : squares<kIn16>(q.grads[t], at, q.sizes[t]);
    }
    sum = over_block(sum, shared);
    if (threadIdx.x == 0) q.sums[blockIdx.x] = sum;
}

__global__ __launch_bounds__(256) void scale_kernel(const ClipParams q)
{
    __shared__ double shared[4];
    double sum = 0.;
    for (int b = threadIdx.x; b < q.blocks; b += 256) sum += q.sums[b];
    const float norm = (float)__builtin_sqrt(over_block(sum, shared));
    if (q.norm && blockIdx.x == 0 && threadIdx.x == 0) *q.norm = norm;
    const float ratio = q.max_norm / (norm + 1e-6f), factor = ratio > 1.f ? 1.f : ratio;         // a NaN stays
    const unsigned units = q.first[q.count];
    for (unsigned b = blockIdx.x; b < units; b += gridDim.x) {
        const unsigned u = units - 1 - b;
        const int t = tensor_of(q, u);
        if (factor == 1.f && q.out[t] == q.grads[t]) continue;
        const long at = (long)(u - q.first[t]) * kUnit;
        if (q.wide[t]) scale<kIn32>(q.grads[t], q.out[t], at, q.sizes[t], factor);
        else scale<kIn16>(q.grads[t], q.out[t], at, q.sizes[t], factor);
    }
}

}  // namespace

static int blocks_of(const ClipParams& q)
{
    const unsigned units = q.first[q.count];
    return units < (unsigned)kBlocks ? (units ? (int)units : 1) : kBlocks;
}

size_t clip_workspace(int count) { return (size_t)((count + kTensors - 1) / kTensors + (count == 0)) * kBlocks * sizeof(double); }

hipError_t launch_clip(int count, const void* const* grads, void* const* out, const long* sizes, const int* types, float max_norm, float* norm, void* workspace,
                       hipStream_t stream)
{
    ClipParams q;
    int filled = -1;
    auto fill = [&](int from) {                         // the tensors of a launch; its number of blocks
        if (from == filled) return blocks_of(q);
        filled = from;
        q.count = count - from < kTensors ? count - from : kTensors;
        q.first[0] = 0;
        for (int i = 0; i < q.count; ++i) {
            q.grads[i] = grads[from + i];
            q.out[i] = out[from + i];
            q.sizes[i] = sizes[from + i] * values_of(types[from + i]);
            q.wide[i] = types[from + i] != kBF16;
            q.first[i + 1] = q.first[i] + (unsigned)((q.sizes[i] + kUnit - 1) / kUnit);
        }
        return blocks_of(q);
    };
    double* sums = static_cast<double*>(workspace);
    int blocks = 0;
    q.max_norm = max_norm;
    q.norm = norm;
    for (int from = 0; from < count || from == 0; from += kTensors) {
        const int grid = fill(from);
        q.sums = sums + blocks;
        q.blocks = 0;
        hipLaunchKernelGGL(squares_kernel, dim3(grid), dim3(256), 0, stream, q);
        if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
        blocks += grid;
    }
    q.sums = sums;
    q.blocks = blocks;
    for (int from = (count > 0 ? (count - 1) / kTensors * kTensors : 0); from >= 0; from -= kTensors) {
        const int grid = fill(from);
        q.norm = from == 0 ? norm : nullptr;
        hipLaunchKernelGGL(scale_kernel, dim3(grid), dim3(256), 0, stream, q);
        if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace tfno
