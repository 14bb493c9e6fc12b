// Gradient of the channel product's weights and bias (turbofno_mix_weight_grad):
//
//   gW[n][k] = sum_p gz[n][p] conj(x[k][p]),   gbias[n] = sum_p gz[n][p]
//
// A contraction over positions, which are contiguous in both operands: a lane reads eight consecutive real values of a row of gz and of a row of
// x, the quarters of a wave 32 of them, and has the operands of its matrix instructions. Complex rows are (re, im) pairs: gz as it is against
// (re, im) of x for the real part, against (-im, re) for the imaginary part. 32-bit values are split into bf16 parts (bf16_split.h), 16-bit ones
// are exact; sums are fp32. gbias takes its sums from the values of gz that pass by.
// A block takes a tile of 64 rows n and 64 real (32 complex) rows k and a part of the positions: its four waves four steps of 32 real values side by
// side, then those as many steps further as all blocks take together. So the blocks move through the rows as one window: with a contiguous part for each
// block they all would stand at the same offset of their parts, on the same few memory channels. The blocks' sums go to the workspace and are added in a second kernel, always in the
// same order: results do not change from call to call.
// An infinite operand, or one above the largest bf16 number (3.3895e38), makes the sums it takes part in infinite or NaN.
#include "columns.h"

namespace tfno {

namespace {

constexpr int kGradRows = 64;                           // rows n of a tile
constexpr int kStep = 32;                               // real values of a step

struct GradParams {
    const void *g, *x;
    long ldg, ldx, columns;                             // real values
    int N, K;
    float* sums;                                        // [splits][N K V + N V]
    int splits, ktiles, tiles;
};

template <int IN> struct Eight;
template <> struct Eight<kIn32> { float4_v lo, hi; };
template <> struct Eight<kIn16> { uint4_v v; };
typedef uint4_v uint4_any __attribute__((aligned(2)));

template <int IN> __device__ __forceinline__ Eight<IN> load8(const void* row, long column, long columns, bool full)
{
    const auto* p = static_cast<const typename Columns<IN>::Value*>(row) + column;
    Eight<IN> e;
    if (full) {
        if constexpr (IN == kIn32) {
            e.lo = *reinterpret_cast<const float4_any*>(p);
            e.hi = *reinterpret_cast<const float4_any*>(p + 4);
        } else e.v = *reinterpret_cast<const uint4_any*>(p);
        return e;
    }
    auto at = [&](int i) { return column + i < columns ? p[i] : (typename Columns<IN>::Value)0; };
    if constexpr (IN == kIn32) {
        e.lo = (float4_v){ at(0), at(1), at(2), at(3) };
        e.hi = (float4_v){ at(4), at(5), at(6), at(7) };
    } else
#pragma unroll
        for (int j = 0; j < 4; ++j) e.v[j] = at(2 * j) | (unsigned)at(2 * j + 1) << 16;
    return e;
}
__device__ __forceinline__ void operand(const Eight<kIn32>& e, SplitOperand& o)
{
    const float v[8] = { e.lo[0], e.lo[1], e.lo[2], e.lo[3], e.hi[0], e.hi[1], e.hi[2], e.hi[3] };
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        unsigned h, m, l;
        split_bf16_pair(v[2 * j], v[2 * j + 1], h, m, l);
        o.h[j] = h; o.m[j] = m; o.l[j] = l;
    }
}
__device__ __forceinline__ void operand(const Eight<kIn16>& e, uint4_v& o) { o = e.v; }
__device__ __forceinline__ uint4_v imaginary(uint4_v v)         // (re, im) -> (-im, re)
{
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = __builtin_amdgcn_alignbit(v[j], v[j], 16) ^ 0x00008000u;
    return v;
}
__device__ __forceinline__ SplitOperand imaginary(const SplitOperand& o) { return { imaginary(o.h), imaginary(o.m), imaginary(o.l) }; }
// sums of the lane's values: of the real and of the imaginary parts, or of all
template <bool COMPLEX> __device__ __forceinline__ void add_values(const Eight<kIn32>& e, float& re, float& im)
{
    if constexpr (COMPLEX) {
        re += (e.lo[0] + e.lo[2]) + (e.hi[0] + e.hi[2]);
        im += (e.lo[1] + e.lo[3]) + (e.hi[1] + e.hi[3]);
    } else re += ((e.lo[0] + e.lo[1]) + (e.lo[2] + e.lo[3])) + ((e.hi[0] + e.hi[1]) + (e.hi[2] + e.hi[3]));
}
template <bool COMPLEX> __device__ __forceinline__ void add_values(const Eight<kIn16>& e, float& re, float&)
{
#pragma unroll
    for (int j = 0; j < 4; ++j) re += __builtin_bit_cast(float, e.v[j] << 16) + __builtin_bit_cast(float, e.v[j] & 0xffff0000u);
}
__device__ __forceinline__ void multiply(const SplitOperand& a, const SplitOperand (&b)[4], float4_v (&c)[4])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = mfma_bf16(a.l, b[i].h, c[i]);
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = mfma_bf16(a.h, b[i].l, c[i]);
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = mfma_bf16(a.m, b[i].m, c[i]);
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = mfma_bf16(a.m, b[i].h, c[i]);
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = mfma_bf16(a.h, b[i].m, c[i]);
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = mfma_bf16(a.h, b[i].h, c[i]);
}
__device__ __forceinline__ void multiply(uint4_v a, const uint4_v (&b)[4], float4_v (&c)[4])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = mfma_bf16(a, b[i], c[i]);
}

template <int IN, bool COMPLEX> __global__ __launch_bounds__(256, 1) void weight_grad_kernel(const GradParams q)
{
    constexpr int V = COMPLEX ? 2 : 1, KT = 4 / V;      // tiles of 16 rows k
    typedef typename std::conditional<IN == kIn32, SplitOperand, uint4_v>::type Op;
    typedef typename Columns<IN>::Value Value;
    __shared__ float4_v half[2][16][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, c = lane & 15, kq = lane >> 4;
    // blocks of one part of the positions are eight apart, on one XCD: they read the same rows
    const int full = q.splits / 8 * 8;
    int split, tile;
    if ((int)blockIdx.x < full * q.tiles) {
        const int group = blockIdx.x / (8 * q.tiles), rest = blockIdx.x % (8 * q.tiles);
        tile = rest / 8;
        split = group * 8 + rest % 8;
    } else {
        const int rest = blockIdx.x - full * q.tiles;
        split = full + rest / q.tiles;
        tile = rest % q.tiles;
    }
    const int n0 = tile / q.ktiles * kGradRows, k0 = tile % q.ktiles * (16 * KT);
    const Value* g[4];
    const Value* x[KT];
#pragma unroll
    for (int t = 0; t < 4; ++t) g[t] = static_cast<const Value*>(q.g) + (n0 + 16 * t + c < q.N ? n0 + 16 * t + c : q.N - 1) * q.ldg;
#pragma unroll
    for (int t = 0; t < KT; ++t) x[t] = static_cast<const Value*>(q.x) + (k0 + 16 * t + c < q.K ? k0 + 16 * t + c : q.K - 1) * q.ldx;

    float4_v acc[4][4] = {};
    float bias_re[4] = {}, bias_im[4] = {};
    const long steps = (q.columns + kStep - 1) / kStep, stride = 4l * q.splits;
    Eight<IN> gv[4], xv[KT];
    auto fetch = [&](long s, Eight<IN> (&gv)[4], Eight<IN> (&xv)[KT]) {
        const long column = s * kStep + 8 * kq;
        const bool inside = (s + 1) * kStep <= q.columns;
#pragma unroll
        for (int t = 0; t < 4; ++t) gv[t] = load8<IN>(g[t], column, q.columns, inside);
#pragma unroll
        for (int t = 0; t < KT; ++t) xv[t] = load8<IN>(x[t], column, q.columns, inside);
    };
    const long first = 4l * split + wave;
    if (first < steps) fetch(first, gv, xv);
    for (long s = first; s < steps; s += stride) {
        Eight<IN> gn[4], xn[KT];
        if (s + stride < steps) fetch(s + stride, gn, xn);
        Op b[4];
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            operand(xv[t], b[V * t]);
            if constexpr (COMPLEX) b[V * t + 1] = imaginary(b[V * t]);
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            Op a;
            operand(gv[t], a);
            if (k0 == 0) add_values<COMPLEX>(gv[t], bias_re[t], bias_im[t]);
            multiply(a, b, acc[t]);
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) gv[t] = gn[t];
#pragma unroll
        for (int t = 0; t < KT; ++t) xv[t] = xn[t];
    }

    // the four waves' sums: 2 + 3 to 0 + 1, 1 to 0
    float4_v* bias4 = &half[0][0][0];
#pragma unroll
    for (int from = 2; from >= 1; --from) {
        if (wave >= from && wave < 2 * from)
#pragma unroll
            for (int t = 0; t < 16; ++t) half[wave - from][t][lane] = acc[t / 4][t % 4];
        __syncthreads();
        if (wave < from)
#pragma unroll
            for (int t = 0; t < 16; ++t) acc[t / 4][t % 4] += half[wave][t][lane];
        __syncthreads();
    }
    float* out = q.sums + (long)split * ((long)q.N * q.K + q.N) * V;
    if (wave == 0)
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int u = 0; u < KT; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int n = n0 + 16 * t + 4 * kq + i, k = k0 + 16 * u + c;
                    if (n < q.N && k < q.K) {
                        float* p = out + ((long)n * q.K + k) * V;
                        p[0] = acc[t][V * u][i];
                        if constexpr (COMPLEX) p[1] = acc[t][V * u + 1][i];
                    }
                }
    if (k0 == 0) {
        bias4[2 * threadIdx.x] = (float4_v){ bias_re[0], bias_re[1], bias_re[2], bias_re[3] };
        bias4[2 * threadIdx.x + 1] = (float4_v){ bias_im[0], bias_im[1], bias_im[2], bias_im[3] };
        __syncthreads();
        // thread r: row n0 + r, over four waves and four quarters
        if (threadIdx.x < 64 * V) {
            const int r = threadIdx.x / V, part = threadIdx.x % V;
            float sum = 0.f;
#pragma unroll
            for (int w = 0; w < 16; ++w) sum += reinterpret_cast<const float*>(bias4)[(2 * (16 * w + r % 16) + part) * 4 + r / 16];
            if (n0 + r < q.N) out[(long)q.N * q.K * V + (n0 + r) * V + part] = sum;
        }
    }
}

// Sums over the parts of the positions; a block: 64 results, four quarters of the parts
__global__ __launch_bounds__(256) void add_parts_kernel(const float* __restrict__ sums, int splits, long count, long weights, int type, void* gW, void* gbias)
{
    __shared__ float part[4][64];
    const long e = (long)blockIdx.x * 64 + (threadIdx.x & 63);
    const int quarter = threadIdx.x >> 6;
    float sum = 0.f;
    if (e < count) {
#pragma unroll 16
        for (int s = quarter; s < splits; s += 4) sum += sums[s * count + e];
    }
    part[quarter][threadIdx.x & 63] = sum;
    __syncthreads();
    if (quarter == 0 && e < count) {
        sum = (part[0][threadIdx.x] + part[1][threadIdx.x]) + (part[2][threadIdx.x] + part[3][threadIdx.x]);
        void* to = e < weights ? gW : gbias;
        const long at = e < weights ? e : e - weights;
        if (to) {
            if (type == kBF16) static_cast<__bf16*>(to)[at] = (__bf16)sum;
            else static_cast<float*>(to)[at] = sum;
        }
    }
}

int tiles_of(int type, int N, int K, int& ktiles)
{
    const int kt = type == kC64 ? 32 : 64;
    ktiles = (K + kt - 1) / kt;
    return (N + kGradRows - 1) / kGradRows * ktiles;
}
// Parts of the positions: about two blocks per CU, at least four steps for each wave
int splits_of(int type, long P, int N, int K)
{
    int ktiles;
    const long steps = (P * values_of(type) + kStep - 1) / kStep, tiles = tiles_of(type, N, K, ktiles);
    long splits = (512 + tiles - 1) / tiles;
    if (splits > (steps + 15) / 16) splits = (steps + 15) / 16;
    if (splits > 8) splits = splits / 8 * 8;
    return splits < 1 ? 1 : (int)splits;
}

}  // namespace

size_t mix_weight_grad_workspace(int type, long P, int N, int K)
{
    return (size_t)splits_of(type, P, N, K) * ((size_t)N * K + N) * values_of(type) * sizeof(float);
}

hipError_t launch_mix_weight_grad(int type, long P, int N, int K, const void* gz, long ldgz, const void* x, long ldx, void* gW, void* gbias, void* workspace,
                                  hipStream_t stream)
{
    const int v = values_of(type);
    GradParams q = { gz, x, ldgz * v, ldx * v, P * v, N, K, static_cast<float*>(workspace), splits_of(type, P, N, K), 0, 0 };
    q.tiles = tiles_of(type, N, K, q.ktiles);
    const dim3 grid((unsigned)(q.splits * q.tiles));
    switch (type) {
    case kC64: hipLaunchKernelGGL((weight_grad_kernel<kIn32, true>), grid, dim3(256), 0, stream, q); break;
    case kF32: hipLaunchKernelGGL((weight_grad_kernel<kIn32, false>), grid, dim3(256), 0, stream, q); break;
    default: hipLaunchKernelGGL((weight_grad_kernel<kIn16, false>), grid, dim3(256), 0, stream, q);
    }
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    const long weights = (long)N * K * v, count = weights + (long)N * v;
    hipLaunchKernelGGL(add_parts_kernel, dim3((unsigned)((count + 63) / 64)), dim3(256), 0, stream, q.sums, q.splits, count, weights, type, gW, gbias);
    return hipGetLastError();
}

}  // namespace tfno
