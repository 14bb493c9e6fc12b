// Gradient of the channel product's weights and bias (turbofno_mix_weight_grad):
//
//   gW[n][k] = sum_p gz[n][p] conj(x[k][p]),   gbias[n] = sum_p gz[n][p]
//
// A contraction over positions, which are contiguous in both operands: a lane reads eight consecutive real values of a row of gz and of a row of
// x, the quarters of a wave 32 of them, and has the operands of its matrix instructions. Complex rows are (re, im) pairs: gz as it is against
// (re, im) of x for the real part, against (-im, re) for the imaginary part. 32-bit values are split into bf16 parts (bf16_split.h), 16-bit ones
// are exact; sums are fp32. gbias takes its sums from the values of gz that pass by.
// A block takes a tile of 64 rows n and 64 rows k, so that up to 64 channels are read once, and a part of the positions: its four waves four steps of 32 real values side by
// side, then those as many steps further as all blocks take together. So the blocks move through the rows as one window: with a contiguous part for each
// block they all would stand at the same offset of their parts, on the same few memory channels. The blocks' sums go to the workspace and are added in a second kernel, always in the
// same order: results do not change from call to call.
// An infinite operand, or one above the largest bf16 number (3.3895e38), makes the sums it takes part in infinite or NaN.
#include "columns.h"
#include "kernels.h"

namespace tfno {

namespace {

constexpr int kGradRows = 64, kGradColumns = 64;        // rows n and rows k of a tile
constexpr int kStep = 32, kRun = 16;                    // real values of a step; steps of a run

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

// A lane's eight values of a step: consecutive ones in 16 bits; in 32 bits four and, 16 further, four more, so that the quarters of a wave read 64
// consecutive bytes of a row with one instruction. (Which position a value belongs to does not matter, as long as it is the same in both operands.)
template <int IN> __device__ __forceinline__ Eight<IN> load8(const typename Columns<IN>::Value* p)
{
    Eight<IN> e;
    if constexpr (IN == kIn32) {
        e.lo = *reinterpret_cast<const float4_any*>(p);
        e.hi = *reinterpret_cast<const float4_any*>(p + 16);
    } else e.v = *reinterpret_cast<const uint4_any*>(p);
    return e;
}
// the first `there` of them, zeros for the others
template <int IN> __device__ __forceinline__ Eight<IN> load8_ragged(const typename Columns<IN>::Value* p, int there)
{
    Eight<IN> e;
    auto at = [&](int i) { return i < there ? p[i] : (typename Columns<IN>::Value)0; };
    if constexpr (IN == kIn32) {
        e.lo = (float4_v){ at(0), at(1), at(2), at(3) };
        e.hi = (float4_v){ at(16), at(17), at(18), at(19) };
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
template <int B> __device__ __forceinline__ void multiply(const SplitOperand& a, const SplitOperand (&b)[B], float4_v (&c)[B])
{
#pragma unroll
    for (int i = 0; i < B; ++i) c[i] = mfma_bf16(a.l, b[i].h, c[i]);
#pragma unroll
    for (int i = 0; i < B; ++i) c[i] = mfma_bf16(a.h, b[i].l, c[i]);
#pragma unroll
    for (int i = 0; i < B; ++i) c[i] = mfma_bf16(a.m, b[i].m, c[i]);
#pragma unroll
    for (int i = 0; i < B; ++i) c[i] = mfma_bf16(a.m, b[i].h, c[i]);
#pragma unroll
    for (int i = 0; i < B; ++i) c[i] = mfma_bf16(a.h, b[i].m, c[i]);
#pragma unroll
    for (int i = 0; i < B; ++i) c[i] = mfma_bf16(a.h, b[i].h, c[i]);
}
template <int B> __device__ __forceinline__ void multiply(uint4_v a, const uint4_v (&b)[B], float4_v (&c)[B])
{
#pragma unroll
    for (int i = 0; i < B; ++i) c[i] = mfma_bf16(a, b[i], c[i]);
}

template <int IN, bool COMPLEX> __global__ __launch_bounds__(256, 1) void weight_grad_kernel(const GradParams q)
{
    constexpr int V = COMPLEX ? 2 : 1, KT = kGradColumns / 16;         // tiles of 16 rows k
    constexpr int LANE = IN == kIn32 ? 4 : 8;           // consecutive values of a lane
    typedef typename std::conditional<IN == kIn32, SplitOperand, uint4_v>::type Op;
    typedef typename Columns<IN>::Value Value;
    constexpr int ACC = 4 * KT * V;
    extern __shared__ float4_v totals[];                // [wave][sum][lane]
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
    const int n0 = tile / q.ktiles * kGradRows, k0 = tile % q.ktiles * kGradColumns;
    const Value* g[4];
    const Value* x[KT];
#pragma unroll
    for (int t = 0; t < 4; ++t) g[t] = static_cast<const Value*>(q.g) + (n0 + 16 * t + c < q.N ? n0 + 16 * t + c : q.N - 1) * q.ldg + LANE * kq;
#pragma unroll
    for (int t = 0; t < KT; ++t) x[t] = static_cast<const Value*>(q.x) + (k0 + 16 * t + c < q.K ? k0 + 16 * t + c : q.K - 1) * q.ldx + LANE * kq;

    float4_v acc[4][KT * V] = {};
    float bias_re[4] = {}, bias_im[4] = {};
    struct Rows {
        Eight<IN> g[4], x[KT];
    };
    auto fetch = [&](long step, Rows& r) {
        const long column = step * kStep;
#pragma unroll
        for (int t = 0; t < 4; ++t) r.g[t] = load8<IN>(g[t] + column);
#pragma unroll
        for (int t = 0; t < KT; ++t) r.x[t] = load8<IN>(x[t] + column);
        __builtin_amdgcn_sched_barrier(0);              // the loads stay ahead of the products that follow
    };
    auto product = [&](const Rows& r) {
        Op b[KT * V];
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            operand(r.x[t], b[V * t]);
            if constexpr (COMPLEX) b[V * t + 1] = imaginary(b[V * t]);
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            Op a;
            operand(r.g[t], a);
            add_values<COMPLEX>(r.g[t], bias_re[t], bias_im[t]);
            multiply(a, b, acc[t]);
        }
    };
    // The sums of kRun steps are added to totals in LDS: each of the six instructions of a step rounds the sum that it adds to, and a sum over a wave's whole
    // part would be rounded at its full size each time (2^20 positions, complex: error 3.5e-6 of the gradient)
    float4_v* total = totals + wave * (ACC * 64) + lane;
    int run = 0;
    bool begun = false;
    auto flush = [&] {
#pragma unroll
        for (int t = 0; t < ACC; ++t) {
            total[t * 64] = begun ? total[t * 64] + acc[t / (KT * V)][t % (KT * V)] : acc[t / (KT * V)][t % (KT * V)];
            acc[t / (KT * V)][t % (KT * V)] = float4_v{};
        }
        begun = true;
        run = 0;
    };
    // whole steps, two on their way at a time (after the last one, the last one again: a branch around loads would be waited at); then the rest of the columns
    const long steps = q.columns / kStep, stride = 8l * q.splits, first = 8l * split + 2 * __builtin_amdgcn_readfirstlane(wave);
    if (first < steps) {
        Rows r0, r1;
        auto at = [&](long s) { return s < steps ? s : steps - 1; };
        fetch(first, r0);
        for (long s = first;; s += stride) {
            fetch(at(s + 1), r1);
            product(r0);
            if (s + 1 >= steps) break;
            fetch(at(s + stride), r0);
            product(r1);
            if (++run == kRun / 2) flush();
            if (s + stride >= steps) break;
        }
    }
    if (steps * kStep < q.columns && steps % stride / 2 * 2 == first) {
        Rows r;
        const int rest = (int)(q.columns - steps * kStep) - LANE * kq;
#pragma unroll
        for (int t = 0; t < 4; ++t) r.g[t] = load8_ragged<IN>(g[t] + steps * kStep, rest);
#pragma unroll
        for (int t = 0; t < KT; ++t) r.x[t] = load8_ragged<IN>(x[t] + steps * kStep, rest);
        product(r);
    }

    flush();
    __syncthreads();
    float* out = q.sums + (long)split * ((long)q.N * q.K + q.N) * V;
    for (int e = threadIdx.x; e < ACC * 64; e += 256) {
        const float4_v sum = (totals[e] + totals[ACC * 64 + e]) + (totals[2 * ACC * 64 + e] + totals[3 * ACC * 64 + e]);
        const int l = e % 64, t = e / 64, n = n0 + 16 * (t / (KT * V)) + 4 * (l / 16), k = k0 + 16 * (t % (KT * V) / V) + l % 16;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n + i < q.N && k < q.K) out[((long)(n + i) * q.K + k) * V + t % V] = sum[i];
    }
    __syncthreads();
    float4_v* bias4 = totals;
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

int tiles_of(int N, int K, int& ktiles)
{
    ktiles = (K + kGradColumns - 1) / kGradColumns;
    return (N + kGradRows - 1) / kGradRows * ktiles;
}
// Parts of the positions: as many blocks as run at a time on 256 CUs (one or two on each, by their registers), two steps for each wave at least
int splits_of(int type, long P, int N, int K)
{
    int ktiles;
    const long steps = (P * values_of(type) + kStep - 1) / kStep, tiles = tiles_of(N, K, ktiles);
    long splits = ((type == kC64 ? 256 : 512) + tiles - 1) / tiles;
    if (splits > (steps + 7) / 8) splits = (steps + 7) / 8;
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
    q.tiles = tiles_of(N, K, q.ktiles);
    const dim3 grid((unsigned)(q.splits * q.tiles));
    const size_t lds = (size_t)4 * 4 * (kGradColumns / 16) * v * 1024;
    if (type == kC64) {
        static std::atomic<unsigned long long> served{ 0 };
        if (hipError_t e = allow_dynamic_lds(reinterpret_cast<const void*>(weight_grad_kernel<kIn32, true>), lds, served); e != hipSuccess) return e;
        hipLaunchKernelGGL((weight_grad_kernel<kIn32, true>), grid, dim3(256), lds, stream, q);
    } else if (type == kF32) hipLaunchKernelGGL((weight_grad_kernel<kIn32, false>), grid, dim3(256), lds, stream, q);
    else hipLaunchKernelGGL((weight_grad_kernel<kIn16, false>), grid, dim3(256), lds, stream, q);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    const long weights = (long)N * K * v, count = weights + (long)N * v;
    hipLaunchKernelGGL(add_parts_kernel, dim3((unsigned)((count + 63) / 64)), dim3(256), 0, stream, q.sums, q.splits, count, weights, type, gW, gbias);
    return hipGetLastError();
}

}  // namespace tfno
