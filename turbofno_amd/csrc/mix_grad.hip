// Gradient of the channel product's weights and bias (turbofno_mix_weight_grad):
//
//   gW[n][k] = sum_p gz[n][p] conj(x[k][p]),   gbias[n] = sum_p gz[n][p]
//
// A contraction over positions, which are contiguous in both operands: a lane reads eight consecutive real values of a row of gz and of a row of
// x, the quarters of a wave 32 of them, and has the operands of its matrix instructions. Complex rows are (re, im) pairs: gz as it is against
// (re, im) of x for the real part, against (-im, re) for the imaginary part. 32-bit values are split into bf16 parts (bf16_split.h), 16-bit ones
// are exact; sums are fp32. gbias takes its sums from the values of gz that pass by.
// A block takes a tile of 64 rows n and 64 rows k, so that up to 64 channels are read once (or of 32 and 32), and a part of the positions: its four waves two steps of 32
// real values side by side, then those as many steps further as all blocks take together. So the blocks move through the rows as one window: with a contiguous part for each
// block they all would stand at the same offset of their parts, on the same few memory channels. The blocks' sums go to the workspace and are added in a second kernel, always in the
// same order: results do not change from call to call.
// Bound by the issue of one wave per SIMD in complex64, whose sums take half of its 512 registers (64 x 64 channels, 2^20 positions: 275 - 330 us, 3.3 - 3.9 TB/s;
// matrix cores busy 32 % of the time, vector instructions 32 %, waits for memory 5 %), by loads on their way in the others (float32 139 - 154 us, 3.5 - 3.9 TB/s; bf16 75 - 90 us, 3.0 - 3.6 TB/s).
// Sums of a wave with operands that the split does not hold (below 2^-110, above the largest bf16 number 3.3895e38, infinite or NaN) are formed again in fp32. Looking
// for them costs 1 - 2.5 % (complex64, 64 x 64 channels, 2^20 positions: 272.4 us without, 275.7 with; with half of x zeros 269 and 278).
#include "columns.h"
#include "kernels.h"

namespace tfno {

namespace {

constexpr int kStep = 32, kRun = 16;                    // real values of a step; steps of a run

struct GradParams {
    const void *g, *x;
    long ldg, ldx, columns;                             // real values
    int N, K;
    float* sums;                                        // [splits][N K V + N V]
    void *gW, *gbias;                                   // gbias may be null
    int splits, ktiles, tiles;
};

// result `at` of weights and bias, which follow one another
template <bool B16> __device__ __forceinline__ void put_gradient(void* gW, void* gbias, long weights, long at, float sum)
{
    void* to = at < weights ? gW : gbias;
    if (at >= weights) at -= weights;
    if (!to) return;
    if constexpr (B16) static_cast<__bf16*>(to)[at] = (__bf16)sum;
    else static_cast<float*>(to)[at] = sum;
}

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
// which of a lane's values an index is, from the first
template <int IN> constexpr int place(int i) { return IN == kIn32 && i >= 4 ? i + 12 : i; }
// the same from a row that has fewer than a step's: the last one stands for those that there are not
template <int IN> __device__ __forceinline__ Eight<IN> load8_short(const typename Columns<IN>::Value* p, int there)
{
    Eight<IN> e;
    auto at = [&](int i) { return p[place<IN>(i) < there ? place<IN>(i) : there - 1]; };
    if constexpr (IN == kIn32) {
        e.lo = (float4_v){ at(0), at(1), at(2), at(3) };
        e.hi = (float4_v){ at(4), at(5), at(6), at(7) };
    } else
#pragma unroll
        for (int j = 0; j < 4; ++j) e.v[j] = at(2 * j) | (unsigned)at(2 * j + 1) << 16;
    return e;
}
// zeros for the values at places below `from` and from `to` on
template <int IN> __device__ __forceinline__ void keep(Eight<IN>& e, int from, int to)
{
    auto in = [&](int i) { return place<IN>(i) >= from && place<IN>(i) < to; };
    if constexpr (IN == kIn32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            e.lo[i] = in(i) ? e.lo[i] : 0.f;
            e.hi[i] = in(4 + i) ? e.hi[i] : 0.f;
        }
    } else
#pragma unroll
        for (int j = 0; j < 4; ++j) e.v[j] &= (in(2 * j) ? 0xffffu : 0u) | (in(2 * j + 1) ? 0xffff0000u : 0u);
}
// sign: 0, or the sign bit where the operand is negated
__device__ __forceinline__ void operand(const Eight<kIn32>& e, SplitOperand& o, unsigned sign = 0)
{
    auto value = [&](float v) { return __builtin_bit_cast(float, __builtin_bit_cast(unsigned, v) ^ sign); };
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float a = j < 2 ? e.lo[2 * j % 4] : e.hi[2 * j % 4], b = j < 2 ? e.lo[2 * j % 4 + 1] : e.hi[2 * j % 4 + 1];
        unsigned h, m, l;
        split_bf16_pair(value(a), value(b), h, m, l);
        o.h[j] = h; o.m[j] = m; o.l[j] = l;
    }
}
__device__ __forceinline__ void operand(const Eight<kIn16>& e, uint4_v& o, unsigned = 0) { o = e.v; }
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
// acc[t][first + i] += a[t] b[i]: T V sums in turn
template <int T, int V, int ACC> __device__ __forceinline__ void multiply(const SplitOperand (&a)[T], const SplitOperand (&b)[V], float4_v (&c)[T][ACC], int first)
{
    auto part = [&](auto of_a, auto of_b) {
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
            for (int i = 0; i < V; ++i) c[t][first + i] = mfma_bf16(of_a(a[t]), of_b(b[i]), c[t][first + i]);
    };
    auto h = [](const SplitOperand& o) { return o.h; };
    auto m = [](const SplitOperand& o) { return o.m; };
    auto l = [](const SplitOperand& o) { return o.l; };
    part(l, h);
    part(h, l);
    part(m, m);
    part(m, h);
    part(h, m);
    part(h, h);
}
template <int T, int V, int ACC> __device__ __forceinline__ void multiply(const uint4_v (&a)[T], const uint4_v (&b)[V], float4_v (&c)[T][ACC], int first)
{
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
        for (int i = 0; i < V; ++i) c[t][first + i] = mfma_bf16(a[t], b[i], c[t][first + i]);
}

// The same of one row of 16 each with the fp32 matrix instructions, from the values themselves: one position of each quarter of the wave per instruction
template <int V> __device__ __forceinline__ void multiply_fp32(const Eight<kIn32>& g, const Eight<kIn32>& x, float4_v (&c)[V])
{
    auto value = [](const Eight<kIn32>& e, int i) { return i < 4 ? e.lo[i % 4] : e.hi[i % 4]; };
#pragma unroll
    for (int j = 0; j < 8; j += V) {
        c[0] = mfma_fp32(value(g, j), value(x, j), c[0]);
        if constexpr (V == 2) {
            c[1] = mfma_fp32(value(g, j + 1), value(x, j), c[1]);
            c[0] = mfma_fp32(value(g, j + 1), value(x, j + 1), c[0]);
            c[1] = mfma_fp32(-value(g, j), value(x, j + 1), c[1]);
        }
    }
}
template <int T> __device__ __forceinline__ bool rows_below_split_range(const Eight<kIn32> (&g)[T], const Eight<kIn32> (&x)[T])
{
    float4_v v[4 * T];
#pragma unroll
    for (int t = 0; t < T; ++t) {
        v[4 * t] = g[t].lo; v[4 * t + 1] = g[t].hi;
        v[4 * t + 2] = x[t].lo; v[4 * t + 3] = x[t].hi;
    }
    return below_split_range(v);
}

// SHORT: rows of fewer than a step's values
template <int IN, bool COMPLEX, int T, bool SHORT> __global__ __launch_bounds__(256, 1) void weight_grad_kernel(const GradParams q)
{
    constexpr int V = COMPLEX ? 2 : 1;
    constexpr int LANE = IN == kIn32 ? 4 : 8;           // consecutive values of a lane
    typedef typename std::conditional<IN == kIn32, SplitOperand, uint4_v>::type Op;
    typedef typename Columns<IN>::Value Value;
    constexpr int ACC = T * T * V;
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
    const int n0 = tile / q.ktiles * (16 * T), k0 = tile % q.ktiles * (16 * T);
    const Value* g[T];
    const Value* x[T];
#pragma unroll
    for (int t = 0; t < T; ++t) g[t] = static_cast<const Value*>(q.g) + (n0 + 16 * t + c < q.N ? n0 + 16 * t + c : q.N - 1) * q.ldg + LANE * kq;
#pragma unroll
    for (int t = 0; t < T; ++t) x[t] = static_cast<const Value*>(q.x) + (k0 + 16 * t + c < q.K ? k0 + 16 * t + c : q.K - 1) * q.ldx + LANE * kq;

    float4_v acc[T][T * V] = {};
    float bias_re[T] = {}, bias_im[T] = {};
    struct Rows {
        Eight<IN> g[T], x[T];
    };
    auto fetch = [&](long column, Rows& r) {
#pragma unroll
        for (int t = 0; t < T; ++t) r.g[t] = load8<IN>(g[t] + column);
#pragma unroll
        for (int t = 0; t < T; ++t) r.x[t] = load8<IN>(x[t] + column);
        __builtin_amdgcn_sched_barrier(0);              // the loads stay ahead of the products that follow
    };
    // operands of gz together, of x one row of 16 after another: all of both would not fit into the registers beside the sums and the rows on their way
    // (complex64, 64 to 64 channels, 2^20 positions: 408 -> 330 us)
    // What a matrix instruction drops from a sum that it returns has one sign whatever the sum's own, and adds up over many steps. Every other wave forms the negative of
    // its sums, so that it cancels: error of the gradient 3.7e-7, 1.7e-6 without (complex64, 2^20 positions), 4.1e-7 and 4.8e-6 (float32, 2^24), 4.4e-7 and 1.35e-5 (2^27)
    const unsigned sign = IN == kIn32 && (__builtin_amdgcn_readfirstlane(wave) & 1) ? 0x80000000u : 0u;
    bool lost = false;                                  // a value was below the range of the split
    auto product = [&](const Rows& r) {
        if constexpr (IN == kIn32) lost |= rows_below_split_range(r.g, r.x);
        Op a[T];
#pragma unroll
        for (int t = 0; t < T; ++t) {
            operand(r.g[t], a[t]);
            add_values<COMPLEX>(r.g[t], bias_re[t], bias_im[t]);
        }
#pragma unroll
        for (int t = 0; t < T; ++t) {
            Op b[V];
            operand(r.x[t], b[0], sign);
            if constexpr (COMPLEX) b[1] = imaginary(b[0]);
            multiply(a, b, acc, V * t);
        }
    };
    // The sums of kRun steps are added to totals in LDS: each of the six instructions of a step rounds the sum that it adds to, and a sum over a wave's whole
    // part would be rounded at its full size each time (complex, 2^20 and 2^23 positions: error 7.0e-7 and 1.9e-6 of the gradient, 3.7e-7 and 3.9e-7 with runs)
    float4_v* total = totals + wave * (ACC * 64) + lane;
    int run = 0;
    bool begun = false;
    auto flush = [&] {
#pragma unroll
        for (int t = 0; t < ACC; ++t) {
            total[t * 64] = begun ? total[t * 64] + acc[t / (T * V)][t % (T * V)] : acc[t / (T * V)][t % (T * V)];
            acc[t / (T * V)][t % (T * V)] = float4_v{};
        }
        begun = true;
        run = 0;
    };
    // whole steps, two on their way at a time (after the last one, the last one again: a branch around loads would be waited at)
    const long steps = q.columns / kStep, stride = 8l * q.splits, first = 8l * split + 2 * __builtin_amdgcn_readfirstlane(wave);
    if (!SHORT && first < steps) {
        Rows r0, r1;
        auto at = [&](long s) { return (s < steps ? s : steps - 1) * kStep; };
        fetch(at(first), r0);
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
    // the rest of the columns: a step that ends with them, less what the one before it has had
    const int rest = (int)(q.columns - steps * kStep);
    const bool takes_rest = rest && steps % stride / 2 * 2 == first;
    if (takes_rest) {
        Rows r;
        if constexpr (SHORT) {
            const int there = rest > LANE * kq ? rest - LANE * kq : 1, back = rest > LANE * kq ? 0 : LANE * kq;
#pragma unroll
            for (int t = 0; t < T; ++t) r.g[t] = load8_short<IN>(g[t] - back, there);
#pragma unroll
            for (int t = 0; t < T; ++t) r.x[t] = load8_short<IN>(x[t] - back, there);
        } else fetch(q.columns - kStep, r);
        const int from = SHORT ? 0 : kStep - rest - LANE * kq, to = SHORT ? rest - LANE * kq : (int)kStep;
#pragma unroll
        for (int t = 0; t < T; ++t) keep<IN>(r.g[t], from, to);
#pragma unroll
        for (int t = 0; t < T; ++t) keep<IN>(r.x[t], from, to);
        product(r);
    }

    flush();
    // Infinities and the top of the range leave the split without a value, small numbers lose their low parts there: then all sums of the wave again, in fp32, those
    // of 16 x 16 channels after those of others, which takes no registers from the loop above
    if constexpr (IN == kIn32) {
        float high = 0.f;
        asm volatile("" ::: "memory");                  // read again: kept in registers, the totals would spill those of the loop
#pragma unroll 8
        for (int t = 0; t < ACC; ++t) high = larger(high, total[t * 64]);
        if (__builtin_expect(lost || any_lane(not_finite(high, 0.f)), 0))
#pragma unroll 1
            for (int pair = 0; pair < T * T; ++pair) {
                const int n = n0 + 16 * (pair / T) + c, k = k0 + 16 * (pair % T) + c;
                const Value* gn = static_cast<const Value*>(q.g) + (n < q.N ? n : q.N - 1) * q.ldg;
                const Value* xk = static_cast<const Value*>(q.x) + (k < q.K ? k : q.K - 1) * q.ldx;
                float4_v part[V] = {}, sum[V] = {};
                auto add = [&] {
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        sum[i] += part[i];
                        part[i] = float4_v{};
                    }
                };
                int n_steps = 0;
#pragma unroll 1
                for (long s = first; s < steps; s = s % 2 ? s - 1 + stride : s + 1) {
                    multiply_fp32(load8<IN>(gn + s * kStep + LANE * kq), load8<IN>(xk + s * kStep + LANE * kq), part);
                    if (++n_steps % kRun == 0) add();
                }
                if (takes_rest) {                       // value by value: those that the lane has of the last columns
                    auto last = [&](const Value* row) {
                        auto at = [&](int i) {
                            const long column = steps * kStep + LANE * kq + place<IN>(i);
                            return column < q.columns ? row[column] : 0.f;
                        };
                        return Eight<IN>{ { at(0), at(1), at(2), at(3) }, { at(4), at(5), at(6), at(7) } };
                    };
                    multiply_fp32(last(gn), last(xk), part);
                }
                add();
#pragma unroll
                for (int i = 0; i < V; ++i) total[(pair * V + i) * 64] = sign ? -sum[i] : sum[i];
            }
    }
    __syncthreads();
    // to the workspace; the sums of all positions to the results
    const long weights = (long)q.N * q.K * V;
    float* out = q.sums + split * (weights + q.N * V);
    auto put = [&](long at, float sum) {
        if (T == 2 && q.splits == 1) put_gradient<IN == kIn16>(q.gW, q.gbias, weights, at, sum);
        else out[at] = sum;
    };
    for (int e = threadIdx.x; e < ACC * 64; e += 256) {
        const float4_v w0 = totals[e], w1 = totals[ACC * 64 + e], w2 = totals[2 * ACC * 64 + e], w3 = totals[3 * ACC * 64 + e];
        const float4_v sum = IN == kIn32 ? (w0 - w1) + (w2 - w3) : (w0 + w1) + (w2 + w3);
        const int l = e % 64, t = e / 64, n = n0 + 16 * (t / (T * V)) + 4 * (l / 16), k = k0 + 16 * (t % (T * V) / V) + l % 16;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n + i < q.N && k < q.K) put(((long)(n + i) * q.K + k) * V + t % V, sum[i]);
    }
    if (k0) return;
    __syncthreads();
    float* bias = reinterpret_cast<float*>(totals);     // [part][t][thread]
#pragma unroll
    for (int t = 0; t < T; ++t) {
        bias[t * 256 + threadIdx.x] = bias_re[t];
        if constexpr (COMPLEX) bias[(T + t) * 256 + threadIdx.x] = bias_im[t];
    }
    __syncthreads();
    // thread r: row n0 + r, over four waves and four quarters
    if (threadIdx.x < 16 * T * V) {
        const int r = threadIdx.x / V, part = threadIdx.x % V;
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < 16; ++w) sum += bias[(T * part + r / 16) * 256 + 16 * w + r % 16];
        if (n0 + r < q.N) put(weights + (n0 + r) * V + part, sum);
    }
}

// Sums over the parts of the positions; a block: 64 results, four quarters of the parts
__global__ __launch_bounds__(256) void add_parts_kernel(const float* __restrict__ sums, int splits, long count, long weights, int type, void* gW, void* gbias)
{
    __shared__ float part[4][64];
    const long e = block_index() * 64 + (threadIdx.x & 63);
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
        if (type == kBF16) put_gradient<true>(gW, gbias, weights, e, sum);
        else put_gradient<false>(gW, gbias, weights, e, sum);
    }
}

// Up to this many steps of tiles of 32 x 32 such tiles are taken: a step of theirs is a quarter of the work, and the loads, of which there are twice as many,
// come from the caches. Both gradients, complex64, gelu, 64 to 64 channels: 24.1 us at 200 positions with 64 x 64, 16.9 with 32 x 32; 50.0 and 36.6
// at 30001; at 2^20, in HBM, 726 and 772 (bf16 206 and 250). Up to 32 x 32 channels there is one tile of either: 2^18 positions of 16 to 16 channels 94 and 61.
constexpr long kSmallWork = 16384;
// Tiles of a product: 16 t rows in both directions
struct Tiling {
    int t, ktiles, tiles, splits;
};
Tiling tiling_of(int type, long P, int N, int K)
{
    Tiling g;
    const long steps = (P * values_of(type) + kStep - 1) / kStep, small = (long)((N + 31) / 32) * ((K + 31) / 32);
    g.t = small == 1 || small * steps <= kSmallWork ? 2 : 4;
    g.ktiles = (K + 16 * g.t - 1) / (16 * g.t);
    g.tiles = (N + 16 * g.t - 1) / (16 * g.t) * g.ktiles;
    // Parts of the positions: as many blocks as run at a time on 256 CUs (one or two on each, by their registers), two steps for each wave at least;
    // one part, without a second kernel, where each wave has up to four steps
    long splits = ((type == kC64 && g.t == 4 ? 256 : 512) + g.tiles - 1) / g.tiles;
    if (splits > (steps + 7) / 8) splits = (steps + 7) / 8;
    if (splits > 8) splits = splits / 8 * 8;
    g.splits = splits < 1 || (g.t == 2 && steps <= 16) ? 1 : (int)splits;
    return g;
}
template <int IN, bool COMPLEX, int T> hipError_t launch_parts(const GradParams& q, hipStream_t stream)
{
    const bool few = q.columns < kStep;
    const size_t lds = (size_t)4 * T * T * (COMPLEX ? 2 : 1) * 1024;
    const auto kernel = few ? weight_grad_kernel<IN, COMPLEX, T, true> : weight_grad_kernel<IN, COMPLEX, T, false>;
    static std::atomic<unsigned long long> served[2];
    if (lds > (64 << 10))
        if (hipError_t e = allow_dynamic_lds(reinterpret_cast<const void*>(kernel), lds, served[few]); e != hipSuccess) return e;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(q.splits * q.tiles)), dim3(256), lds, stream, q);
    return hipGetLastError();
}
template <int IN, bool COMPLEX> hipError_t launch_tiles(int t, const GradParams& q, hipStream_t stream)
{
    return t == 2 ? launch_parts<IN, COMPLEX, 2>(q, stream) : launch_parts<IN, COMPLEX, 4>(q, stream);
}

}  // namespace

size_t mix_weight_grad_workspace(int type, long P, int N, int K)
{
    return (size_t)tiling_of(type, P, N, K).splits * ((size_t)N * K + N) * values_of(type) * sizeof(float);
}

hipError_t launch_mix_weight_grad(int type, long P, int N, int K, const void* gz, long ldgz, const void* x, long ldx, void* gW, void* gbias, void* workspace,
                                  hipStream_t stream)
{
    const int v = values_of(type);
    const Tiling g = tiling_of(type, P, N, K);
    const GradParams q = { gz, x, ldgz * v, ldx * v, P * v, N, K, static_cast<float*>(workspace), gW, gbias, g.splits, g.ktiles, g.tiles };
    const hipError_t e = type == kC64 ? launch_tiles<kIn32, true>(g.t, q, stream) : type == kF32 ? launch_tiles<kIn32, false>(g.t, q, stream) : launch_tiles<kIn16, false>(g.t, q, stream);
    if (e != hipSuccess || (g.t == 2 && g.splits == 1)) return e;
    const long weights = (long)N * K * v, count = weights + (long)N * v;
    hipLaunchKernelGGL(add_parts_kernel, grid_of((count + 63) / 64), dim3(256), 0, stream, q.sums, q.splits, count, weights, type, gW, gbias);
    return hipGetLastError();
}

}  // namespace tfno
