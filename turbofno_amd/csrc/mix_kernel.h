// Channel product with bias, residual and activation (turbofno_mix), its 8-bit form and the gradient of its input:
//
//   forward   z[n][p] = sum_k W[n][k] x[k][p] + bias[n] + residual[n][p],   y = act(z)
//   8 bit     the same with x = xscale[p] xq[k][p] and W = wscale[n] Wq[n][k]
//   gradient  gz[n][p] = gy[n][p] act'(z[n][p]),   gx[k][p] = sum_n conj(W[n][k]) gz[n][p]
//
// All three are one product "out[rows][positions] = A[rows][contraction] B[contraction][positions]" whose positions are contiguous in memory
// and whose A is small. A complex row of P positions is a row of 2 P real columns here: everything below counts real columns. A wave takes 64 real columns
// (64 real positions, 32 complex ones) and 16 NT rows, a lane four consecutive columns, 4 c ... 4 c + 3 with c = lane % 16, of the
// input, the residual and the results: each access is 16 lanes x four values of one row, 256 bytes in 32 bits.
// Contraction steps hold 32 real values (32 real channels, 16 complex ones), eight of them in each quarter of the wave, so a lane has, after
// a transposition of its own registers, the operands of four matrix instructions per step and 16 rows:
//   real      four columns, eight channels of each;
//   complex   two positions, four channels (re, im) of each, twice: (re, -im) for the real part of the product and (im, re) for the imaginary
//             part, against the one operand (re, im) of A; conjugated weights take (re, im) and (im, -re).
// The input goes from memory to the matrix cores without passing LDS, and is read once where 16 NT rows are all of them.
// 32-bit operands are split into three bf16 parts each, six products (bf16_split.h); sums that are not finite are formed again in fp32, so that
// infinities and the top of the range behave as in fp32. 16-bit operands are exact on the matrix cores; 8-bit ones are widened to bf16, which holds
// them exactly: the matrix instructions for 8-bit operands keep fewer bits of their sums (off by 3e-5 of the result with 8 channels). Sums are fp32
// throughout, results are rounded once; the gradient's product takes gz as it is returned, in 16 bits rounded to them.
#pragma once
#include "bf16_split.h"
#include "columns.h"

namespace tfno {

enum { kColumns = 64 };                                 // real columns of a wave

struct MixParams {
    const void *x, *zin, *W, *bias, *residual;          // x: the input, or gy; zin: z of the gradient
    const float *xscale, *wscale;
    void *y, *z;                                        // z: the pre-activation, or gz; may be null
    long columns, ldx, ldzin, ldr, ldy, ldz;            // in real values of their tensors
    int rows, contraction, ldw;                         // channels of the result, channels of the input, channels in a row of W
    int act;
};

// ---- activations ----
__device__ __forceinline__ float sigmoid(float v)       // off by at most 2^-22 + |v| 2^-24 of itself
{
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504088896f * v));
}
constexpr float kGelu0 = 1.5957691216057308f, kGelu1 = 0.044715f;     // gelu_tanh(z) = z sigmoid(2 sqrt(2 / pi) (z + 0.044715 z^3))
__device__ __forceinline__ float activate(int act, float z)
{
    if (act == kActGeluTanh) return z * sigmoid(kGelu0 * z * __builtin_fmaf(kGelu1 * z, z, 1.f));
    if (act == kActSilu) return z * sigmoid(z);
    if (act == kActRelu) return z <= 0.f ? 0.f : z;     // a NaN stays
    return z;
}
// gy times the activation's slope at z
__device__ __forceinline__ float through_activation(int act, float gy, float z)
{
    if (act == kActGeluTanh) {
        const float s = sigmoid(kGelu0 * z * __builtin_fmaf(kGelu1 * z, z, 1.f)), t = s * (1.f - s);
        return gy * (t == 0.f ? s : __builtin_fmaf(z * t, kGelu0 * __builtin_fmaf(3.f * kGelu1 * z, z, 1.f), s));       // t = 0: z may be infinite
    }
    if (act == kActSilu) {
        const float s = sigmoid(z), t = s * (1.f - s);
        return gy * (t == 0.f ? s : __builtin_fmaf(z, t, s));
    }
    if (act == kActRelu) return z > 0.f ? gy : 0.f;
    return gy;
}

// ---- operands of the matrix instructions: eight values of the contraction per lane ----
template <int IN> struct Operand;
template <> struct Operand<kIn32> : SplitOperand { };
template <> struct Operand<kIn16> { uint4_v v; };
template <> struct Operand<kIn8> { uint4_v v; };

// halves of two registers: (low half of a, low half of b), (high, high)
__device__ __forceinline__ unsigned low_halves(unsigned a, unsigned b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ __forceinline__ unsigned high_halves(unsigned a, unsigned b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }
// four e4m3 values as bf16, which holds them exactly
__device__ __forceinline__ uint2_v widen(unsigned bytes)
{
    return (uint2_v){ __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)bytes, 1.f, false)),
                      __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)bytes, 1.f, true)) };
}
// a complex operand's two forms from (re, im) pairs; CONJ: for conjugated weights
template <bool CONJ> __device__ __forceinline__ unsigned real_form(unsigned v) { return CONJ ? v : v ^ 0x80000000u; }
template <bool CONJ> __device__ __forceinline__ unsigned imag_form(unsigned v)
{
    v = __builtin_amdgcn_alignbit(v, v, 16);
    return CONJ ? v ^ 0x80000000u : v;
}

// the lane's rows of a step (eight channels of four columns, or four complex channels of two positions) -> operands of the four products
template <int IN, bool COMPLEX, bool CONJ> __device__ __forceinline__ void make_operands(const RawOf<IN> (&raw)[COMPLEX ? 4 : 8], Operand<IN> (&b)[4])
{
    if constexpr (IN == kIn32 && COMPLEX) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                unsigned h, m, l;
                split_bf16_pair(raw[j][2 * t], raw[j][2 * t + 1], h, m, l);
                b[2 * t].h[j] = real_form<CONJ>(h); b[2 * t].m[j] = real_form<CONJ>(m); b[2 * t].l[j] = real_form<CONJ>(l);
                b[2 * t + 1].h[j] = imag_form<CONJ>(h); b[2 * t + 1].m[j] = imag_form<CONJ>(m); b[2 * t + 1].l[j] = imag_form<CONJ>(l);
            }
    } else if constexpr (IN == kIn32) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                unsigned h, m, l;
                split_bf16_pair(raw[2 * j][t], raw[2 * j + 1][t], h, m, l);
                b[t].h[j] = h; b[t].m[j] = m; b[t].l[j] = l;
            }
    } else if constexpr (COMPLEX) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint2_v v = widen(raw[j]);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                b[2 * t].v[j] = real_form<CONJ>(v[t]);
                b[2 * t + 1].v[j] = imag_form<CONJ>(v[t]);
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint2_v even, odd;
            if constexpr (IN == kIn8) { even = widen(raw[2 * j]); odd = widen(raw[2 * j + 1]); }
            else { even = raw[2 * j]; odd = raw[2 * j + 1]; }
#pragma unroll
            for (int t = 0; t < 4; ++t) b[t].v[j] = t & 1 ? high_halves(even[t / 2], odd[t / 2]) : low_halves(even[t / 2], odd[t / 2]);
        }
    }
}

// eight consecutive values of the contraction of one row of A: entries e ... e + 7 of `count` real entries, zeros beyond. The row is row `row` of
// W (forward), or column `row` of W (gradient; its entries are `ld` channels apart).
template <int IN, bool COMPLEX, bool GRAD>
__device__ __forceinline__ void load_weights(const void* W, int row, int rows, int e, int count, int ld, Operand<IN>& a)
{
    constexpr int V = COMPLEX ? 2 : 1;
    typedef typename Columns<IN>::Value Value;
    Value w[8];
    const Value* p = static_cast<const Value*>(W);
    const bool inside = row < rows;
#pragma unroll
    for (int j = 0; j < 8; j += V) {
        const int k = (e + j) / V;                       // channel of the contraction
        const bool there = inside && e + j < count;
        const long at = there ? (GRAD ? (long)k * ld + row : (long)row * ld + k) * V : 0;
#pragma unroll
        for (int i = 0; i < V; ++i) w[j + i] = there ? p[at + i] : (Value)0;
    }
    if constexpr (IN == kIn32) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            unsigned h, m, l;
            split_bf16_pair(w[2 * j], w[2 * j + 1], h, m, l);
            a.h[j] = h; a.m[j] = m; a.l[j] = l;
        }
    } else if constexpr (IN == kIn16) {
#pragma unroll
        for (int j = 0; j < 4; ++j) a.v[j] = w[2 * j] | (unsigned)w[2 * j + 1] << 16;
    } else {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint2_v v = widen(w[4 * j] | (unsigned)w[4 * j + 1] << 8 | (unsigned)w[4 * j + 2] << 16 | (unsigned)w[4 * j + 3] << 24);
            a.v[2 * j] = v[0];
            a.v[2 * j + 1] = v[1];
        }
    }
}

// c[i] += a b[i]: four independent chains
template <int IN> __device__ __forceinline__ void multiply(const Operand<IN>& a, const Operand<IN> (&b)[4], float4_v (&c)[4])
{
    if constexpr (IN == kIn32) {
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
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = mfma_bf16(a.v, b[i].v, c[i]);
    }
}

// One element of the product in fp32, channel by channel: for sums that the split left without a value. `column` is a real column.
template <bool COMPLEX, bool GRAD> __device__ __forceinline__ float product_fp32(const MixParams& q, int row, long column)
{
    const float *W = static_cast<const float*>(q.W), *x = static_cast<const float*>(q.x), *z = static_cast<const float*>(q.zin);
    auto value = [&](int k, long c) {
        const float v = x[k * q.ldx + c];
        if constexpr (GRAD) return q.act == kActNone ? v : through_activation(q.act, v, z[k * q.ldzin + c]);
        else return v;
    };
    float sum = 0.f;
    for (int k = 0; k < q.contraction; ++k) {
        const long w = GRAD ? (long)k * q.ldw + row : (long)row * q.ldw + k;
        if constexpr (COMPLEX) {
            const bool imag = column & 1;
            const float wr = W[2 * w], wi = GRAD ? -W[2 * w + 1] : W[2 * w + 1], xr = value(k, column & ~1L), xi = value(k, column | 1L);
            sum = __builtin_fmaf(wr, imag ? xi : xr, sum);
            sum = __builtin_fmaf(imag ? wi : -wi, imag ? xr : xi, sum);
        } else sum = __builtin_fmaf(W[w], value(k, column), sum);
    }
    return sum;
}

// What a wave does with its columns: the input of a step, and the results
template <int IN, int OUT, bool COMPLEX, bool GRAD, int NT> struct MixWave {
    static constexpr int V = COMPLEX ? 2 : 1, CHANNELS = 32 / V, PER_LANE = 8 / V;      // channels of a step, of a lane
    const MixParams& q;
    int lane, c, kq;
    __device__ __forceinline__ MixWave(const MixParams& params) : q(params), lane(threadIdx.x & 63), c(lane & 15), kq(lane >> 4) { }

    struct Input {
        RawOf<IN> x[PER_LANE];
        RawOf<IN> z[GRAD ? PER_LANE : 1];
    };
    // rows of step `step` at column0 ... column0 + 63
    __device__ __forceinline__ void fetch(long column0, int step, Input& in) const
    {
        const int first = step * CHANNELS + kq * PER_LANE;
        const long column = column0 + 4 * c;
        const auto* x = static_cast<const typename Columns<IN>::Value*>(q.x);
        const auto* z = static_cast<const typename Columns<IN>::Value*>(q.zin);
        const bool slopes = GRAD && q.act != kActNone;
        if ((step + 1) * CHANNELS <= q.contraction && column0 + kColumns <= q.columns) {
#pragma unroll
            for (int j = 0; j < PER_LANE; ++j) in.x[j] = load4<IN>(x + (first + j) * q.ldx, column);
            if constexpr (GRAD) if (slopes)
#pragma unroll
                for (int j = 0; j < PER_LANE; ++j) in.z[j] = load4<IN>(z + (first + j) * q.ldzin, column);
            return;
        }
#pragma unroll
        for (int j = 0; j < PER_LANE; ++j) {
            const bool there = first + j < q.contraction;
            const int k = there ? first + j : q.contraction - 1;
            in.x[j] = load4_ragged<IN>(x + k * q.ldx, column, q.columns);
            if constexpr (GRAD) if (slopes) in.z[j] = load4_ragged<IN>(z + k * q.ldzin, column, q.columns);
            if (!there) {
                in.x[j] = zero4<IN>();
                if constexpr (GRAD) in.z[j] = zero4<IN>();
            }
        }
    }
    // gradient: the input through the activation, written out by one of the waves that share these columns
    __device__ __forceinline__ void slope(long column0, int step, Input& in, bool write) const
    {
        if constexpr (GRAD) {
            if (q.act == kActNone) return;
            const int first = step * CHANNELS + kq * PER_LANE;
            auto* gz = static_cast<typename Columns<IN>::Value*>(q.z);
#pragma unroll
            for (int j = 0; j < PER_LANE; ++j) {
                const float4_v gy = to_float<IN>(in.x[j]), z = to_float<IN>(in.z[j]);
                float4_v g;
#pragma unroll
                for (int i = 0; i < 4; ++i) g[i] = through_activation(q.act, gy[i], z[i]);
                in.x[j] = from_float<IN>(g);
                if (write && first + j < q.contraction) {
                    if (column0 + kColumns <= q.columns) store4<IN>(gz + (first + j) * q.ldz, column0 + 4 * c, in.x[j]);
                    else store4_ragged<IN>(gz + (first + j) * q.ldz, column0 + 4 * c, q.columns, in.x[j]);
                }
            }
        }
    }
    // results of rows row0 + 16 t + 4 kq + i: acc[t][b][i] belongs to column 4 c + b
    __device__ __forceinline__ void finish(long column0, int row0, float4_v (&acc)[NT][4]) const
    {
        const long column = column0 + 4 * c;
        const bool full = column0 + kColumns <= q.columns;
        typedef typename Columns<OUT>::Value Value;
        float4_v xs = { 1.f, 1.f, 1.f, 1.f };
        if constexpr (IN == kIn8) {                     // scales of the lane's columns
#pragma unroll
            for (int b = 0; b < 4; ++b) xs[b] = q.xscale[(column + b < q.columns ? column + b : q.columns - 1) / V];
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = row0 + 16 * t + 4 * kq + i;
                if (row >= q.rows) continue;
                float4_v v = { acc[t][0][i], acc[t][1][i], acc[t][2][i], acc[t][3][i] };
                if constexpr (IN == kIn32) {
                    if (__builtin_expect(not_finite(larger(0.f, v), 0.f), 0))
                        for (int b = 0; b < 4; ++b)
                            if (not_finite(__builtin_fabsf(v[b]), 0.f)) v[b] = product_fp32<COMPLEX, GRAD>(q, row, column + b < q.columns ? column + b : q.columns - 1);
                }
                if constexpr (IN == kIn8) v *= xs * q.wscale[row];
                if constexpr (!GRAD) {
                    if (q.bias) {
                        const Value* bias = static_cast<const Value*>(q.bias) + (long)row * V;
                        const float b0 = value_of(bias[0]), b1 = COMPLEX ? value_of(bias[V - 1]) : b0;
                        v += (float4_v){ b0, b1, b0, b1 };
                    }
                    if (q.residual) {
                        const Value* r = static_cast<const Value*>(q.residual) + row * q.ldr;
                        v += to_float<OUT>(full ? load4<OUT>(r, column) : load4_ragged<OUT>(r, column, q.columns));
                    }
                    if (q.z) write(static_cast<Value*>(q.z) + row * q.ldz, column, full, from_float<OUT>(v));
                    if (q.act != kActNone)
#pragma unroll
                        for (int b = 0; b < 4; ++b) v[b] = activate(q.act, v[b]);
                }
                write(static_cast<Value*>(q.y) + row * q.ldy, column, full, from_float<OUT>(v));
            }
    }
    __device__ __forceinline__ void write(void* row, long column, bool full, RawOf<OUT> v) const
    {
        if (full) store4<OUT>(row, column, v);
        else store4_ragged<OUT>(row, column, q.columns, v);
    }
};

// A wave for 64 columns and 16 NT rows, weights from memory
template <int IN, int OUT, bool COMPLEX, bool GRAD, int NT>
__global__ __launch_bounds__(256, 2) void mix_direct_kernel(const MixParams q, int row_groups)
{
    typedef MixWave<IN, OUT, COMPLEX, GRAD, NT> Wave;
    const Wave w(q);
    const long id = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const long column0 = id / row_groups * kColumns;
    const int row0 = (int)(id % row_groups) * (16 * NT);
    if (column0 >= q.columns) return;
    const int steps = (q.contraction + Wave::CHANNELS - 1) / Wave::CHANNELS;
    float4_v acc[NT][4] = {};
    typename Wave::Input in;
    w.fetch(column0, 0, in);
    for (int s = 0; s < steps; ++s) {
        typename Wave::Input next = in;
        if (s + 1 < steps) w.fetch(column0, s + 1, next);
        w.slope(column0, s, in, row0 == 0);
        Operand<IN> b[4];
        make_operands<IN, COMPLEX, GRAD>(in.x, b);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            Operand<IN> a;
            load_weights<IN, COMPLEX, GRAD>(q.W, row0 + 16 * t + w.c, q.rows, 32 * s + 8 * w.kq, q.contraction * Wave::V, q.ldw, a);
            multiply<IN>(a, b, acc[t]);
        }
        in = next;
    }
    w.finish(column0, row0, acc);
}

}  // namespace tfno
