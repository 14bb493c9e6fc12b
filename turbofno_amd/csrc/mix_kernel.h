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
// 32-bit operands are split into three bf16 parts each, six products (bf16_split.h); sums that are not finite, and all sums of a wave that met operands below
// the range of the split, are formed again in fp32, so that the whole range of floats behaves as in fp32 (complex64, 64 to 64 channels at 2^20 positions, all of
// them around 1e-35: 756 us, 224 with ordinary ones). Looking for small operands costs 0.1 - 1 % where memory bounds the product (64 to 64 channels with residual, z and
// gelu: 410.4 us without, 411.7 with), 1.5 - 4 % where the matrix cores do (256 to 256 at 65536: 223 and 231), 5 - 17 % in the direct kernel with 64 rows.
// 16-bit operands are exact on the matrix cores; 8-bit ones are widened to bf16, which holds
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
    int scale_rows = 0;                                 // rows of a wscale: 2^scale_rows
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

// Eight consecutive values of the contraction of one row of A: entries e ... e + 7 of `count` real entries. The row is row `row` of W (forward), or
// column `row` of W (gradient; its entries are `ld` channels apart). First the loads, without a branch: entries that there are not are read from some
// other place in W, of 8 values at least (FEW: of fewer), rows beyond the last from the last one.
template <int IN> struct RawWeights {
    typename Columns<IN>::Value w[8];
};
template <int IN, bool COMPLEX, bool GRAD, bool FEW>
__device__ __forceinline__ void fetch_weights(const void* W, int row, int rows, int e, int count, int ld, RawWeights<IN>& r)
{
    constexpr int V = COMPLEX ? 2 : 1;
    const auto* p = static_cast<const typename Columns<IN>::Value*>(W);
    row = row < rows ? row : rows - 1;
    if constexpr (GRAD || FEW) {
#pragma unroll
        for (int j = 0; j < 8; j += V) {
            const int k = e + j < count ? (e + j) / V : count / V - 1;     // channel of the contraction
#pragma unroll
            for (int i = 0; i < V; ++i) r.w[j + i] = p[(GRAD ? (long)k * ld + row : (long)row * ld + k) * V + i];
        }
    } else {
        const long at = (long)row * ld * V + e, last = (long)(rows - 1) * ld * V + count - 8;
        p += at < last ? at : last;
        if constexpr (IN == kIn8) {
            const RawOf<kIn16> raw = *reinterpret_cast<const uint2_bytes*>(p);
            __builtin_memcpy(r.w, &raw, 8);
        } else {
            const RawOf<IN> lo = load4<IN>(p, 0), hi = load4<IN>(p, 4);
            __builtin_memcpy(r.w, &lo, sizeof lo);
            __builtin_memcpy(r.w + 4, &hi, sizeof hi);
        }
    }
}
// then the operand that they make, with zeros for entries that there are not
template <int IN, bool COMPLEX, bool GRAD, bool FEW>
__device__ __forceinline__ void form_weights(RawWeights<IN> r, int row, int rows, int e, int count, int ld, Operand<IN>& a)
{
    constexpr int V = COMPLEX ? 2 : 1;
    if (e + 8 > count) {
        if constexpr (!GRAD && !FEW) {                 // entries that were read from before their place
            const long at = (long)(row < rows ? row : rows - 1) * ld * V + e, last = (long)(rows - 1) * ld * V + count - 8;
            const int by = at <= last ? 0 : at - last < 8 ? (int)(at - last) : 7;
#pragma unroll
            for (int bit = 1; bit < 8; bit *= 2)
#pragma unroll
                for (int j = 0; j < 8 - bit; ++j) r.w[j] = by & bit ? r.w[j + bit] : r.w[j];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) r.w[j] = e + j < count ? r.w[j] : 0;
    }
    if constexpr (IN == kIn32) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            unsigned h, m, l;
            split_bf16_pair(r.w[2 * j], r.w[2 * j + 1], h, m, l);
            a.h[j] = h; a.m[j] = m; a.l[j] = l;
        }
    } else if constexpr (IN == kIn16) {
#pragma unroll
        for (int j = 0; j < 4; ++j) a.v[j] = r.w[2 * j] | (unsigned)r.w[2 * j + 1] << 16;
    } else {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint2_v v = widen(r.w[4 * j] | (unsigned)r.w[4 * j + 1] << 8 | (unsigned)r.w[4 * j + 2] << 16 | (unsigned)r.w[4 * j + 3] << 24);
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

// of weights that were fetched (those of other entries among them: at worst a product in fp32 that need not be)
__device__ __forceinline__ bool below_split_range(const RawWeights<kIn32>& r)
{
    const float4_v v[2] = { { r.w[0], r.w[1], r.w[2], r.w[3] }, { r.w[4], r.w[5], r.w[6], r.w[7] } };
    return below_split_range(v);
}

// Columns of a wave: column0 ... column0 + 63, of which `there` exist
struct Window {
    long column0;
    int there;
};

// What a wave does with its columns: the input of a step, and the results. An address is a uniform part, 64 bits in scalar registers, and the lane's
// part; FAR: the lane's part may take more than 32 bits (the direct kernel), RAGGED: and columns beyond the last may be asked for.
template <int IN, int OUT, bool COMPLEX, bool GRAD, int NT, bool FAR, bool RAGGED> struct MixWave {
    static constexpr int V = COMPLEX ? 2 : 1, CHANNELS = 32 / V, PER_LANE = 8 / V;      // channels of a step, of a lane
    typedef RawOf<IN> Rows[PER_LANE];                   // a lane's part of a step
    typedef typename Columns<OUT>::Value OutValue;
    const MixParams& q;
    int lane, c, kq;
    __device__ __forceinline__ MixWave(const MixParams& params) : q(params), lane(threadIdx.x & 63), c(lane & 15), kq(lane >> 4) { }

    // four columns of row `row` (uniform) + lane_row of a field of `rows`; of row `row`, or the last one, where there is none (GUARD)
    template <int TYPE, bool GUARD> __device__ __forceinline__ RawOf<TYPE> read(const void* base, long ld, int row, int lane_row, int rows, const Window& w) const
    {
        typedef typename Columns<TYPE>::Value Value;
        const bool there = !GUARD || row + lane_row < rows;
        if (GUARD) row = row < rows ? row : rows - 1;
        const long at = row * ld + w.column0;
        if constexpr (FAR) {
            const Value* p = static_cast<const Value*>(base) + at + (there ? lane_row * ld : 0);
            return RAGGED ? load4_ragged<TYPE>(p, 4 * c, w.there) : load4<TYPE>(p, 4 * c);
        } else {
            unsigned offset = fresh(((unsigned)lane_row * (unsigned)ld + 4 * c) * (unsigned)sizeof(Value));
            if (GUARD) offset = there ? offset : 4 * c * (unsigned)sizeof(Value);
            return near_load4<TYPE>(scalar(base, at * (long)sizeof(Value)), offset);
        }
    }
    template <int TYPE> __device__ __forceinline__ void write(void* base, long ld, int row, int lane_row, const Window& w, RawOf<TYPE> v) const
    {
        typedef typename Columns<TYPE>::Value Value;
        const long at = row * ld + w.column0;
        if constexpr (FAR) {
            Value* p = static_cast<Value*>(base) + at + lane_row * ld;
            if constexpr (RAGGED) store4_ragged<TYPE>(p, 4 * c, w.there, v);
            else store4<TYPE>(p, 4 * c, v);
        } else near_store4<TYPE>(scalar(base, at * (long)sizeof(Value)), fresh(((unsigned)lane_row * (unsigned)ld + 4 * c) * (unsigned)sizeof(Value)), v);
    }
    // the lane's rows of step `step` of `base`. GUARD: channels beyond the last may be among them; then some other row is read, and clear() has to follow.
    // No branch: a load whose result meets another one where branches join is waited for there
    template <bool GUARD> __device__ __forceinline__ void fetch(const void* base, long ld, const Window& w, int step, Rows& rows) const
    {
#pragma unroll
        for (int j = 0; j < PER_LANE; ++j) rows[j] = read<IN, GUARD>(base, ld, step * CHANNELS + j, kq * PER_LANE, q.contraction, w);
    }
    // channels beyond the last: zeros
    __device__ __forceinline__ void clear(int step, Rows& rows) const
    {
        if ((step + 1) * CHANNELS <= q.contraction) return;
#pragma unroll
        for (int j = 0; j < PER_LANE; ++j)
            if (step * CHANNELS + j + kq * PER_LANE >= q.contraction) rows[j] = zero4<IN>();
    }
    // gradient: gy through the activation at z, written out by one of the waves that share these columns
    __device__ __forceinline__ void slope(const Window& w, int step, Rows& x, const Rows& zin, bool writes) const
    {
        if (q.act == kActGeluTanh) slope_of<kActGeluTanh>(w, step, x, zin, writes);
        else if (q.act == kActSilu) slope_of<kActSilu>(w, step, x, zin, writes);
        else slope_of<kActRelu>(w, step, x, zin, writes);
    }
    template <int ACT> __device__ __forceinline__ void slope_of(const Window& w, int step, Rows& x, const Rows& zin, bool writes) const
    {
        const int first = step * CHANNELS, lane_row = kq * PER_LANE;
        const bool whole = first + CHANNELS <= q.contraction;
#pragma unroll
        for (int j = 0; j < PER_LANE; ++j) {
            const float4_v gy = to_float<IN>(x[j]), z = to_float<IN>(zin[j]);
            float4_v g;
#pragma unroll
            for (int i = 0; i < 4; ++i) g[i] = through_activation(ACT, gy[i], z[i]);
            x[j] = from_float<IN>(g);
            if (writes && (whole || first + lane_row + j < q.contraction)) write<IN>(q.z, q.ldz, first + j, lane_row, w, x[j]);
        }
    }
    // Sums that the split left without a value, again in fp32, and all of them where an operand was below the range of the split: four channels
    // per matrix instruction, one in each quarter of the wave, out of memory
    __device__ __forceinline__ void mend(const Window& w, int row0, bool small, float4_v (&acc)[NT][4]) const
    {
        float high = 0.f;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int b = 0; b < 4; ++b) high = larger(high, acc[t][b]);
        if (__builtin_expect(!small && !any_lane(not_finite(high, 0.f)), 1)) return;
        unsigned low = ~0u;                             // small numbers again: a NaN among the values of a lane hides them from a minimum
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int row = row0 + 16 * t + c < q.rows ? row0 + 16 * t + c : q.rows - 1;
            float4_v sum[4] = {};
#pragma unroll 1
            for (int first = 0; first < q.contraction; first += 4) {
                const int k = first + kq < q.contraction ? first + kq : q.contraction - 1;
                float4_v v = here(q.x, q.ldx, k, w);
                if constexpr (GRAD)
                    if (q.act != kActNone) {
                        const float4_v z = here(q.zin, q.ldzin, k, w);
#pragma unroll
                        for (int b = 0; b < 4; ++b) v[b] = through_activation(q.act, v[b], z[b]);
                    }
                const float* at = static_cast<const float*>(q.W) + (GRAD ? (long)k * q.ldw + row : (long)row * q.ldw + k) * V;
                float re = at[0], im = COMPLEX ? (GRAD ? -at[V - 1] : at[V - 1]) : 0.f;
                if (first + kq >= q.contraction) {
                    v = zero4<kIn32>();
                    re = im = 0.f;
                }
                low = lower(lower(lower(low, float2{ v[0], v[1] }), float2{ v[2], v[3] }), float2{ re, im });
#pragma unroll
                for (int b = 0; b < 4; ++b) sum[b] = mfma_fp32(re, v[b], sum[b]);
                if constexpr (COMPLEX)
#pragma unroll
                    for (int b = 0; b < 4; ++b) sum[b] = mfma_fp32(b & 1 ? im : -im, v[b ^ 1], sum[b]);
            }
            small = small || any_lane(low < kSplitLow);
#pragma unroll
            for (int b = 0; b < 4; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[t][b][i] = small || not_finite(__builtin_fabsf(acc[t][b][i]), 0.f) ? sum[b][i] : acc[t][b][i];
        }
    }
    // the lane's four columns of a row
    __device__ __forceinline__ float4_v here(const void* base, long ld, int row, const Window& w) const
    {
        const float* p = static_cast<const float*>(base) + row * ld + w.column0;
        return RAGGED ? load4_ragged<kIn32>(p, 4 * c, w.there) : load4<kIn32>(p, 4 * c);
    }
    // results of rows row0 + 16 t + 4 kq + i: acc[t][b][i] belongs to column 4 c + b
    // small: an operand was below the range of the split
    // bias(t): the bias of the lane's four rows of 16 rows t, real and imaginary parts apart; row_scale(t): their scales, of 8-bit operands
    template <typename Bias, typename Scale>
    __device__ __forceinline__ void finish(const Window& w, int row0, bool small, float4_v (&acc)[NT][4], Bias bias, Scale row_scale) const
    {
        if constexpr (IN == kIn32) mend(w, row0, small, acc);
        RawOf<OUT> residual[GRAD ? 1 : NT][4];          // all loads first
        float4_v xs = { 1.f, 1.f, 1.f, 1.f };
        if constexpr (!GRAD) {
            if (q.residual)
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) residual[t][i] = read<OUT, true>(q.residual, q.ldr, row0 + 16 * t + i, 4 * kq, q.rows, w);
        }
        if constexpr (IN == kIn8)                       // scales of the lane's columns
#pragma unroll
            for (int b = 0; b < 4; ++b) xs[b] = q.xscale[(w.column0 + (!FAR || 4 * c + b < w.there ? 4 * c + b : w.there - 1)) / V];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            if (row0 + 16 * t >= q.rows) break;
            float4_v v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = (float4_v){ acc[t][0][i], acc[t][1][i], acc[t][2][i], acc[t][3][i] };
            if constexpr (IN == kIn8) {
                const float4_v ws = row_scale(t);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = v[i] * ws[i] * xs;       // the product of two small scales may be no normal number where the result is one
            }
            if constexpr (!GRAD) {
                if (q.bias) {
                    const Parts p = bias(t);
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] += (float4_v){ p.v[0][i], p.v[V - 1][i], p.v[0][i], p.v[V - 1][i] };
                }
                if (q.residual)
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] += to_float<OUT>(residual[t][i]);
                if (q.z) put(q.z, q.ldz, row0 + 16 * t, w, v);
                if (q.act == kActGeluTanh) act_rows<kActGeluTanh>(v);
                else if (q.act == kActSilu) act_rows<kActSilu>(v);
                else if (q.act == kActRelu) act_rows<kActRelu>(v);
            }
            put(q.y, q.ldy, row0 + 16 * t, w, v);
        }
    }
    struct Parts {
        float4_v v[V];
    };
    __device__ __forceinline__ Parts bias_of(int first) const       // of rows first ... first + 3; of the last one beyond it
    {
        Parts p;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) p.v[j][i] = value_of(static_cast<const OutValue*>(q.bias)[(long)(first + i < q.rows ? first + i : q.rows - 1) * V + j]);
        return p;
    }
    __device__ __forceinline__ float4_v scale_of(int first) const
    {
        float4_v v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = q.wscale[(first + i < q.rows ? first + i : q.rows - 1) >> q.scale_rows];
        return v;
    }
    template <int ACT> static __device__ __forceinline__ void act_rows(float4_v (&v)[4])
    {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int b = 0; b < 4; ++b) v[i][b] = activate(ACT, v[i][b]);
    }
    // rows first + 4 kq + i
    __device__ __forceinline__ void put(void* base, long ld, int first, const Window& w, const float4_v (&v)[4]) const
    {
        if (first + 16 <= q.rows)
#pragma unroll
            for (int i = 0; i < 4; ++i) write<OUT>(base, ld, first + i, 4 * kq, w, from_float<OUT>(v[i]));
        else
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (first + 4 * kq + i < q.rows) write<OUT>(base, ld, first + i, 4 * kq, w, from_float<OUT>(v[i]));
    }
};

// f(0) ... f(N - 1) with no loop left, so that registers are indexed by constants
template <int N, int I = 0, typename F> __device__ __forceinline__ void unrolled(F&& f)
{
    if constexpr (I < N) {
        f(I);
        unrolled<N, I + 1>(f);
    }
}

// Few columns: a wave for 64 columns and 16 NT rows, weights from memory
template <int IN, int OUT, bool COMPLEX, bool GRAD, bool SLOPES, int NT, bool RAGGED, bool FEW>
__global__ __launch_bounds__(256, 2) void mix_direct_kernel(const MixParams q, int row_groups)
{
    typedef MixWave<IN, OUT, COMPLEX, GRAD, NT, true, RAGGED> Wave;
    const Wave wave(q);
    const long id = block_index() * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long column = id / row_groups * kColumns, left = q.columns - column;
    const int row0 = (int)(id % row_groups) * (16 * NT);
    if (left <= 0) return;
    const Window w = { RAGGED || left >= kColumns ? column : q.columns - kColumns, RAGGED && left < kColumns ? (int)left : (int)kColumns };
    const int steps = (q.contraction + Wave::CHANNELS - 1) / Wave::CHANNELS, count = q.contraction * Wave::V;
    float4_v acc[NT][4] = {};
    bool small = false;
    constexpr bool AHEAD = NT == 1;                     // the weights of a step are asked for with its rows: there are registers for them
    struct Step {
        typename Wave::Rows x, z;
        RawWeights<IN> a[NT];
    } s0, s1;
    auto fetch_a = [&](int s, int t, RawWeights<IN>& a) {
        fetch_weights<IN, COMPLEX, GRAD, FEW>(q.W, row0 + 16 * t + wave.c, q.rows, 32 * s + 8 * wave.kq, count, q.ldw, a);
    };
    auto fetch = [&](int s, Step& r) {
        s = s < steps ? s : steps - 1;
        wave.template fetch<true>(q.x, q.ldx, w, s, r.x);
        if constexpr (SLOPES) wave.template fetch<true>(q.zin, q.ldzin, w, s, r.z);
        if constexpr (AHEAD) fetch_a(s, 0, r.a[0]);
        __builtin_amdgcn_sched_barrier(0);              // the loads stay ahead of the products that follow
    };
    auto product = [&](int s, Step& r) {
        if constexpr (!AHEAD) unrolled<NT>([&](int t) { fetch_a(s, t, r.a[t]); });
        if constexpr (SLOPES) wave.slope(w, s, r.x, r.z, row0 == 0);
        if constexpr (IN == kIn32) small |= below_split_range(r.x);
        wave.clear(s, r.x);
        Operand<IN> b[4];
        make_operands<IN, COMPLEX, GRAD>(r.x, b);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            Operand<IN> a;
            if constexpr (IN == kIn32) small |= below_split_range(r.a[t]);
            form_weights<IN, COMPLEX, GRAD, FEW>(r.a[t], row0 + 16 * t + wave.c, q.rows, 32 * s + 8 * wave.kq, count, q.ldw, a);
            multiply<IN>(a, b, acc[t]);
        }
    };
    fetch(0, s0);
    for (int s = 0; s < steps; s += 2) {
        fetch(s + 1, s1);
        product(s, s0);
        if (s + 1 >= steps) break;
        fetch(s + 2, s0);
        product(s + 1, s1);
    }
    wave.finish(w, row0, small, acc, [&](int t) { return wave.bias_of(row0 + 16 * t + 4 * wave.kq); }, [&](int t) { return wave.scale_of(row0 + 16 * t + 4 * wave.kq); });
}

// gz of the gradient by itself: units of 2048 columns of a row, in turns
template <int IN, int ACT> __device__ __forceinline__ void slope_unit(const MixParams& q, long row, long column0)
{
    typedef typename Columns<IN>::Value Value;
    const Value *gy = static_cast<const Value*>(q.x) + row * q.ldx, *zin = static_cast<const Value*>(q.zin) + row * q.ldzin;
    Value* gz = static_cast<Value*>(q.z) + row * q.ldz;
    auto product = [&](RawOf<IN> g, RawOf<IN> z) {
        const float4_v a = to_float<IN>(g), b = to_float<IN>(z);
        float4_v v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = through_activation(ACT, a[i], b[i]);
        return from_float<IN>(v);
    };
    if (column0 + 2048 <= q.columns) {
        const long column = column0 + 4 * threadIdx.x;
        const RawOf<IN> g0 = load4<IN>(gy, column), g1 = load4<IN>(gy, column + 1024), z0 = load4<IN>(zin, column), z1 = load4<IN>(zin, column + 1024);
        store4<IN>(gz, column, product(g0, z0));
        store4<IN>(gz, column + 1024, product(g1, z1));
    } else
        for (long column = column0 + 4 * threadIdx.x; column < q.columns; column += 1024)
            store4_ragged<IN>(gz, column, q.columns, product(load4_ragged<IN>(gy, column, q.columns), load4_ragged<IN>(zin, column, q.columns)));
}
template <int IN> __global__ __launch_bounds__(256) void slope_kernel(const MixParams q, long units, long of_row)
{
    for (long u = blockIdx.x; u < units; u += gridDim.x) {
        const long row = u / of_row, column0 = (u - row * of_row) * 2048;
        if (q.act == kActGeluTanh) slope_unit<IN, kActGeluTanh>(q, row, column0);
        else if (q.act == kActSilu) slope_unit<IN, kActSilu>(q, row, column0);
        else slope_unit<IN, kActRelu>(q, row, column0);
    }
}

// Many columns: the operands of the block's rows of A stay in LDS, in the order in which lanes read them (16 bytes per lane, part, 16 rows and step), and
// its waves walk the columns without meeting again: no barrier, and 16 NT rows of sums in registers. HELD = 0: steps of the input are read two ahead, again for
// every 16 NT rows (out of the L2 cache), the next rows' or columns' first one during the results. HELD > 0: all steps of the input, HELD or up to `SPARE` fewer,
// stay in registers, in 16 and 8 bits as operands, while the rows are walked.
// Bound by memory up to about 64 channels (complex64, 64 to 64 with residual, z and gelu at 2^20 positions: 404 - 427 us, 5.0 - 5.3 TB/s, the rate of a
// copy); then by the matrix cores, six products for one in 32 bits (complex64, 256 to 256 with residual at 65536: 206 us, 1.0 PFLOP/s of bf16 products), and by the vector
// instructions that form operands and activations (8 bits, 256 to 256 at 262144: 86 us, 3.9 TB/s and 0.40 PFLOP/s).
constexpr int kWaveParts(int in) { return in == kIn32 ? 3 : 1; }
constexpr int kResidentThreads = 512;
// numbers of steps that there are kernels for
constexpr int held_for(int steps) { return steps <= 4 ? steps : steps <= 6 ? 6 : 8; }
template <int IN, int OUT, bool COMPLEX, bool GRAD, bool SLOPES, int NT, int HELD>
__global__ __launch_bounds__(kResidentThreads, 2) void mix_resident_kernel(const MixParams q, int block_rows, int tiles)
{
    extern __shared__ uint4_v weights[];
    typedef MixWave<IN, OUT, COMPLEX, GRAD, NT, false, false> Wave;
    typedef typename Wave::Parts Parts;
    constexpr int PARTS = kWaveParts(IN), SPARE = HELD > 4 ? 2 : 1;     // steps from HELD - SPARE on may reach beyond the last channel
    const Wave wave(q);
    const int row_first = blockIdx.y * block_rows, groups = block_rows / (16 * NT);
    const int steps = HELD ? HELD : (q.contraction + Wave::CHANNELS - 1) / Wave::CHANNELS;
    const bool writes = blockIdx.y == 0;
    // tiles are counted in 32 bits: 64-bit numbers are compared in vector registers. A last tile that is not whole ends with the columns; tiles beyond it are it
    auto window = [&](int tile) { return Window{ scalar(tile < tiles - 1 ? (long)tile * kColumns : q.columns - kColumns), kColumns }; };
    const int stride = gridDim.x * (blockDim.x >> 6);
    int tile = blockIdx.x * (blockDim.x >> 6) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Window w = window(tile);
    auto fetch = [&](const void* base, long ld, const Window& w, int s, typename Wave::Rows& rows) {
        if (s < HELD - SPARE) wave.template fetch<false>(base, ld, w, s, rows);
        else wave.template fetch<true>(base, ld, w, s, rows);
    };
    typename Wave::Rows x[HELD ? HELD : 1], x0, z0;
    auto ahead = [&](const Window& w, int s, typename Wave::Rows& x, typename Wave::Rows& z) {
        wave.template fetch<true>(q.x, q.ldx, w, s, x);
        if constexpr (SLOPES) wave.template fetch<true>(q.zin, q.ldzin, w, s, z);
        __builtin_amdgcn_sched_barrier(0);
    };
    unrolled<HELD>([&](int s) { fetch(q.x, q.ldx, w, s, x[s]); });      // on their way while the operands of A are formed
    if constexpr (HELD == 0) ahead(w, 0, x0, z0);
    unsigned low = ~0u;                                 // of the weights, as lower() counts it
    {
        const int per_step = block_rows / 16 * 64, count = steps * per_step;
#pragma unroll 4
        for (int e = threadIdx.x; e < count; e += blockDim.x) {
            const int s = e / per_step, rest = e % per_step, l = rest % 64, row = row_first + rest / 64 * 16 + (l & 15), entry = 32 * s + 8 * (l >> 4);
            RawWeights<IN> raw;
            Operand<IN> a;
            fetch_weights<IN, COMPLEX, GRAD, false>(q.W, row, q.rows, entry, q.contraction * Wave::V, q.ldw, raw);
            if constexpr (IN == kIn32)
#pragma unroll
                for (int j = 0; j < 8; j += 2) low = lower(low, float2{ raw.w[j], raw.w[j + 1] });
            form_weights<IN, COMPLEX, GRAD, false>(raw, row, q.rows, entry, q.contraction * Wave::V, q.ldw, a);
            uint4_v* to = weights + (long)(e / 64) * (64 * PARTS) + l;
            if constexpr (IN == kIn32) { to[0] = a.h; to[64] = a.m; to[128] = a.l; }
            else to[0] = a.v;
        }
    }
    Parts* biases = reinterpret_cast<Parts*>(weights + (long)steps * block_rows * (4 * PARTS));
    if constexpr (!GRAD)
        if (q.bias)
            for (int e = threadIdx.x; e < block_rows / 4; e += blockDim.x) biases[e] = wave.bias_of(row_first + 4 * e);
    float4_v* scales = reinterpret_cast<float4_v*>(biases + block_rows / 4);
    if constexpr (IN == kIn8)
        for (int e = threadIdx.x; e < block_rows / 4; e += blockDim.x) scales[e] = wave.scale_of(row_first + 4 * e);
    unsigned* lows = reinterpret_cast<unsigned*>(scales);       // 32-bit operands have no scales: a word for each wave
    if constexpr (IN == kIn32) {
        const bool found = any_lane(low < kSplitLow);
        if (wave.lane == 0) lows[threadIdx.x >> 6] = found;
    }
    __syncthreads();
    if (tile >= tiles) return;
    bool small_weights = false;
    if constexpr (IN == kIn32) {
        unsigned any = 0;
        for (unsigned i = 0; i < blockDim.x >> 6; ++i) any |= lows[i];
        small_weights = __builtin_amdgcn_readfirstlane(any);
    }

    auto weight = [&](int s, int t16) {                 // operand of step s, 16 rows t16
        const uint4_v* from = weights + (long)(s * (block_rows / 16) + t16) * (64 * PARTS) + wave.lane;
        Operand<IN> a;
        if constexpr (IN == kIn32) { a.h = from[0]; a.m = from[64]; a.l = from[128]; }
        else a.v = from[0];
        return a;
    };
    auto finish = [&](int g, bool small, float4_v (&acc)[NT][4]) {
        wave.finish(w, row_first + g * (16 * NT), small, acc, [&](int t) { return biases[(g * NT + t) * 4 + wave.kq]; }, [&](int t) { return scales[(g * NT + t) * 4 + wave.kq]; });
    };
    if constexpr (HELD > 0) {
        for (;;) {
            if constexpr (SLOPES) {
                constexpr int AHEAD = IN == kIn32 ? (COMPLEX && HELD > 1 ? 2 : 1) : HELD < 4 ? HELD : 4;      // steps of z on their way
                typename Wave::Rows z[AHEAD];
                unrolled<AHEAD>([&](int s) { fetch(q.zin, q.ldzin, w, s, z[s]); });
                unrolled<HELD>([&](int s) {
                    wave.slope(w, s, x[s], z[s % AHEAD], writes);
                    if (s + AHEAD < HELD) fetch(q.zin, q.ldzin, w, s + AHEAD, z[s % AHEAD]);
                    __builtin_amdgcn_sched_barrier(0);
                });
            }
            const Window wn = window(tile + stride);
            if constexpr (IN != kIn32) {
                // 16- and 8-bit rows: all operands at once, in the registers that the rows leave
                Operand<IN> b[HELD][4];
                unrolled<HELD>([&](int s) {
                    if (s >= HELD - SPARE) wave.clear(s, x[s]);
                    make_operands<IN, COMPLEX, GRAD>(x[s], b[s]);
                });
                for (int g = 0; g < groups; ++g) {
                    float4_v acc[NT][4] = {};
                    unrolled<HELD>([&](int s) {
#pragma unroll
                        for (int t = 0; t < NT; ++t) multiply<IN>(weight(s, g * NT + t), b[s], acc[t]);
                        __builtin_amdgcn_sched_barrier(0);
                    });
                    finish(g, false, acc);
                }
                unrolled<HELD>([&](int s) { fetch(q.x, q.ldx, wn, s, x[s]); });
            } else
                for (int g = 0; g < groups; ++g) {
                    // asked for again as they are used up: for the rows that follow, out of the caches, or for the next columns (after the last tile, the
                    // last one again). Without a branch: loads whose results meet others where branches join are waited for there
                    const Window wf = g < groups - 1 ? w : wn;
                    float4_v acc[NT][4] = {};
                    bool small = small_weights;
                    unrolled<HELD>([&](int s) {
                        small |= below_split_range(x[s]);
                        if (s >= HELD - SPARE) wave.clear(s, x[s]);
                        Operand<IN> b[4];
                        make_operands<IN, COMPLEX, GRAD>(x[s], b);
                        fetch(q.x, q.ldx, wf, s, x[s]);
                        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                        for (int t = 0; t < NT; ++t) multiply<IN>(weight(s, g * NT + t), b, acc[t]);
                        __builtin_amdgcn_sched_barrier(0);
                    });
                    finish(g, small, acc);
                }
            tile += stride;
            if (tile >= tiles) return;
            w = wn;
        }
    } else {
        for (; tile < tiles; tile += stride) {
            const Window wn = window(tile + stride);
            for (int g = 0; g < groups; ++g) {
                const Window wf = g < groups - 1 ? w : wn;
                float4_v acc[NT][4] = {};
                bool small = small_weights;
                auto product = [&](int s, typename Wave::Rows& x, typename Wave::Rows& z) {
                    if constexpr (SLOPES) wave.slope(w, s, x, z, writes && g == 0);
                    if constexpr (IN == kIn32) small |= below_split_range(x);
                    wave.clear(s, x);
                    Operand<IN> b[4];
                    make_operands<IN, COMPLEX, GRAD>(x, b);
#pragma unroll
                    for (int t = 0; t < NT; ++t) multiply<IN>(weight(s, g * NT + t), b, acc[t]);
                };
                typename Wave::Rows x1, z1;
                for (int s = 0; s < steps; s += 2) {
                    ahead(w, s + 1 < steps ? s + 1 : s, x1, z1);
                    product(s, x0, z0);
                    // after the last step the first one of what follows
                    ahead(s + 2 < steps ? w : wf, s + 2 < steps ? s + 2 : 0, x0, z0);
                    if (s + 1 < steps) product(s + 1, x1, z1);
                }
                finish(g, small, acc);
            }
            w = wn;
        }
    }
}

}  // namespace tfno
