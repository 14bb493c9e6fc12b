// Channel product of 8-bit operands with a scale for each block of 128 channels (turbofno_mix_8bit_blocks):
//
//   z[n][p] = sum_b xscale[b][p] wscale[n / 128][b] (sum over the channels k of block b of Wq[n][k] xq[k][p]) + bias[n] + residual[n][p],   y = act(z)
//
// As in the other channel products a complex row of P positions is a row of 2 P real columns, and a wave takes 64 columns. A step holds 128 real values of the contraction,
// one block of channels (complex: half of one). A quarter kq of the wave has the values 16 kq ... 16 kq + 15 of each half of a step, in this order in the operands of both
// sides. The sum of a step is multiplied by both scales and added to the total, in fp32.
//   bf16 result    one matrix instruction takes a step of 16 rows and columns, 128 products of 8-bit operands. It drops what lies more than about 2^-19 below the
//                  largest product: at most 2^-12 of the sum of magnitudes together, 1e-5 of a typical sum (the result's rounding: 2^-9 of it).
//   fp32 result    the operands are widened to bf16, which holds them exactly, and take four matrix instructions whose sums are fp32.
// Kernels, from many columns to few:
//   direct         bf16, whole steps and 16-byte pieces: tiles of 128 or 64 rows and 128 columns, x and W read into LDS past the registers and ahead of time, x taken from
//                  there by transposing reads. 1024 to 1024 channels at 65536 positions with GELU 134 us, 1.02 PFLOP/s; without it 123, of which 26 are the result's stores at
//                  a copy's rate; each further 1024 channels 81 us, 1.7 PFLOP/s (passes among others, two sets of inputs in turns). With 2048 channels waves wait for data
//                  36 % of their time, for their turn to issue 33 %; matrix instructions take 28 % of the cycles, vector instructions, which count those too, 28 %, LDS 19 %;
//                  with 1024 and GELU 35, 28, 20, 36 and 17 %.
//   staged         the same through registers: any strides, ends of steps and fp32 results. 1024 to 1024 at 65536 with W one byte on 120 us where direct takes 110 (inputs
//                  in the caches); float32 181
//   tile           complex: x through registers, whose lanes transpose 4 x 4 bytes; W through LDS. 200 to 136 at 30011 with SiLU and residual 27.4 us, 2.8 TB/s of 77.6 MB:
//                  235 x 3 tiles, less than two rounds
//   split          few columns: the eight waves of a block divide the steps of 64 columns and 16 rows. 2048 to 2048 at 16 positions 6.8 us, of which an empty launch
//                  after launch takes 3; 4096 to 4096 at 64 10.7 us, 16.8 MB of weights
// Direct and staged tiles that are fewer than compute units: two groups of waves with half of the steps each.
// Up to 64 real values of the contraction the kernels of the product with one scale per row are ahead, and take this one's scales.
#include "direct_lds.h"
#include "kernels.h"
#include "mix_blocks_choice.h"
#include "mix_kernel.h"
#include <algorithm>

namespace tfno {

namespace {

typedef int int8_v __attribute__((ext_vector_type(8)));
typedef uint4_v uint4_any __attribute__((aligned(1)));
constexpr int kStep = kBlocksStep;
static_assert(kColumns == 64, "mix_blocks_choice.h counts tiles of 64 columns");

// ---- the input of the tile and split kernels: a lane has four consecutive columns, 4 c ... 4 c + 3 with c = lane % 16, and transposes them ----

template <bool COMPLEX> constexpr int kRowsOfHalf = COMPLEX ? 8 : 16;
template <bool COMPLEX> struct RawStep {
    unsigned row[2][kRowsOfHalf<COMPLEX>];              // four columns of the lane's channels
    float4_v scale;                                     // of the columns
};
// 64 columns of a wave, from column0 on. kWindow: all of them exist, a row's place is a scalar part and the lane's 32 bits. Otherwise `there` of them do, at least one, and a word that
// would end behind the last value of all starts earlier and is shifted (what it holds beyond its row's end is not used): kNarrow by 32-bit offsets from the first value, kFar64
// whatever lies between the channels. For few columns kNarrow is ahead of kWindow also where all 64 exist, by the rows' scalar parts: 4096 to 4096 channels at 64 10.7 us, 14.8
enum { kWindow = 0, kNarrow = 1, kFar64 = 2 };
template <bool COMPLEX, int MODE> struct Input {
    static_assert(COMPLEX || MODE != kWindow, "the tiles of real fields read x their own way");
    static constexpr int V = COMPLEX ? 2 : 1, HALF = kRowsOfHalf<COMPLEX>;
    const MixBlocksParams& q;
    const int c, kq, there;
    const long column0;
    __device__ __forceinline__ Input(const MixBlocksParams& params, long first) : q(params), c(threadIdx.x & 15), kq(threadIdx.x >> 4 & 3),
        there(params.columns - first < kColumns ? (int)(params.columns - first) : (int)kColumns), column0(first) { }
    // GUARD: channels beyond the last are some other one's values, which clear() removes
    template <bool GUARD> __device__ __forceinline__ void fetch(int step, RawStep<COMPLEX>& raw) const
    {
        const int first = step * (kStep / V);
        const unsigned quarter = fresh((unsigned)(kq * HALF) * (unsigned)q.ldx + (MODE == kWindow || 4 * c < there ? 4 * c : 0) + (MODE == kNarrow ? (unsigned)column0 : 0));
        const unsigned end = MODE == kNarrow ? (unsigned)((q.contraction - 1) * q.ldx + q.columns - 4) : 0;     // of the last word
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < HALF; ++j) {
                const int k = first + h * 4 * HALF + j;         // the first quarter's
                if constexpr (MODE == kFar64) {
                    const long row = k + kq * HALF < q.contraction ? k + kq * HALF : q.contraction - 1;
                    const long at = row * q.ldx + column0 + (4 * c < there ? 4 * c : 0), last = (q.contraction - 1) * q.ldx + q.columns - 4;
                    raw.row[h][j] = *reinterpret_cast<const uint_any*>(static_cast<const unsigned char*>(q.x) + (at < last ? at : last)) >> (at > last ? 8 * (int)(at - last) : 0);
                } else if constexpr (MODE == kNarrow) {
                    const unsigned at = quarter + (unsigned)k * (unsigned)q.ldx, by = at < end ? at : end;      // rows beyond the last: the last word, any shift
                    raw.row[h][j] = near_load4<kIn8>(scalar(q.x, 0), by) >> (8 * (at - by) & 31);
                } else if constexpr (GUARD) {
                    const int common = k < q.contraction ? k : q.contraction - 1;
                    raw.row[h][j] = near_load4<kIn8>(scalar(q.x, common * q.ldx + column0), fresh(k + kq * HALF < q.contraction ? quarter : 4 * c));
                } else raw.row[h][j] = near_load4<kIn8>(scalar(q.x, k * q.ldx + column0), quarter);
            }
        const long scales = step / V * q.positions;
        if constexpr (MODE != kWindow)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const long column = column0 + 4 * c + i;
                raw.scale[i] = q.xscale[scales + (column >= q.columns ? q.columns - 1 : column) / V];
            }
        else {
            const uint2_v v = near_load4<kIn16>(scalar(q.xscale, (scales + column0 / 2) * 4), fresh(8 * c));        // two floats, any multiple of 4 bytes
            const float2_v f = __builtin_bit_cast(float2_v, v);
            raw.scale = (float4_v){ f[0], f[0], f[1], f[1] };
        }
    }
    __device__ __forceinline__ void clear(int step, RawStep<COMPLEX>& raw) const
    {
        const int first = step * (kStep / V);
        if (first + kStep / V <= q.contraction) return;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < HALF; ++j)
                if (first + (h * 4 + kq) * HALF + j >= q.contraction) raw.row[h][j] = 0;
    }
};

// four bytes of four rows -> of four columns
__device__ __forceinline__ void transpose4(const unsigned* rows, unsigned (&columns)[4])
{
    const unsigned a = __builtin_amdgcn_perm(rows[1], rows[0], 0x05010400u), b = __builtin_amdgcn_perm(rows[1], rows[0], 0x07030602u),
                   c = __builtin_amdgcn_perm(rows[3], rows[2], 0x05010400u), d = __builtin_amdgcn_perm(rows[3], rows[2], 0x07030602u);
    columns[0] = low_halves(a, c);
    columns[1] = high_halves(a, c);
    columns[2] = low_halves(b, d);
    columns[3] = high_halves(b, d);
}

// Operands of a step: of the lane's four columns, and of 16 rows of W
template <bool COMPLEX, bool EXACT> struct Operands;
template <> struct Operands<false, false> {
    int8_v b[4];
    __device__ __forceinline__ void make(const RawStep<false>& raw)
    {
#pragma unroll
        for (int g = 0; g < 8; ++g) {
            unsigned v[4];
            transpose4(&raw.row[g / 4][4 * (g % 4)], v);
#pragma unroll
            for (int i = 0; i < 4; ++i) b[i][g] = (int)v[i];
        }
    }
    // with columns first ... first + COUNT - 1 of the four
    template <int COUNT> __device__ __forceinline__ void product(const uint4_v (&w)[2], int first, float4_v (&part)[COUNT]) const
    {
        const int8_v a = { (int)w[0][0], (int)w[0][1], (int)w[0][2], (int)w[0][3], (int)w[1][0], (int)w[1][1], (int)w[1][2], (int)w[1][3] };
#pragma unroll
        for (int i = 0; i < COUNT; ++i) part[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b[first + i], (float4_v){ 0.f, 0.f, 0.f, 0.f }, 0, 0, 0, 0, 0, 0);
    }
};
template <bool COMPLEX> struct Operands<COMPLEX, true> {
    Operand<kIn8> b[4][4];
    __device__ __forceinline__ void make(const RawStep<COMPLEX>& raw)
    {
        constexpr int ROWS = COMPLEX ? 4 : 8;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            unsigned rows[ROWS];
#pragma unroll
            for (int j = 0; j < ROWS; ++j) rows[j] = raw.row[u / 2][u % 2 * ROWS + j];
            make_operands<kIn8, COMPLEX, false>(rows, b[u]);
        }
    }
    template <int COUNT> __device__ __forceinline__ void product(const uint4_v (&w)[2], int, float4_v (&part)[COUNT]) const
    {
        static_assert(COUNT == 4, "all columns");
#pragma unroll
        for (int i = 0; i < 4; ++i) part[i] = (float4_v){ 0.f, 0.f, 0.f, 0.f };
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const uint2_v lo = widen(w[u / 2][u % 2 * 2]), hi = widen(w[u / 2][u % 2 * 2 + 1]);
            const Operand<kIn8> a = { { lo[0], lo[1], hi[0], hi[1] } };
            multiply<kIn8>(a, b[u], part);
        }
    }
};

// a scale of the weights, read past the vector unit: one for the wave, and its wait holds up no other load
__device__ __forceinline__ float common_scale(const float* p) { return *reinterpret_cast<const __attribute__((address_space(4))) float*>(scalar(reinterpret_cast<long>(p))); }
// Both scales of a step in one number. `out`: in some lane it is no positive normal number, and the scales may have to be multiplied one after the other, the larger one first
__device__ __forceinline__ float4_v joint_scale(float4_v x, float w, bool& out)
{
    x *= w;
#pragma unroll
    for (int i = 0; i < 4; ++i) out |= !__builtin_amdgcn_classf(x[i], 0x100);
    return x;
}
// Whether they do, in some step of a wave's 64 columns: both are finite and not zero. A scale of zero, infinite or NaN makes of the sum what it would have made alone.
template <bool COMPLEX> __device__ __forceinline__ bool scales_apart(const MixBlocksParams& q, const float* wscale, long column0)
{
    constexpr int kFiniteNotZero = 0x198;
    const long column = column0 + (threadIdx.x & 63), last = q.columns - 1;
    const int blocks = (q.contraction + kScaleBlock - 1) / kScaleBlock;
    bool apart = false;
#pragma unroll 1
    for (int b = 0; b < blocks; ++b) {
        const float x = q.xscale[b * q.positions + (column < last ? column : last) / (COMPLEX ? 2 : 1)], w = wscale[b];
        apart |= __builtin_amdgcn_classf(x, kFiniteNotZero) & __builtin_amdgcn_classf(w, kFiniteNotZero) & !__builtin_amdgcn_classf(x * w, 0x100);
    }
    return any_lane(apart);
}
template <int COUNT> __device__ __forceinline__ void add_scaled(float4_v joint, int first, const float4_v (&part)[COUNT], float4_v (&total)[4])
{
#pragma unroll
    for (int b = 0; b < COUNT; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) total[first + b][i] = __builtin_fmaf(part[b][i], joint[first + b], total[first + b][i]);
}
// total += part x w, the larger scale first
__device__ __forceinline__ void add_scaled_apart(float4_v x, float w, const float4_v (&part)[4], float4_v (&total)[4])
{
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        const float larger = x[b] > w ? x[b] : w, smaller = x[b] > w ? w : x[b];
#pragma unroll
        for (int i = 0; i < 4; ++i) total[b][i] = __builtin_fmaf(part[b][i] * larger, smaller, total[b][i]);
    }
}

// ---- the weights: 16 bytes of a row ----

// Bytes e ... e + 15 of a row of `count`, from memory; where they would end behind the last weight, earlier ones, and mend_weights() has to follow
__device__ __forceinline__ uint4_v fetch_weights(const void* W, int row, int rows, int count, int e)
{
    const unsigned char* w = static_cast<const unsigned char*>(W);
    const long at = (long)(row < rows ? row : rows - 1) * count + e, last = (long)rows * count - 16;
    return *reinterpret_cast<const uint4_any*>(w + (at < last ? at : last));
}
// zeros for bytes from `count` on
__device__ __forceinline__ uint4_v mend_weights(uint4_v v, int row, int rows, int count, int e)
{
    if (e + 16 <= count) return v;
    const long at = (long)(row < rows ? row : rows - 1) * count + e, last = (long)rows * count - 16;
    const int by = at <= last ? 0 : at - last < 16 ? (int)(at - last) : 15;
#pragma unroll
    for (int words = 1; words < 4; words *= 2)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = by & 4 * words ? (i + words < 4 ? v[i + words] : 0u) : v[i];
    const int bits = by % 4 * 8;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (unsigned)(((unsigned long)(i < 3 ? v[i < 3 ? i + 1 : i] : 0u) << 32 | v[i]) >> bits);
    const int left = count - e;                         // bytes that there are
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int n = left - 4 * i;
        v[i] = n >= 4 ? v[i] : n <= 0 ? 0u : v[i] & ((1u << 8 * n) - 1u);
    }
    return v;
}

// ---- results ----

template <int ACT, int ROWS> __device__ __forceinline__ void activate_rows(float4_v (&v)[ROWS])
{
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
#pragma unroll
        for (int b = 0; b < 4; ++b) v[i][b] = activate(ACT, v[i][b]);
}
// Rows row0 + lane_row + i and four columns each, column0 + 4 c ..., of a lane: columns before `from` and beyond the last, and rows beyond the last, are left alone.
// WHOLE: there are none of them in the wave; then an address is a uniform part and one of 32 bits
template <int OUT, bool COMPLEX, int ROWS> struct Results {
    typedef typename Columns<OUT>::Value Value;
    static constexpr int V = COMPLEX ? 2 : 1;
    const MixBlocksParams& q;
    const long column0, from;
    const int c, lane_row;
    __device__ __forceinline__ unsigned offset(long ld) const { return fresh(((unsigned)lane_row * (unsigned)ld + 4 * c) * (unsigned)sizeof(Value)); }
    __device__ __forceinline__ long row_at(int row) const { return row + lane_row < q.rows ? row + lane_row : q.rows - 1; }
    template <bool WHOLE> __device__ __forceinline__ void fetch(int row0, RawOf<OUT> (&residual)[ROWS]) const
    {
        if constexpr (WHOLE) {
            const unsigned at = offset(q.ldr);
#pragma unroll
            for (int i = 0; i < ROWS; ++i) residual[i] = near_load4<OUT>(scalar(q.residual, ((row0 + i) * q.ldr + column0) * (long)sizeof(Value)), at);
        } else
#pragma unroll
            for (int i = 0; i < ROWS; ++i) residual[i] = load4_ragged<OUT>(static_cast<const Value*>(q.residual) + row_at(row0 + i) * q.ldr, column0 + 4 * c, q.columns);
    }
    __device__ __forceinline__ void finish(float4_v (&v)[ROWS], const float* bias, const RawOf<OUT> (&residual)[ROWS]) const
    {
        if (q.bias)
#pragma unroll
            for (int i = 0; i < ROWS; ++i) {
                const float re = bias[i * V], im = bias[i * V + V - 1];
                v[i] += (float4_v){ re, im, re, im };
            }
        if (q.residual)
#pragma unroll
            for (int i = 0; i < ROWS; ++i) v[i] += to_float<OUT>(residual[i]);
        if (q.act == kActGeluTanh) activate_rows<kActGeluTanh>(v);
        else if (q.act == kActSilu) activate_rows<kActSilu>(v);
        else if (q.act == kActRelu) activate_rows<kActRelu>(v);
    }
    template <bool WHOLE> __device__ __forceinline__ void store(int row0, const float4_v (&v)[ROWS]) const
    {
        if constexpr (WHOLE) {
            const unsigned at = offset(q.ldy);
#pragma unroll
            for (int i = 0; i < ROWS; ++i) near_store4<OUT>(scalar(q.y, ((row0 + i) * q.ldy + column0) * (long)sizeof(Value)), at, from_float<OUT>(v[i]));
        } else
#pragma unroll
            for (int i = 0; i < ROWS; ++i) {
                if (row0 + lane_row + i >= q.rows) break;
                Value* p = static_cast<Value*>(q.y) + (row0 + lane_row + i) * q.ldy;
                const RawOf<OUT> raw = from_float<OUT>(v[i]);
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const long column = column0 + 4 * c + b;
                    if (column < from || column >= q.columns) continue;
                    if constexpr (OUT == kIn32) p[column] = raw[b];
                    else p[column] = (unsigned short)(b & 1 ? raw[b / 2] >> 16 : raw[b / 2]);
                }
            }
    }
    __device__ __forceinline__ float bias_at(int row, int part) const { return value_of(static_cast<const Value*>(q.bias)[(long)(row < q.rows ? row : q.rows - 1) * V + part]); }
};
__device__ __forceinline__ float4_v row_of(const float4_v (&total)[4], int i) { return (float4_v){ total[0][i], total[1][i], total[2][i], total[3][i] }; }

// ---- one value of the product, in plain fp32 ----
template <bool COMPLEX> __device__ __forceinline__ float plain_sum(const MixBlocksParams& q, long row, long column)
{
    constexpr int V = COMPLEX ? 2 : 1;
    const int part = (int)(column % V), blocks = (q.contraction + kScaleBlock - 1) / kScaleBlock;
    const unsigned char *W = static_cast<const unsigned char*>(q.W) + row * q.contraction * V, *x = static_cast<const unsigned char*>(q.x) + column - part;
    auto value = [](unsigned char v) { return __builtin_amdgcn_cvt_f32_fp8((int)v, 0); };
    float total = 0.f;
#pragma unroll 1
    for (int b = 0; b < blocks; ++b) {
        float sum = 0.f;
#pragma unroll 1
        for (int k = b * kScaleBlock; k < (b + 1) * kScaleBlock && k < q.contraction; ++k) {
            sum = __builtin_fmaf(value(W[k * V]), value(x[k * q.ldx + part]), sum);
            if constexpr (COMPLEX) sum = __builtin_fmaf(part ? value(W[k * V + 1]) : -value(W[k * V + 1]), value(x[k * q.ldx + 1 - part]), sum);
        }
        const float xs = q.xscale[b * q.positions + column / V], ws = q.wscale[row / kScaleBlock * blocks + b];
        total = __builtin_fmaf(sum * (xs > ws ? xs : ws), xs > ws ? ws : xs, total);
    }
    return total;
}
// the results of a wave whose scales may not be multiplied first: rows row0 + 16 t + i of the lane, value by value
template <int OUT, bool COMPLEX> __device__ __forceinline__ void put_plain(const MixBlocksParams& q, const Results<OUT, COMPLEX, 4>& results, int row0, int tiles16, const float* biases)
{
#pragma unroll 1
    for (int t = 0; t < tiles16 && row0 + 16 * t < q.rows; ++t) {
        float4_v v[4];
        RawOf<OUT> residual[4];
        if (q.residual) results.template fetch<false>(row0 + 16 * t, residual);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const long column = results.column0 + 4 * results.c + b;
                v[i][b] = plain_sum<COMPLEX>(q, results.row_at(row0 + 16 * t + i), column < q.columns ? column : q.columns - 1);
            }
        results.finish(v, biases + (16 * t + results.lane_row) * (COMPLEX ? 2 : 1), residual);
        results.template store<false>(row0 + 16 * t, v);
    }
}

// ---- 16 rows of one wave, steps wave, wave + waves ...: weights straight from memory ----

template <int OUT, bool COMPLEX, int MODE>
__device__ __forceinline__ void sum_steps(const MixBlocksParams& q, const Input<COMPLEX, MODE>& in, int row0, int first, int stride, float4_v (&total)[4])
{
    const int count = q.contraction * (COMPLEX ? 2 : 1), steps = (count + kStep - 1) / kStep;
    const int blocks = (q.contraction + kScaleBlock - 1) / kScaleBlock;
    const float* wscale = q.wscale + (long)(row0 / kScaleBlock) * blocks;
    RawStep<COMPLEX> raw;
    uint4_v w[2];
    auto ask = [&](int s) {
        in.template fetch<true>(s, raw);
#pragma unroll
        for (int h = 0; h < 2; ++h) w[h] = fetch_weights(q.W, row0 + in.c, q.rows, count, s * kStep + 64 * h + 16 * in.kq);
    };
    if (first < steps) ask(first);
    for (int s = first; s < steps; s += stride) {
        in.clear(s, raw);
        if ((s + 1) * kStep > count)
#pragma unroll
            for (int h = 0; h < 2; ++h) w[h] = mend_weights(w[h], row0 + in.c, q.rows, count, s * kStep + 64 * h + 16 * in.kq);
        const float4_v scale = raw.scale;
        const float ws = common_scale(wscale + s / (COMPLEX ? 2 : 1));
        bool out = false;
        const float4_v joint = joint_scale(scale, ws, out);
        Operands<COMPLEX, OUT == kIn32> ops;
        ops.make(raw);
        const uint4_v a[2] = { w[0], w[1] };
        ask(s + stride < steps ? s + stride : s);
        float4_v part[4];
        ops.product(a, 0, part);
        if (any_lane(out)) add_scaled_apart(scale, ws, part, total);
        else add_scaled(joint, 0, part, total);
    }
}

// ---- many columns, complex: four waves side by side share 16 NT rows of W ----

// Blocks go to the eight XCDs in turns (block_order.h). With many columns, tiles side by side go to one: bf16, 512 to 512 channels at 65551 positions 44.8 us (in turns 48.4), 2048 to 2048 at
// 32768 197 (205); not for float32, 512 to 512 at 65536 63.0 (58.7)
// The weights of a step pass LDS, in the order in which lanes read them: 16 bytes per lane, half and 16 rows. Two buffers: a step's are written while those of the
// step before are read, after they were asked for ahead of its products, like the rows of x of the next step. A wave whose 64 columns are not all there takes the last
// 64 and leaves those that it shares with others alone; one that has none goes along for its part of the weights.
template <int NT>
__global__ __launch_bounds__(256, 2) void mix_blocks_tile_kernel(const MixBlocksParams q, int row_tiles, long column_tiles, bool by_xcd)
{
    constexpr int CHUNKS = NT * 128, EACH = CHUNKS / 256;       // 16 bytes each; of a thread
    constexpr int V = 2;
    __shared__ uint4_v weights[2 * CHUNKS];
    __shared__ float biases[16 * NT * V];
    const long id = block_index();
    const Tile tile = tile_of(id, row_tiles, column_tiles, by_xcd, false);
    if (tile.column >= column_tiles) return;
    const int row0 = tile.row * (16 * NT), lane = threadIdx.x & 63;
    const long from = tile.column * (4 * kColumns) + (long)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * kColumns;
    const Input<true, kWindow> in(q, scalar(from + kColumns <= q.columns ? from : q.columns - kColumns));
    const int count = q.contraction * V, steps = (count + kStep - 1) / kStep;
    const float* wscale = q.wscale + (long)(row0 / kScaleBlock) * ((q.contraction + kScaleBlock - 1) / kScaleBlock);
    const int whole = count / kStep;                    // steps of 128 values
    uint4_v w[EACH];
    auto chunk = [&](int i) { return (int)threadIdx.x + 256 * i; };
    auto chunk_row = [&](int e) { return e / 128 * 16 + (e & 15); };
    auto chunk_entry = [&](int e) { return (e >> 6 & 1) * 64 + (e >> 4 & 3) * 16; };
    auto ask = [&](int s, auto guard, uint4_v (&w)[EACH]) {
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int e = chunk(i), row = row0 + chunk_row(e) < q.rows ? chunk_row(e) : q.rows - 1 - row0;
            if constexpr (decltype(guard)::value) w[i] = fetch_weights(q.W, row0 + row, q.rows, count, s * kStep + chunk_entry(e));
            else w[i] = *reinterpret_cast<const TFNO_GLOBAL uint4_any*>(scalar(q.W, (long)row0 * count + s * kStep) + fresh((unsigned)row * (unsigned)count + chunk_entry(e)));
        }
    };
    auto keep = [&](int s, auto guard, uint4_v (&w)[EACH]) {
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int e = chunk(i);
            if constexpr (decltype(guard)::value) w[i] = mend_weights(w[i], row0 + chunk_row(e), q.rows, count, s * kStep + chunk_entry(e));
            weights[(s & 1) * CHUNKS + e] = w[i];
        }
    };
    RawStep<true> raw;
    const Results<kIn32, true, 4> results = { q, in.column0, from, in.c, 4 * in.kq };
    auto begin = [&](auto guard) {
        in.template fetch<decltype(guard)::value>(0, raw);
        ask(0, guard, w);
        if (q.bias)
            for (int e = threadIdx.x; e < 16 * NT * V; e += 256) biases[e] = results.bias_at(row0 + e / V, e % V);
        keep(0, guard, w);
    };
    float4_v total[NT][4] = {};
    bool out = false;
    float weight_scale = common_scale(wscale);
    // step s; NEXT: the one after it is asked for, GUARD: which is the last one and not whole
    auto body = [&](int s, auto next, auto guard) {
        constexpr bool NEXT = decltype(next)::value, GUARD = decltype(guard)::value;
        const float4_v joint = joint_scale(raw.scale, weight_scale, out);
        if constexpr (NEXT) weight_scale = common_scale(wscale + (s + 1) / V);
        Operands<true, true> ops;
        ops.make(raw);
        if constexpr (NEXT) {
            in.template fetch<GUARD>(s + 1, raw);
            ask(s + 1, guard, w);
        }
        __builtin_amdgcn_sched_barrier(0);              // the loads stay ahead of the products
        const uint4_v* from_lds = weights + (s & 1) * CHUNKS + lane;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const uint4_v a[2] = { from_lds[t * 128], from_lds[t * 128 + 64] };
            float4_v part[4];
            ops.product(a, 0, part);
            add_scaled(joint, 0, part, total[t]);
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (NEXT) {
            keep(s + 1, guard, w);
            __syncthreads();
        }
    };
    if (whole) begin(std::false_type());
    else begin(std::true_type());
    __syncthreads();
    for (int s = 0; s < whole - 1; ++s) body(s, std::true_type(), std::false_type());
    if (whole < steps) {
        if (whole) body(whole - 1, std::true_type(), std::true_type());
        in.clear(whole, raw);
    }
    body(steps - 1, std::false_type(), std::false_type());
    if (from >= q.columns) return;
    if (__builtin_expect(any_lane(out), 0) && scales_apart<true>(q, wscale, in.column0)) {
        put_plain<kIn32, true>(q, results, row0, NT, biases);
        return;
    }
    // 32 rows at a time, always from the same registers, which the next rows' sums are moved to: unrolled, the code would not stay in the instruction cache
    auto put = [&](auto whole_wave) {
        constexpr bool WHOLE = decltype(whole_wave)::value;
#pragma unroll 1
        for (int t = 0; t < NT; t += 2) {
            const int row = row0 + 16 * t;
            if (!WHOLE && row >= q.rows) break;
            RawOf<kIn32> residual[2][4];
            if (q.residual)
#pragma unroll
                for (int u = 0; u < 2; ++u) results.template fetch<WHOLE>(row + 16 * u, residual[u]);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                float4_v v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = row_of(total[u], i);
                results.finish(v, biases + (16 * (t + u) + 4 * in.kq) * V, residual[u]);
                results.template store<WHOLE>(row + 16 * u, v);
            }
#pragma unroll
            for (int u = 0; u + 2 < NT; ++u)
#pragma unroll
                for (int b = 0; b < 4; ++b) total[u][b] = total[u + 2][b];
        }
    };
    if (from + kColumns <= q.columns && row0 + 16 * NT <= q.rows) put(std::true_type());
    else put(std::false_type());
}

// ---- many columns, real: waves RG deep and CG side by side share 16 NT RG rows of W and 64 CG columns of x ----

// Both pass LDS in two buffers: a step's values are on their way from memory, 16 bytes a load, during the products of the step before, and written when those are done.
// W lies there in the order in which lanes read it. x lies there as in memory, 16 columns of a row together; ds_read_b64_tr_b8 hands a lane eight rows of one column.
// The places of a row's 16-byte pieces are exchanged by its number, so that a read of 32 rows takes all banks. A lane's column of 16 is c here, not 4 c ... 4 c + 3: the results
// pass LDS once more on their way out.
template <int OUT, int NT, int RG, int CG> struct Staged {
    static constexpr int THREADS = 64 * RG * CG, ROWS = 16 * NT * RG, COLUMNS = 64 * CG, PIECES = COLUMNS / 16;
    static constexpr int X_EACH = kStep * PIECES / THREADS, W_EACH = ROWS * 8 / THREADS, X_ROWS = THREADS / PIECES;      // 16-byte pieces of a thread; rows of x at a time
    static constexpr int X_BYTES = kStep * COLUMNS, W_BYTES = ROWS * kStep;
    static_assert(X_BYTES >= RG * CG * 4096, "the results' way out");
    static constexpr int GROUP_BYTES = 2 * (X_BYTES + W_BYTES + COLUMNS * 4);
    static constexpr size_t lds(int groups) { return groups * GROUP_BYTES + ROWS * 4; }
    // what a row's pieces are exchanged by
    static __device__ __forceinline__ int place_of(int row) { return PIECES == 16 ? (row & 7) | (row >> 1 & 8) : (row & 7) ^ (row >> 4 & 1); }
    static_assert(PIECES == 8 || PIECES == 16, "columns of a block");
};
typedef int int2_v __attribute__((ext_vector_type(2)));
__device__ __forceinline__ int2_v read_transposed(const unsigned char* lds)
{
    return __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) int2_v*)lds);
}
// What a wave makes of its sums, 16 rows of 64 columns at a time through 4 KB of LDS of its own (`way`; columns exchanged by kq, for the banks); `biases`: of its rows
template <int OUT, int NT>
__device__ __forceinline__ void put_staged(const MixBlocksParams& q, bool out, const float* wscale, float4_v (&total)[NT][4], float* way, const float* biases, int wave_row, long wave_column, long from)
{
    const int lane = threadIdx.x & 63, c = lane & 15, kq = lane >> 4;
    const Results<OUT, false, 4> results = { q, wave_column, from, c, 4 * kq };
    if (__builtin_expect(any_lane(out), 0) && scales_apart<false>(q, wscale, wave_column)) {
        put_plain<OUT, false>(q, results, wave_row, NT, biases);
        return;
    }
    auto put = [&](auto whole_wave) {
        constexpr bool WHOLE = decltype(whole_wave)::value;
#pragma unroll 1
        for (int t = 0; t < NT; t += 2) {
            const int row = wave_row + 16 * t;
            if (!WHOLE && row >= q.rows) break;
            RawOf<OUT> residual[2][4];
            if (q.residual)
#pragma unroll
                for (int u = 0; u < 2; ++u) results.template fetch<WHOLE>(row + 16 * u, residual[u]);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                float4_v v[4];
#pragma unroll
                for (int b = 0; b < 4; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) way[(4 * kq + i) * 64 + (b ^ kq) * 16 + c] = total[u][b][i];
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const float4_v*>(way + (4 * kq + i) * 64 + (c / 4 ^ kq) * 16 + c % 4 * 4);
                results.finish(v, biases + 16 * (t + u) + 4 * kq, residual[u]);
                results.template store<WHOLE>(row + 16 * u, v);
            }
#pragma unroll
            for (int u = 0; u + 2 < NT; ++u)
#pragma unroll
                for (int b = 0; b < 4; ++b) total[u][b] = total[u + 2][b];
        }
    };
    if (wave_column >= from && wave_row + 16 * NT <= q.rows) put(std::true_type());
    else put(std::false_type());
}
// GROUPS = 2: the block's threads twice, the second half of the steps by the second half of them, with LDS of their own. Both take as many, `each` (and meet at the same barriers): of an
// odd number the one in the middle twice, for nothing the second time. The sums of the second group are added to the first one's, which goes on alone; false for the other
template <int NT, int GROUPS, typename S>
__device__ __forceinline__ bool join_groups(int group, int tid, unsigned char* own, unsigned char* others, float4_v (&total)[NT][4], bool& out)
{
    if constexpr (GROUPS == 2) {
        static_assert(NT * 4 * S::THREADS * sizeof(float4_v) <= 2 * S::X_BYTES, "the sums' place");
        __syncthreads();                                // the last step's reads are done
        if (group) {
            float4_v* sums = reinterpret_cast<float4_v*>(own);
            int* flags = reinterpret_cast<int*>(own + 2 * S::X_BYTES);
#pragma unroll
            for (int i = 0; i < NT * 4; ++i) sums[i * S::THREADS + tid] = total[i / 4][i % 4];
            flags[tid] = out;
        }
        __syncthreads();
        if (group) return false;
        const float4_v* sums = reinterpret_cast<const float4_v*>(others);
        out |= reinterpret_cast<const int*>(others + 2 * S::X_BYTES)[tid] != 0;
#pragma unroll
        for (int i = 0; i < NT * 4; ++i) total[i / 4][i % 4] += sums[i * S::THREADS + tid];
    }
    return true;
}
template <int OUT, int NT, int RG, int CG, int WAVES, int GROUPS>
__global__ __launch_bounds__((GROUPS * Staged<OUT, NT, RG, CG>::THREADS), WAVES) void mix_blocks_staged_kernel(const MixBlocksParams q, int row_tiles, long column_tiles, bool by_xcd)
{
    typedef Staged<OUT, NT, RG, CG> S;
    constexpr bool EXACT = OUT == kIn32;
    extern __shared__ uint4_v staged[];
    const int group = GROUPS == 2 ? __builtin_amdgcn_readfirstlane(threadIdx.x / S::THREADS) : 0;
    unsigned char* const bytes = reinterpret_cast<unsigned char*>(staged);
    unsigned char* const xs = bytes + group * S::GROUP_BYTES;       // two buffers each
    unsigned char* const ws = xs + 2 * S::X_BYTES;
    float* const scales = reinterpret_cast<float*>(ws + 2 * S::W_BYTES);
    float* const biases = reinterpret_cast<float*>(bytes + GROUPS * S::GROUP_BYTES);
    const long id = block_index();
    const Tile tile = tile_of(id, row_tiles, column_tiles, by_xcd, OUT == kIn32);
    if (tile.column >= column_tiles) return;
    const int row0 = tile.row * S::ROWS, tid = threadIdx.x % S::THREADS, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, kq = lane >> 4;
    const int wr = wave / CG, wc = wave % CG, wave_row = row0 + wr * 16 * NT;
    const long from = tile.column * S::COLUMNS, column0 = scalar(from + S::COLUMNS <= q.columns ? from : q.columns - S::COLUMNS);      // the last tile ends with the columns
    const int count = q.contraction, steps = (count + kStep - 1) / kStep, whole = count / kStep, each = (steps + GROUPS - 1) / GROUPS, first = group ? steps - each : 0;
    const bool twice = group && 2 * each > steps;
    const float* wscale = q.wscale + (long)(wave_row / kScaleBlock) * ((q.contraction + kScaleBlock - 1) / kScaleBlock);
    const int x_row = tid / S::PIECES, x_piece = tid % S::PIECES;

    uint4_v x[S::X_EACH], w[S::W_EACH];
    float scale = 0.f;
    // pieces of W: eight side by side make 128 bytes of a row
    auto w_row = [&](int e) { return e / 8; };
    auto w_entry = [&](int e) { return e % 8 * 16; };
    // piece j of the thread, of x and then of W, and at last the scale
    auto ask = [&](int s, int j, auto guard) {
        constexpr bool GUARD = decltype(guard)::value;
        if (j < S::X_EACH) {
            const int k = s * kStep + j * S::X_ROWS;
            if constexpr (GUARD) {
                const long row = k + x_row < q.contraction ? k + x_row : q.contraction - 1;
                x[j] = *reinterpret_cast<const uint4_any*>(static_cast<const unsigned char*>(q.x) + row * q.ldx + column0 + 16 * x_piece);
            } else x[j] = *reinterpret_cast<const TFNO_GLOBAL uint4_any*>(scalar(q.x, k * q.ldx + column0) + fresh((unsigned)x_row * (unsigned)q.ldx + 16 * x_piece));
        } else if (j < S::X_EACH + S::W_EACH) {
            const int e = tid + S::THREADS * (j - S::X_EACH), row = row0 + w_row(e) < q.rows ? w_row(e) : q.rows - 1 - row0;
            if constexpr (GUARD) w[j - S::X_EACH] = fetch_weights(q.W, row0 + row, q.rows, count, s * kStep + w_entry(e));
            else w[j - S::X_EACH] = *reinterpret_cast<const TFNO_GLOBAL uint4_any*>(scalar(q.W, (long)row0 * count + s * kStep) + fresh((unsigned)row * (unsigned)count + w_entry(e)));
        } else scale = q.xscale[s * q.positions + column0 + tid % S::COLUMNS];
    };
    constexpr int PIECES = S::X_EACH + S::W_EACH + 1;
    auto keep = [&](int s, auto guard) {
        constexpr bool GUARD = decltype(guard)::value;
        unsigned char* const to = xs + (s & 1) * S::X_BYTES;
#pragma unroll
        for (int i = 0; i < S::X_EACH; ++i) {
            const int row = i * S::X_ROWS + x_row;
            if (GUARD && s * kStep + row >= q.contraction) x[i] = (uint4_v){ 0u, 0u, 0u, 0u };
            *reinterpret_cast<uint4_v*>(to + row * S::COLUMNS + (x_piece ^ S::place_of(row)) * 16) = x[i];
        }
#pragma unroll
        for (int i = 0; i < S::W_EACH; ++i) {
            const int e = tid + S::THREADS * i, row = w_row(e), p = e % 8;
            if constexpr (GUARD) w[i] = mend_weights(w[i], row0 + row, q.rows, count, s * kStep + w_entry(e));
            reinterpret_cast<uint4_v*>(ws + (s & 1) * S::W_BYTES)[row / 16 * 128 + p * 16 + ((row & 15) ^ p)] = w[i];
        }
        scales[(s & 1) * S::COLUMNS + tid % S::COLUMNS] = scale;        // by all threads, without a branch: more than one of them write the same
    };
    auto begin = [&](auto guard) {
#pragma unroll
        for (int j = 0; j < PIECES; ++j) ask(first, j, guard);
        keep(first, guard);
    };
    if (first < whole) begin(std::false_type());
    else begin(std::true_type());
    if (q.bias)
        for (int e = threadIdx.x; e < S::ROWS; e += GROUPS * S::THREADS)
            biases[e] = value_of(static_cast<const typename Columns<OUT>::Value*>(q.bias)[row0 + e < q.rows ? row0 + e : q.rows - 1]);
    __syncthreads();

    float4_v total[NT][4] = {};
    bool out = false;
    float weight_scale = common_scale(wscale + first);
    // a lane reads one half of a row's piece: lanes 2 j and 2 j + 1 row j of eight
    const int piece = wc * 4 ^ S::place_of(16 * kq + (c >> 1));
    const unsigned char* const x_from = xs + (16 * kq + (c >> 1)) * S::COLUMNS + 8 * (c & 1);
    const uint4_v* const w_from = reinterpret_cast<const uint4_v*>(ws) + wr * NT * 128 + kq * 16;
    auto body = [&](int s, auto next, auto guard) {
        constexpr bool NEXT = decltype(next)::value;
        const unsigned char* const here = x_from + (s & 1) * S::X_BYTES;
        const uint4_v *const lower = w_from + (s & 1) * (S::W_BYTES / 16) + (c ^ kq), *const upper = w_from + (s & 1) * (S::W_BYTES / 16) + 64 + (c ^ (4 + kq));
        float4_v joint;
#pragma unroll
        for (int b = 0; b < 4; ++b) joint[b] = scales[(s & 1) * S::COLUMNS + wc * 64 + 16 * b + c];
        joint = joint_scale(joint, weight_scale, out);
        if (GROUPS == 2 && twice && s == first) joint = (float4_v){ 0.f, 0.f, 0.f, 0.f };
        if constexpr (NEXT) weight_scale = common_scale(wscale + s + 1);
        Operands<false, EXACT> ops;
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int2_v v = read_transposed(here + (piece ^ b) * 16 + (u / 2 * 64 + u % 2 * 8) * S::COLUMNS);
                if constexpr (EXACT) {
                    const uint2_v lo = widen((unsigned)v[0]), hi = widen((unsigned)v[1]);
                    ops.b[u][b].v = (uint4_v){ lo[0], lo[1], hi[0], hi[1] };
                } else { ops.b[b][2 * u] = v[0]; ops.b[b][2 * u + 1] = v[1]; }
            }
        // the loads of the next step among the products: all at once, they would keep the waves from their products
        constexpr int TURNS = EXACT ? NT : 2 * NT;
        auto ask_some = [&](int turn) {
            if constexpr (NEXT)
#pragma unroll
                for (int j = 0; j < PIECES; ++j)
                    if (j * TURNS / PIECES == turn) ask(s + 1, j, guard);
        };
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (EXACT) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const uint4_v a[2] = { lower[t * 128], upper[t * 128] };
                float4_v part[4];
                ask_some(t);
                ops.product(a, 0, part);
                add_scaled(joint, 0, part, total[t]);
                __builtin_amdgcn_sched_barrier(0);
            }
        } else {
            // two columns' products at a time; they are added while the next two are formed
            float4_v part[2][2];
            uint4_v a[2] = { lower[0], upper[0] };
            ops.product(a, 0, part[0]);
#pragma unroll
            for (int i = 1; i <= 2 * NT; ++i) {
                ask_some(i - 1);
                if (i < 2 * NT) {
                    if (i % 2 == 0) { a[0] = lower[i / 2 * 128]; a[1] = upper[i / 2 * 128]; }
                    ops.product(a, i % 2 * 2, part[i % 2]);
                }
                add_scaled(joint, (i - 1) % 2 * 2, part[(i - 1) % 2], total[(i - 1) / 2]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if constexpr (NEXT) {
            keep(s + 1, guard);
            __syncthreads();
        }
    };
    const int end = first + each;
    int s = first;
    for (; s < end - 1 && s + 1 < whole; ++s) body(s, std::true_type(), std::false_type());
    if (s < end - 1) body(s++, std::true_type(), std::true_type());
    body(s, std::false_type(), std::false_type());

    if (!join_groups<NT, GROUPS, S>(group, tid, xs, bytes + S::GROUP_BYTES, total, out)) return;
    // the results' way out: the buffer that the last step did not read
    put_staged<OUT, NT>(q, out, wscale, total, reinterpret_cast<float*>(xs + (end & 1) * S::X_BYTES) + wave * 1024, biases + wr * 16 * NT, wave_row,
                        scalar(column0 + wc * 64), from);
}

// The same where whole steps and 16-byte pieces are all there is, for bf16 results: memory is read into LDS directly, past the registers. The registers that this leaves hold the
// operands of x of the next step, read in the second half of this one. So a buffer of x is free again a step earlier than one of W: x is asked for two steps ahead, W one.
// Loads arrive in their order, and the loop has no others: in the middle of a step those of the step before have, at its end those of W too. Each wait is followed by a barrier,
// for the other waves' loads; the last step ends with none on the way.
template <int NT, int GROUPS> __global__ __launch_bounds__(256 * GROUPS, (NT == 4 || GROUPS == 2 ? 2 : 3)) void mix_blocks_direct_kernel(const MixBlocksParams q, int row_tiles, long column_tiles, bool by_xcd)
{
    typedef Staged<kIn16, NT, 2, 2> S;
    extern __shared__ uint4_v staged[];
    const int group = GROUPS == 2 ? __builtin_amdgcn_readfirstlane(threadIdx.x / S::THREADS) : 0;
    unsigned char* const bytes = reinterpret_cast<unsigned char*>(staged);
    unsigned char *const xs = bytes + group * S::GROUP_BYTES, *const ws = xs + 2 * S::X_BYTES;
    float* const scales = reinterpret_cast<float*>(ws + 2 * S::W_BYTES);
    float* const biases = reinterpret_cast<float*>(bytes + GROUPS * S::GROUP_BYTES);
    const long id = block_index();
    const Tile tile = tile_of(id, row_tiles, column_tiles, by_xcd, false);
    if (tile.column >= column_tiles) return;
    const int row0 = tile.row * S::ROWS, tid = threadIdx.x % S::THREADS, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, kq = lane >> 4;
    const int wr = wave / 2, wc = wave % 2, wave_row = row0 + wr * 16 * NT;
    const long from = tile.column * S::COLUMNS, column0 = scalar(from + S::COLUMNS <= q.columns ? from : q.columns - S::COLUMNS);
    const int count = q.contraction, steps = count / kStep, each = (steps + GROUPS - 1) / GROUPS, first = group ? steps - each : 0;
    const bool twice = group && 2 * each > steps;
    const float* wscale = q.wscale + (long)(row0 / kScaleBlock) * steps;
    const unsigned x_offset = (unsigned)(lane / 8) * (unsigned)q.ldx + 16 * ((lane % 8) ^ S::place_of(8 * wave + lane / 8));
    constexpr int X_CALLS = S::X_BYTES / 4096, W_CALLS = S::W_BYTES / 4096;
    unsigned w_offset[W_CALLS];
#pragma unroll
    for (int j = 0; j < W_CALLS; ++j) {
        const int u = (4 * j + wave) * 64 + lane, p = u / 16 % 8, row = u / 128 * 16 + ((u & 15) ^ p);
        w_offset[j] = (unsigned)(row0 + row < q.rows ? row : q.rows - 1 - row0) * (unsigned)count + 16 * p;
    }
    long x_at = scalar((first * kStep + wave * 8) * q.ldx + column0);     // of the step that is asked for next
    const long x_part = scalar(32 * q.ldx);
    auto ask_x = [&](int s, int j) {
        direct_to_lds(scalar(q.x, x_at), x_offset, place_in_lds(xs) + (s & 1) * S::X_BYTES + (4 * j + wave) * 1024);
        x_at += x_part;
    };
    auto ask_w = [&](int s, int j) {
        direct_to_lds(scalar(q.W, (long)row0 * count + s * kStep), w_offset[j], place_in_lds(ws) + (s & 1) * S::W_BYTES + (4 * j + wave) * 1024);
    };
    auto ask_scales = [&](int s) {                      // by two waves each half of them
        direct_word_to_lds(scalar(q.xscale, 4 * (s * q.positions + column0 + wc * 64)), 4 * lane, place_in_lds(scales) + ((s & 1) * S::COLUMNS + wc * 64) * 4);
    };
    // all but the last `later` of each wave's loads have arrived
    auto arrived = [&](auto later) {
        asm volatile("s_waitcnt vmcnt(%0)" : : "n"(decltype(later)::value) : "memory");
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    };
    constexpr std::integral_constant<int, 0> none;
    if (q.bias)
        for (int e = threadIdx.x; e < S::ROWS; e += GROUPS * S::THREADS) biases[e] = value_of(static_cast<const unsigned short*>(q.bias)[row0 + e < q.rows ? row0 + e : q.rows - 1]);
#pragma unroll
    for (int j = 0; j < X_CALLS; ++j) ask_x(first, j);
    ask_scales(first);
#pragma unroll
    for (int j = 0; j < W_CALLS; ++j) ask_w(first, j);
    if (each > 1) {
#pragma unroll
        for (int j = 0; j < X_CALLS; ++j) ask_x(first + 1, j);
        ask_scales(first + 1);
    }
    const int piece = wc * 4 ^ S::place_of(16 * kq + (c >> 1));
    const unsigned char* const x_from = xs + (16 * kq + (c >> 1)) * S::COLUMNS + 8 * (c & 1);
    const uint4_v* const w_from = reinterpret_cast<const uint4_v*>(ws) + wr * NT * 128 + kq * 16;
    int8_v next[4];
    float4_v next_scale;
    float weight_scale = common_scale(wscale + first);
    auto read_x = [&](int s, int b) {                   // 16 columns
        const unsigned char* const here = x_from + (s & 1) * S::X_BYTES;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int2_v v = read_transposed(here + (piece ^ b) * 16 + (u / 2 * 64 + u % 2 * 8) * S::COLUMNS);
            next[b][2 * u] = v[0];
            next[b][2 * u + 1] = v[1];
        }
        next_scale[b] = scales[(s & 1) * S::COLUMNS + wc * 64 + 16 * b + c];
    };
    if (each > 1) arrived(std::integral_constant<int, X_CALLS + 1>());
    else arrived(none);
#pragma unroll
    for (int b = 0; b < 4; ++b) read_x(first, b);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    float4_v total[NT][4] = {};
    bool out = false;
    // LEFT: steps after this one, 2 for more
    auto body = [&](int s, auto left) {
        constexpr int LEFT = decltype(left)::value;
        Operands<false, false> ops;
#pragma unroll
        for (int b = 0; b < 4; ++b) ops.b[b] = next[b];
        float4_v joint = joint_scale(next_scale, weight_scale, out);
        if (GROUPS == 2 && twice && s == first) joint = (float4_v){ 0.f, 0.f, 0.f, 0.f };
        const uint4_v *const lower = w_from + (s & 1) * (S::W_BYTES / 16) + (c ^ kq), *const upper = w_from + (s & 1) * (S::W_BYTES / 16) + 64 + (c ^ (4 + kq));
        constexpr int CALLS = X_CALLS + W_CALLS + 1;
        auto ask_some = [&](int turn) {
#pragma unroll
            for (int j = 0; j < CALLS; ++j)
                if (j * (NT - 1) / CALLS == turn) {
                    if (j < W_CALLS) { if constexpr (LEFT >= 1) ask_w(s + 1, j); }
                    else if (j < W_CALLS + X_CALLS) { if constexpr (LEFT >= 2) ask_x(s + 2, j - W_CALLS); }
                    else if constexpr (LEFT >= 2) ask_scales(s + 2);
                }
        };
        float4_v part[2][2];
        uint4_v a[2][2] = { { lower[0], upper[0] } };
        if constexpr (LEFT >= 1) weight_scale = common_scale(wscale + s + 1);
        __builtin_amdgcn_sched_barrier(0);
        ops.product(a[0], 0, part[0]);
#pragma unroll
        for (int i = 1; i <= 2 * NT; ++i) {
            if (i % 2 && i / 2 + 1 < NT) { a[(i / 2 + 1) % 2][0] = lower[(i / 2 + 1) * 128]; a[(i / 2 + 1) % 2][1] = upper[(i / 2 + 1) * 128]; }
            ask_some(i - 1);
            if (i < 2 * NT) ops.product(a[i / 2 % 2], i % 2 * 2, part[i % 2]);
            add_scaled(joint, (i - 1) % 2 * 2, part[(i - 1) % 2], total[(i - 1) / 2]);
            if (LEFT >= 1 && i == NT) arrived(std::integral_constant<int, LEFT == 2 ? CALLS : W_CALLS>());
            if constexpr (LEFT >= 1)
#pragma unroll
                for (int b = 0; b < 4; ++b)
                    if (i == NT + 1 + b * NT / 4) read_x(s + 1, b);
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (LEFT >= 1) arrived(std::integral_constant<int, LEFT == 2 ? X_CALLS + 1 : 0>());
    };
    const int end = first + each;
    int s = first;
    for (; s < end - 2; ++s) body(s, std::integral_constant<int, 2>());
    if (s == end - 2) body(s++, std::integral_constant<int, 1>());
    body(s, std::integral_constant<int, 0>());
    if (!join_groups<NT, GROUPS, S>(group, tid, xs, bytes + S::GROUP_BYTES, total, out)) return;
    put_staged<kIn16, NT>(q, out, wscale, total, reinterpret_cast<float*>(xs) + wave * 1024, biases + wr * 16 * NT, wave_row, scalar(column0 + wc * 64), from);
}

// ---- few columns: the waves of a block share 64 columns and 16 rows, and the steps are divided among them ----

constexpr int kSplitWaves = 8;
template <int OUT, bool COMPLEX, int MODE>
__device__ __forceinline__ void split(const MixBlocksParams& q, float4_v* sums, long column0, int row0)
{
    constexpr int V = COMPLEX ? 2 : 1;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const Input<COMPLEX, MODE> in(q, column0);
    // what wave i < 4 finishes in the end, the rows 4 kq + i: asked for ahead of the products
    const Results<OUT, COMPLEX, 1> results = { q, column0, column0, in.c, 4 * in.kq + (wave & 3) };
    float bias[V];
    RawOf<OUT> residual[1];
    if (q.bias)
#pragma unroll
        for (int i = 0; i < V; ++i) bias[i] = results.bias_at(row0 + results.lane_row, i);
    if (q.residual && column0 + 4 * in.c < q.columns) results.template fetch<false>(row0, residual);
    float4_v total[4] = {};
    sum_steps<OUT, COMPLEX, MODE>(q, in, row0, wave, kSplitWaves, total);
    // joined in a fixed order
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[(wave * 4 + i) * 64 + lane] = row_of(total, i);
    __syncthreads();
    if (wave >= 4) return;
    float4_v v[1] = { sums[wave * 64 + lane] };
#pragma unroll
    for (int u = 1; u < kSplitWaves; ++u) v[0] += sums[(u * 4 + wave) * 64 + lane];
    if (row0 + results.lane_row >= q.rows || column0 + 4 * in.c >= q.columns) return;
    results.finish(v, bias, residual);
    results.template store<false>(row0, v);
}
template <int OUT, bool COMPLEX, int MODE> __global__ __launch_bounds__(64 * kSplitWaves, 2) void mix_blocks_split_kernel(const MixBlocksParams q, int row_tiles)
{
    __shared__ float4_v sums[kSplitWaves * 4 * 64];
    const long id = block_index(), column0 = id / row_tiles * kColumns;
    if (column0 < q.columns) split<OUT, COMPLEX, MODE>(q, sums, column0, (int)(id % row_tiles) * 16);
}

// The launches refuse fewer columns than a wave or a block reads: it would read ahead of its operands
template <int NT> hipError_t launch_tiles(const MixBlocksParams& q, hipStream_t stream)
{
    if (q.columns < kColumns) return hipErrorInvalidValue;
    const long column_tiles = (q.columns + 4 * kColumns - 1) / (4 * kColumns);
    const int row_tiles = (q.rows + 16 * NT - 1) / (16 * NT);
    const bool by_xcd = tiles_by_xcd(column_tiles);
    hipLaunchKernelGGL((mix_blocks_tile_kernel<NT>), grid_of(tile_blocks(row_tiles, column_tiles)), dim3(256), 0, stream, q, row_tiles,
                       column_tiles, by_xcd);
    return hipGetLastError();
}
template <int OUT, int NT, int RG, int CG, int WAVES, int GROUPS> hipError_t launch_staged(const MixBlocksParams& q, hipStream_t stream)
{
    typedef Staged<OUT, NT, RG, CG> S;
    if (q.columns < S::COLUMNS) return hipErrorInvalidValue;
    static std::atomic<unsigned long long> served{ 0 };
    if (hipError_t e = allow_dynamic_lds(reinterpret_cast<const void*>(mix_blocks_staged_kernel<OUT, NT, RG, CG, WAVES, GROUPS>), S::lds(GROUPS), served); e != hipSuccess) return e;
    const long column_tiles = (q.columns + S::COLUMNS - 1) / S::COLUMNS;
    const int row_tiles = (q.rows + S::ROWS - 1) / S::ROWS;
    const bool by_xcd = tiles_by_xcd(column_tiles);
    hipLaunchKernelGGL((mix_blocks_staged_kernel<OUT, NT, RG, CG, WAVES, GROUPS>), grid_of(tile_blocks(row_tiles, column_tiles)), dim3(GROUPS * S::THREADS), S::lds(GROUPS), stream, q,
                       row_tiles, column_tiles, by_xcd);
    return hipGetLastError();
}
template <int NT, int GROUPS> hipError_t launch_direct(const MixBlocksParams& q, hipStream_t stream)
{
    typedef Staged<kIn16, NT, 2, 2> S;
    if (q.columns < S::COLUMNS) return hipErrorInvalidValue;
    static std::atomic<unsigned long long> served{ 0 };
    if (hipError_t e = allow_dynamic_lds(reinterpret_cast<const void*>(mix_blocks_direct_kernel<NT, GROUPS>), S::lds(GROUPS), served); e != hipSuccess) return e;
    const long column_tiles = (q.columns + S::COLUMNS - 1) / S::COLUMNS;
    const int row_tiles = (q.rows + S::ROWS - 1) / S::ROWS;
    const bool by_xcd = tiles_by_xcd(column_tiles);
    hipLaunchKernelGGL((mix_blocks_direct_kernel<NT, GROUPS>), grid_of(tile_blocks(row_tiles, column_tiles)), dim3(GROUPS * S::THREADS), S::lds(GROUPS), stream, q,
                       row_tiles, column_tiles, by_xcd);
    return hipGetLastError();
}
template <int OUT, bool COMPLEX> hipError_t launch(const MixBlocksParams& q, int type, hipStream_t stream)
{
    const BlocksChoice choice = blocks_choice({ COMPLEX, OUT == kIn32, q.columns, q.ldx, q.ldr, q.ldy, q.rows, q.contraction, (((long)q.x | (long)q.W) & 15) == 0 });
    if (choice.kernel == BlocksKernel::kOneScale) {
        const MixParams p = { q.x, nullptr, q.W, q.bias, q.residual, q.xscale, q.wscale, q.y, nullptr, q.columns, q.ldx, 0, q.ldr, q.ldy, 0, q.rows, q.contraction, q.contraction, q.act,
                              kScaleShift };
        return launch_mix_8bit(p, type, stream);
    }
    if (choice.kernel == BlocksKernel::kSplitNear || choice.kernel == BlocksKernel::kSplitFar) {
        const int tiles16 = (q.rows + 15) / 16;
        const dim3 grid = grid_of((q.columns + kColumns - 1) / kColumns * tiles16), block(64 * kSplitWaves);
        if (choice.kernel == BlocksKernel::kSplitNear) hipLaunchKernelGGL((mix_blocks_split_kernel<OUT, COMPLEX, kNarrow>), grid, block, 0, stream, q, tiles16);
        else hipLaunchKernelGGL((mix_blocks_split_kernel<OUT, COMPLEX, kFar64>), grid, block, 0, stream, q, tiles16);
        return hipGetLastError();
    }
    if constexpr (COMPLEX) return choice.nt == 4 ? launch_tiles<4>(q, stream) : launch_tiles<2>(q, stream);
    else {
        if constexpr (OUT == kIn16)
            if (choice.kernel == BlocksKernel::kDirect) return choice.nt == 4 ? launch_direct<4, 1>(q, stream) : choice.groups == 2 ? launch_direct<2, 2>(q, stream) : launch_direct<2, 1>(q, stream);
        if (choice.nt == 4) return launch_staged<OUT, 4, 2, OUT == kIn32 ? 4 : 2, 2, 1>(q, stream);
        return choice.groups == 2 ? launch_staged<OUT, 2, 2, 2, 2, 2>(q, stream) : launch_staged<OUT, 2, 2, 2, 3, 1>(q, stream);
    }
}

}  // namespace

hipError_t launch_mix_8bit_blocks(const MixBlocksParams& q, int type, hipStream_t stream)
{
    if (q.columns == 0) return hipSuccess;
    switch (type) {
    case kC64: return launch<kIn32, true>(q, type, stream);
    case kF32: return launch<kIn32, false>(q, type, stream);
    default: return launch<kIn16, false>(q, type, stream);
    }
}

}  // namespace tfno
