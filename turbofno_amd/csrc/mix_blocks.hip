// Channel product of 8-bit operands with a scale for each block of 128 channels (turbofno_mix_8bit_blocks):
//
//   z[n][p] = sum_b xscale[b][p] wscale[n / 128][b] (sum over the channels k of block b of Wq[n][k] xq[k][p]) + bias[n] + residual[n][p],   y = act(z)
//
// As in the other channel products a complex row of P positions is a row of 2 P real columns, a wave takes 64 columns, a lane four consecutive ones,
// 4 c ... 4 c + 3 with c = lane % 16, of the input, the residual and the result. A step holds 128 real values of the contraction, one block of channels (complex: half
// of one). A quarter kq of the wave has the values 16 kq ... 16 kq + 15 of each half of a step, in this order in the operands of both sides: the lane reads whole
// rows of x, four columns each, and transposes them in its own registers; x passes no LDS.
//   bf16 result    one matrix instruction takes a step of 16 rows and columns, 128 products of 8-bit operands. It drops what lies more than about 2^-19 below the
//                  largest product: at most 2^-12 of the sum of magnitudes together, 1e-5 of a typical sum (the result's rounding: 2^-9 of it).
//   fp32 result    the operands are widened to bf16, which holds them exactly, and take four matrix instructions whose sums are fp32.
// The sum of a step is multiplied by both scales and added to the total, in fp32.
#include "kernels.h"
#include "mix_kernel.h"

namespace tfno {

namespace {

typedef int int8_v __attribute__((ext_vector_type(8)));
typedef uint4_v uint4_any __attribute__((aligned(1)));
constexpr int kStep = 128;                              // real values of a step

// ---- the input ----

template <bool COMPLEX> constexpr int kRowsOfHalf = COMPLEX ? 8 : 16;
template <bool COMPLEX> struct RawStep {
    unsigned row[2][kRowsOfHalf<COMPLEX>];              // four columns of the lane's channels
    float4_v scale;                                     // of the columns
};
// Columns of a wave, from column0 on, of which `there` exist, at least one. CAREFUL: fewer than 64 may exist, channels may lie any distance apart
template <bool COMPLEX, bool CAREFUL> struct Input {
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
        const unsigned quarter = fresh((unsigned)(kq * HALF) * (unsigned)q.ldx + 4 * c);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < HALF; ++j) {
                const int k = first + h * 4 * HALF + j;         // the first quarter's
                if constexpr (CAREFUL) {
                    // a word that would end behind the last value of all starts earlier and is shifted; what it holds beyond its row's end is not used
                    const long row = k + kq * HALF < q.contraction ? k + kq * HALF : q.contraction - 1;
                    const long at = row * q.ldx + column0 + (4 * c < there ? 4 * c : 0), last = (q.contraction - 1) * q.ldx + q.columns - 4;
                    const unsigned char* x = static_cast<const unsigned char*>(q.x);
                    if (last < 0) {                             // fewer than four values
                        unsigned v = 0;
                        for (int i = 0; i < 4; ++i) v |= at + i < last + 4 ? (unsigned)x[at + i] << 8 * i : 0u;
                        raw.row[h][j] = v;
                    } else raw.row[h][j] = *reinterpret_cast<const uint_any*>(x + (at < last ? at : last)) >> (at > last ? 8 * (int)(at - last) : 0);
                } else if constexpr (GUARD) {
                    const int common = k < q.contraction ? k : q.contraction - 1;
                    raw.row[h][j] = near_load4<kIn8>(scalar(q.x, common * q.ldx + column0), fresh(k + kq * HALF < q.contraction ? quarter : 4 * c));
                } else raw.row[h][j] = near_load4<kIn8>(scalar(q.x, k * q.ldx + column0), quarter);
            }
        const long scales = step / V * q.positions;
        if constexpr (CAREFUL)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const long column = column0 + 4 * c + i;
                raw.scale[i] = q.xscale[scales + (column >= q.columns ? q.columns - 1 : column) / V];
            }
        else if constexpr (COMPLEX) {
            const uint2_v v = near_load4<kIn16>(scalar(q.xscale, (scales + column0 / 2) * 4), fresh(8 * c));        // two floats, any multiple of 4 bytes
            const float2_v f = __builtin_bit_cast(float2_v, v);
            raw.scale = (float4_v){ f[0], f[0], f[1], f[1] };
        } else raw.scale = near_load4<kIn32>(scalar(q.xscale, (scales + column0) * 4), fresh(16 * c));
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

// total += part x w, both scales of a step: by their product, an ordinary number (`out`: it is none in some lane), or the larger one first
__device__ __forceinline__ float4_v joint_scale(float4_v x, float w, bool& out)
{
    x *= w;
#pragma unroll
    for (int i = 0; i < 4; ++i) out |= !(x[i] >= 0x1p-126f && x[i] <= 0x1p127f);
    return x;
}
template <int COUNT> __device__ __forceinline__ void add_scaled(float4_v joint, int first, const float4_v (&part)[COUNT], float4_v (&total)[4])
{
#pragma unroll
    for (int b = 0; b < COUNT; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) total[first + b][i] = __builtin_fmaf(part[b][i], joint[first + b], total[first + b][i]);
}
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

// Bytes e ... e + 15 of a row of `count`, from memory; where they would end behind the last weight, earlier ones, and mend_weights() has to follow. `few`: there are
// fewer than 16 weights
__device__ __forceinline__ uint4_v fetch_weights(const void* W, int row, int rows, int count, int e, bool few)
{
    const unsigned char* w = static_cast<const unsigned char*>(W);
    const long at = (long)(row < rows ? row : rows - 1) * count + e, last = (long)rows * count - 16;
    if (few) {
        uint4_v v = {};
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i / 4] |= at + i < last + 16 ? (unsigned)w[at + i] << i % 4 * 8 : 0u;
        return v;
    }
    return *reinterpret_cast<const uint4_any*>(w + (at < last ? at : last));
}
// zeros for bytes from `count` on
__device__ __forceinline__ uint4_v mend_weights(uint4_v v, int row, int rows, int count, int e, bool few)
{
    if (e + 16 <= count) return v;
    const long at = (long)(row < rows ? row : rows - 1) * count + e, last = (long)rows * count - 16;
    const int by = few || at <= last ? 0 : at - last < 16 ? (int)(at - last) : 15;
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
// ROWS rows row0 + i, four columns each from `column` on, of which those of lower numbers than `from` and those beyond the last are left alone: bias, residual,
// activation. All loads first
template <int OUT, bool COMPLEX, int ROWS>
__device__ __forceinline__ void put_rows(const MixBlocksParams& q, long column, long from, int row0, float4_v (&v)[ROWS])
{
    typedef typename Columns<OUT>::Value Value;
    constexpr int V = COMPLEX ? 2 : 1;
    if (column >= q.columns || column + 4 <= from) return;
    const bool whole = column >= from && column + 4 <= q.columns;
    auto at = [&](int i) { return (long)(row0 + i < q.rows ? row0 + i : q.rows - 1); };
    RawOf<OUT> residual[ROWS];
    if (q.residual)
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const Value* p = static_cast<const Value*>(q.residual) + at(i) * q.ldr;
            residual[i] = whole ? load4<OUT>(p, column) : load4_ragged<OUT>(p, column, q.columns);
        }
    if (q.bias)
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const Value* p = static_cast<const Value*>(q.bias) + at(i) * V;
            const float re = value_of(p[0]), im = value_of(p[V - 1]);
            v[i] += (float4_v){ re, im, re, im };
        }
    if (q.residual)
#pragma unroll
        for (int i = 0; i < ROWS; ++i) v[i] += to_float<OUT>(residual[i]);
    if (q.act == kActGeluTanh) activate_rows<kActGeluTanh>(v);
    else if (q.act == kActSilu) activate_rows<kActSilu>(v);
    else if (q.act == kActRelu) activate_rows<kActRelu>(v);
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        if (row0 + i >= q.rows) break;
        Value* p = static_cast<Value*>(q.y) + at(i) * q.ldy;
        const RawOf<OUT> raw = from_float<OUT>(v[i]);
        if (whole) store4<OUT>(p, column, raw);
        else
#pragma unroll
            for (int b = 0; b < 4; ++b)
                if (column + b >= from && column + b < q.columns) {
                    if constexpr (OUT == kIn32) p[column + b] = raw[b];
                    else p[column + b] = (unsigned short)(b & 1 ? raw[b / 2] >> 16 : raw[b / 2]);
                }
    }
}
__device__ __forceinline__ float4_v row_of(const float4_v (&total)[4], int i) { return (float4_v){ total[0][i], total[1][i], total[2][i], total[3][i] }; }

// ---- 16 rows of one wave, steps wave, wave + waves ...: weights straight from memory ----

template <int OUT, bool COMPLEX, bool CAREFUL>
__device__ __forceinline__ void sum_steps(const MixBlocksParams& q, const Input<COMPLEX, CAREFUL>& in, int row0, int first, int stride, bool few, float4_v (&total)[4])
{
    const int count = q.contraction * (COMPLEX ? 2 : 1), steps = (count + kStep - 1) / kStep;
    const int blocks = (q.contraction + kScaleBlock - 1) / kScaleBlock;
    const float* wscale = q.wscale + (long)(row0 / kScaleBlock) * blocks;
    RawStep<COMPLEX> raw;
    uint4_v w[2];
    auto ask = [&](int s) {
        in.template fetch<true>(s, raw);
#pragma unroll
        for (int h = 0; h < 2; ++h) w[h] = fetch_weights(q.W, row0 + in.c, q.rows, count, s * kStep + 64 * h + 16 * in.kq, CAREFUL && few);
    };
    if (first < steps) ask(first);
    for (int s = first; s < steps; s += stride) {
        in.clear(s, raw);
        if ((s + 1) * kStep > count)
#pragma unroll
            for (int h = 0; h < 2; ++h) w[h] = mend_weights(w[h], row0 + in.c, q.rows, count, s * kStep + 64 * h + 16 * in.kq, CAREFUL && few);
        const float4_v scale = raw.scale;
        const float ws = wscale[s / (COMPLEX ? 2 : 1)];
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

// ---- many columns: four waves side by side share 16 NT rows of W ----

// The weights of a step pass LDS, in the order in which lanes read them: 16 bytes per lane, half and 16 rows. Two buffers: a step's are written while those of the
// step before are read, after they were asked for ahead of its products, like the rows of x of the next step. A wave whose 64 columns are not all there takes the last
// 64 and leaves those that it shares with others alone; one that has none goes along for its part of the weights.
template <int OUT, bool COMPLEX, int NT>
__global__ __launch_bounds__(256, 2) void mix_blocks_tile_kernel(const MixBlocksParams q, int row_tiles, long column_tiles, bool by_xcd)
{
    constexpr bool EXACT = OUT == kIn32;
    constexpr int CHUNKS = NT * 128, PHASES = NT == 8 ? 2 : 1, EACH = CHUNKS / 256 / PHASES;        // 16 bytes each; asked for at once by a thread
    __shared__ uint4_v weights[2 * CHUNKS];
    const long id = block_index();
    // Blocks go to the eight XCDs in turns: with many columns those of the same columns follow one another on one XCD, whose L2 cache then holds them
    const long slot = by_xcd ? id / 8 : id, column_tile = by_xcd ? slot / row_tiles * 8 + id % 8 : slot / row_tiles;
    if (column_tile >= column_tiles) return;
    const int row0 = (int)(slot % row_tiles) * (16 * NT), lane = threadIdx.x & 63;
    const long from = column_tile * (4 * kColumns) + (long)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * kColumns;
    const Input<COMPLEX, false> in(q, scalar(from + kColumns <= q.columns ? from : q.columns - kColumns));
    const int count = q.contraction * (COMPLEX ? 2 : 1), steps = (count + kStep - 1) / kStep;
    const float* wscale = q.wscale + (long)(row0 / kScaleBlock) * ((q.contraction + kScaleBlock - 1) / kScaleBlock);
    const int whole = count / kStep;                    // steps of 128 values
    uint4_v w[EACH];
    auto chunk = [&](int i) { return (int)threadIdx.x + 256 * i; };
    auto chunk_row = [&](int e) { return e / 128 * 16 + (e & 15); };
    auto chunk_entry = [&](int e) { return (e >> 6 & 1) * 64 + (e >> 4 & 3) * 16; };
    auto ask = [&](int s, int phase, auto guard) {
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int e = chunk(phase * EACH + i), row = row0 + chunk_row(e) < q.rows ? chunk_row(e) : q.rows - 1 - row0;
            if constexpr (decltype(guard)::value) w[i] = fetch_weights(q.W, row0 + row, q.rows, count, s * kStep + chunk_entry(e), false);
            else w[i] = *reinterpret_cast<const TFNO_GLOBAL uint4_any*>(scalar(q.W, (long)row0 * count + s * kStep) + fresh((unsigned)row * (unsigned)count + chunk_entry(e)));
        }
    };
    auto keep = [&](int s, int phase, auto guard) {
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int e = chunk(phase * EACH + i);
            if constexpr (decltype(guard)::value) w[i] = mend_weights(w[i], row0 + chunk_row(e), q.rows, count, s * kStep + chunk_entry(e), false);
            weights[(s & 1) * CHUNKS + e] = w[i];
        }
    };
    RawStep<COMPLEX> raw;
    auto begin = [&](auto guard) {
        in.template fetch<decltype(guard)::value>(0, raw);
#pragma unroll
        for (int p = 0; p < PHASES; ++p) {
            ask(0, p, guard);
            keep(0, p, guard);
        }
    };
    float4_v total[NT][4] = {};
    bool out = false;
    // step s; NEXT: the one after it is asked for, GUARD: which is the last one and not whole
    auto body = [&](int s, auto next, auto guard) {
        constexpr bool NEXT = decltype(next)::value, GUARD = decltype(guard)::value;
        const float4_v joint = joint_scale(raw.scale, wscale[s / (COMPLEX ? 2 : 1)], out);
        Operands<COMPLEX, EXACT> ops;
        ops.make(raw);
        if constexpr (NEXT) {
            in.template fetch<GUARD>(s + 1, raw);
            ask(s + 1, 0, guard);
        }
        __builtin_amdgcn_sched_barrier(0);              // the loads stay ahead of the products
        const uint4_v* from_lds = weights + (s & 1) * CHUNKS + lane;
        if constexpr (EXACT) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const uint4_v a[2] = { from_lds[t * 128], from_lds[t * 128 + 64] };
                float4_v part[4];
                ops.product(a, 0, part);
                add_scaled(joint, 0, part, total[t]);
                __builtin_amdgcn_sched_barrier(0);
            }
        } else {
            // two columns' products at a time; they are added while the next two are formed
            float4_v part[2][2];
            uint4_v a[2] = { from_lds[0], from_lds[64] };
            ops.product(a, 0, part[0]);
#pragma unroll
            for (int i = 1; i <= 2 * NT; ++i) {
                if (i < 2 * NT) {
                    if (i % 2 == 0) { a[0] = from_lds[i / 2 * 128]; a[1] = from_lds[i / 2 * 128 + 64]; }
                    ops.product(a, i % 2 * 2, part[i % 2]);
                }
                add_scaled(joint, (i - 1) % 2 * 2, part[(i - 1) % 2], total[(i - 1) / 2]);
                if (NEXT && PHASES == 2 && i == NT) {
                    keep(s + 1, 0, guard);
                    ask(s + 1, 1, guard);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if constexpr (NEXT) {
            keep(s + 1, PHASES - 1, guard);
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
    const long column = in.column0 + 4 * in.c;
    if (__builtin_expect(any_lane(out), 0)) {           // scales that may not be multiplied first: the sums once more, 16 rows at a time
#pragma unroll 1
        for (int row = row0; row < row0 + 16 * NT && row < q.rows; row += 16) {
            float4_v sums[4] = {}, v[4];
            sum_steps<OUT, COMPLEX, false>(q, in, row, 0, 1, false, sums);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = row_of(sums, i);
            put_rows<OUT, COMPLEX, 4>(q, column, from, row + 4 * in.kq, v);
        }
        return;
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        if (row0 + 16 * t >= q.rows) break;
        float4_v v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = row_of(total[t], i);
        put_rows<OUT, COMPLEX, 4>(q, column, from, row0 + 16 * t + 4 * in.kq, v);
    }
}

// ---- few columns: the waves of a block share 64 columns and 16 rows, and the steps are divided among them ----

constexpr int kSplitWaves = 8;
template <int OUT, bool COMPLEX, bool CAREFUL>
__device__ __forceinline__ void split(const MixBlocksParams& q, float4_v* sums, long column0, int row0, bool few)
{
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const Input<COMPLEX, CAREFUL> in(q, column0);
    float4_v total[4] = {};
    sum_steps<OUT, COMPLEX, CAREFUL>(q, in, row0, wave, kSplitWaves, few, total);
    // joined in a fixed order: wave i takes the rows 4 kq + i
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[(wave * 4 + i) * 64 + lane] = row_of(total, i);
    __syncthreads();
    if (wave >= 4) return;
    float4_v v[1] = { sums[wave * 64 + lane] };
#pragma unroll
    for (int u = 1; u < kSplitWaves; ++u) v[0] += sums[(u * 4 + wave) * 64 + lane];
    put_rows<OUT, COMPLEX, 1>(q, in.column0 + 4 * in.c, 0, row0 + 4 * in.kq + wave, v);
}
template <int OUT, bool COMPLEX> __global__ __launch_bounds__(64 * kSplitWaves, 2) void mix_blocks_split_kernel(const MixBlocksParams q, int row_tiles, bool careful, bool few)
{
    __shared__ float4_v sums[kSplitWaves * 4 * 64];
    const long id = block_index(), column0 = id / row_tiles * kColumns;
    if (column0 >= q.columns) return;
    const int row0 = (int)(id % row_tiles) * 16;
    if (careful || column0 + kColumns > q.columns) split<OUT, COMPLEX, true>(q, sums, column0, row0, few);
    else split<OUT, COMPLEX, false>(q, sums, column0, row0, few);
}

template <int OUT, bool COMPLEX, int NT> hipError_t launch_tiles(const MixBlocksParams& q, hipStream_t stream)
{
    const long column_tiles = (q.columns + 4 * kColumns - 1) / (4 * kColumns);
    const int row_tiles = (q.rows + 16 * NT - 1) / (16 * NT);
    const bool by_xcd = column_tiles >= 64;
    hipLaunchKernelGGL((mix_blocks_tile_kernel<OUT, COMPLEX, NT>), grid_of((by_xcd ? (column_tiles + 7) / 8 * 8 : column_tiles) * row_tiles), dim3(256), 0, stream, q, row_tiles,
                       column_tiles, by_xcd);
    return hipGetLastError();
}
template <int OUT, bool COMPLEX> hipError_t launch(const MixBlocksParams& q, hipStream_t stream)
{
    // a lane's part of an address in 32 bits, 48 rows of the input (complex: 24); weights that cannot be read by 16
    const bool few = (long)q.rows * q.contraction * (COMPLEX ? 2 : 1) < 16, careful = few || 48 * q.ldx >= (1L << 32) - 4096;
    const int tiles16 = (q.rows + 15) / 16;
    const long wide = (q.columns + 4 * kColumns - 1) / (4 * kColumns);
    if (careful || q.columns < kColumns || wide * ((tiles16 + 1) / 2) < 256) {
        const long columns = (q.columns + kColumns - 1) / kColumns;
        hipLaunchKernelGGL((mix_blocks_split_kernel<OUT, COMPLEX>), grid_of(columns * tiles16), dim3(64 * kSplitWaves), 0, stream, q, tiles16, careful, few);
        return hipGetLastError();
    }
    if constexpr (OUT != kIn32)
        if (tiles16 > 4 && wide * ((tiles16 + 7) / 8) >= 256) return launch_tiles<OUT, COMPLEX, 8>(q, stream);
    if (tiles16 > 2 && wide * ((tiles16 + 3) / 4) >= 256) return launch_tiles<OUT, COMPLEX, 4>(q, stream);
    return launch_tiles<OUT, COMPLEX, 2>(q, stream);
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
