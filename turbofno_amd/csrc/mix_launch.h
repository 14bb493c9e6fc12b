// Launch of the channel product: which kernel runs for which sizes
#pragma once
#include "kernels.h"
#include "mix_kernel.h"
#include <algorithm>

namespace tfno {

template <int IN, int OUT, bool COMPLEX, bool GRAD, bool SLOPES, int NT, bool RAGGED, bool FEW> hipError_t launch_direct(const MixParams& q, hipStream_t stream)
{
    const long tiles = (q.columns + kColumns - 1) / kColumns;
    const int groups = (q.rows + 16 * NT - 1) / (16 * NT);
    const long blocks = (tiles * groups + 3) / 4;
    hipLaunchKernelGGL((mix_direct_kernel<IN, OUT, COMPLEX, GRAD, SLOPES, NT, RAGGED, FEW>), grid_of(blocks), dim3(256), 0, stream, q, groups);
    return hipGetLastError();
}

constexpr size_t kResidentLds = 152 << 10, kResidentBias = 8 << 10;    // operands of A; bias and scales of up to 640 complex rows

template <int IN, int OUT, bool COMPLEX, bool GRAD, bool SLOPES, int NT, int HELD> hipError_t launch_resident(const MixParams& q, int block_rows, size_t lds, hipStream_t stream)
{
    static std::atomic<unsigned long long> served{ 0 };
    if (hipError_t e = allow_dynamic_lds(reinterpret_cast<const void*>(mix_resident_kernel<IN, OUT, COMPLEX, GRAD, SLOPES, NT, HELD>), kResidentLds + kResidentBias, served); e != hipSuccess)
        return e;
    const long tiles = (q.columns + kColumns - 1) / kColumns;
    const int chunks = (q.rows + block_rows - 1) / block_rows;
    // two blocks of 256 threads on a CU where their operands fit, one of 512 otherwise (float32, 64 to 64 channels at 262144 positions: 48 us, 50 with 512)
    const int threads = lds > (kResidentLds / 2) ? 512 : 256;
    const long most = cu_count() * (512 / threads) / chunks, want = (tiles + threads / 64 - 1) / (threads / 64);
    const long blocks = want < most ? want : most > 0 ? most : 1;
    hipLaunchKernelGGL((mix_resident_kernel<IN, OUT, COMPLEX, GRAD, SLOPES, NT, HELD>), dim3((unsigned)blocks, (unsigned)chunks), dim3(threads), lds, stream, q,
                       block_rows, (int)tiles);
    return hipGetLastError();
}

// Up to this many tiles of 64 columns x 16 rows a wave of the direct kernel takes one of them: the resident one would form its operands of A on few CUs
// first. complex64, gelu, residual: 64 to 64 channels at 200 ... 4096 positions 7.4 ... 7.7 us, 12.2 ... 12.6 in the resident one; 128 to 128 at
// 4096 13.2 and 14.2; bf16, 256 to 256 at 4096 11.4 and 13.7. Above, the operands are formed once for all tiles of a block.
constexpr long kFewTiles = 1024;
// Fewer tiles than this number of waves (eight on each of 256 CUs): the rows of A are divided too. bf16, 256 to 256 channels at 20000 positions: 17 us, 33 with all
// rows in every block; complex64, 128 to 256 at 10000: 25 and 39.
constexpr long kWaves = 2048;

// steps that registers hold, and beyond how many of them the sums of 64 rows find no room beside them
template <int IN> constexpr int kMostSteps = IN == kIn32 ? 1 : 8;
template <int IN, int OUT> constexpr int kMostWideSteps = OUT == kIn32 ? 4 : 8;

template <int IN, int OUT, bool COMPLEX, bool GRAD, bool SLOPES, int HELD = kMostSteps<IN>>
hipError_t launch_steps(const MixParams& q, int nt, int held, int block_rows, size_t lds, hipStream_t stream)
{
    if constexpr (HELD != held_for(HELD)) return launch_steps<IN, OUT, COMPLEX, GRAD, SLOPES, HELD - 1>(q, nt, held, block_rows, lds, stream);
    else {
        if (held == HELD) {
            if constexpr (HELD <= kMostWideSteps<IN, OUT>)
                if (nt == 4) return launch_resident<IN, OUT, COMPLEX, GRAD, SLOPES, 4, HELD>(q, block_rows, lds, stream);
            if constexpr (HELD <= 1 || HELD > kMostWideSteps<IN, OUT>)     // up to 32 rows are walked once, and more steps than one streamed
                if (nt == 2) return launch_resident<IN, OUT, COMPLEX, GRAD, SLOPES, 2, HELD>(q, block_rows, lds, stream);
            return hipErrorInvalidValue;
        }
        if constexpr (HELD > 0) return launch_steps<IN, OUT, COMPLEX, GRAD, SLOPES, HELD - 1>(q, nt, held, block_rows, lds, stream);
        else return hipErrorInvalidValue;
    }
}

// From this number of blocks or waves that would form the slopes of the same columns, gz is formed by a kernel of its own and the product reads it. Both gradients, gelu:
// complex64, 256 to 256 channels at 65536 positions 422 us, 467 in one kernel; float32, 128 to 512 at 65536 203 and 229; bf16, 128 to 1300 at 20000 107 and
// 163, 128 to 128 at 30000 28.4 and 30.5. Two in 32 bits: complex64, 128 to 128 at 65536 135 us, 131 in one kernel.
template <int IN> constexpr int kSlopesApart = IN == kIn32 ? 3 : 2;
template <int IN, int OUT, bool COMPLEX, bool GRAD, bool SLOPES> hipError_t launch_mix(const MixParams& q, hipStream_t stream);

// The gradient in two kernels: gz, then the product
template <int IN, int OUT, bool COMPLEX> hipError_t launch_slopes(const MixParams& q, hipStream_t stream)
{
    const long of_row = (q.columns + 2047) / 2048, units = of_row * q.contraction, most = 8l * cu_count();
    hipLaunchKernelGGL(slope_kernel<IN>, dim3((unsigned)(units < most ? units : most)), dim3(256), 0, stream, q, units, of_row);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    MixParams rest = q;
    rest.x = q.z;
    rest.ldx = q.ldz;
    rest.zin = nullptr;
    rest.z = nullptr;
    rest.ldz = rest.ldzin = 0;
    rest.act = kActNone;
    return launch_mix<IN, OUT, COMPLEX, true, false>(rest, stream);
}

template <int IN, int OUT, bool COMPLEX, bool GRAD, bool SLOPES> hipError_t launch_mix(const MixParams& q, hipStream_t stream)
{
    if (q.columns == 0) return hipSuccess;
    // Columns that do not fill a tile: the last tile ends with them, among columns of the one before it. Where those may be results by then (the residuals
    // are in their place), and where there are no others, a kernel takes them one by one
    const long last = q.columns % kColumns, head = q.columns - last;
    if (last && head == 0) return launch_direct<IN, OUT, COMPLEX, GRAD, SLOPES, 1, true, !GRAD>(q, stream);
    if (last && q.residual && (q.residual == q.y || q.residual == q.z)) {
        constexpr size_t SIZE = sizeof(typename Columns<OUT>::Value);
        MixParams whole = q, rest = q;
        whole.columns = head;
        rest.columns = last;
        auto ahead = [&](auto* p, size_t size) { return p ? decltype(p)((size_t)p + head * size) : p; };
        rest.x = ahead(q.x, sizeof(typename Columns<IN>::Value));
        rest.residual = ahead(q.residual, SIZE);
        rest.y = ahead(q.y, SIZE);
        rest.z = ahead(q.z, SIZE);
        if (q.xscale) rest.xscale = q.xscale + head / (COMPLEX ? 2 : 1);
        if (hipError_t e = launch_mix<IN, OUT, COMPLEX, GRAD, SLOPES>(whole, stream); e != hipSuccess) return e;
        return launch_direct<IN, OUT, COMPLEX, GRAD, SLOPES, 1, true, !GRAD>(rest, stream);
    }
    if constexpr (!GRAD)        // weights that cannot be read by eight
        if (((long)(q.rows - 1) * q.ldw + q.contraction) * (COMPLEX ? 2 : 1) < 8) return launch_direct<IN, OUT, COMPLEX, GRAD, SLOPES, 1, false, true>(q, stream);
    constexpr int CHANNELS = COMPLEX ? 16 : 32;
    const long tiles = (q.columns + kColumns - 1) / kColumns;
    const int tiles16 = (q.rows + 15) / 16, steps = (q.contraction + CHANNELS - 1) / CHANNELS;
    // a lane's part of an address in 32 bits: up to 24 (complex: 12) rows of the input and 64 columns, up to 12 rows of the results
    const long in_rows = (COMPLEX ? 12 : 24) * std::max(std::max(q.ldx, q.ldzin), GRAD ? q.ldz : 0), out_rows = 12 * std::max(q.ldr, std::max(q.ldy, q.ldz));
    const bool near = std::max(in_rows * (long)sizeof(typename Columns<IN>::Value), out_rows * (long)sizeof(typename Columns<OUT>::Value)) < (1L << 32) - 4096 &&
                      tiles < (1L << 30);
    struct Plan {
        int nt, block_rows, groups;                     // 16 rows at a time; rows of a block, and how often it walks its columns for them
        size_t lds16;                                   // operands of 16 rows
    };
    auto plan = [&](bool held) {
        Plan p;
        p.lds16 = (size_t)(held ? held_for(steps) : steps) * kWaveParts(IN) * 1024;
        p.nt = tiles16 <= 2 || (held && steps > kMostWideSteps<IN, OUT>) ? 2 : 4;
        // 32 rows where the operands of 64 do not fit (complex64, 256 to 256 channels with residual at 65536 positions: 203 us, 221 in the direct kernel; both
        // gradients, float32, 64 to 512 at 65536: 141 and 173; bf16, 64 to 1300 at 30000: 115 and 148; complex64, 64 to 256 at 65536: 159 - 165 and 156)
        if (p.nt * p.lds16 > kResidentLds) p.nt = 2;
        if (p.nt * p.lds16 > kResidentLds) return p.groups = 0, p;
        const int groups = (tiles16 + p.nt - 1) / p.nt, fit = std::min((int)(kResidentLds / (p.nt * p.lds16)), 640 / (16 * p.nt));
        int chunks = (groups + fit - 1) / fit;
        while (chunks < groups && tiles * chunks < kWaves) ++chunks;
        // 64 rows per block: walking the columns again would form the slopes again in the same wave (float32, 128 to 128 channels, both gradients at
        // 262144 positions: 236 us, 253 with all rows in one block)
        if (SLOPES && IN == kIn32) chunks = groups;
        p.groups = (groups + chunks - 1) / chunks;
        p.block_rows = p.groups * p.nt * 16;
        return p;
    };
    if (near && tiles * tiles16 > kFewTiles) {
        Plan p = plan(false);
        // Steps are held where 16- or 8-bit columns are walked more than once (bf16, 72 to 200 channels at 100003 positions: 24.3 us, streamed 27.6; 8 bits, 256
        // to 256 at 262144: 81 and 105), and a single one. Otherwise they are streamed: the first products do not wait for the last rows, and 32-bit
        // operands would have to be formed again all the same (complex64, 128 to 128 at 262144: 212 us, held 244; bf16, 256 to 256 at 20000: 17.4 and 20.8)
        const bool held = steps == 1 || (IN != kIn32 && p.groups > 1 && steps <= kMostSteps<IN>);
        if (held) p = plan(true);
        const size_t lds = p.block_rows / 16 * p.lds16 + p.block_rows * ((COMPLEX ? 8 : 4) + (IN == kIn8 ? 4 : 0)) + (IN == kIn32 ? 32 : 0);
        if constexpr (SLOPES)
            if (p.groups && (tiles16 + p.nt * p.groups - 1) / (p.nt * p.groups) >= kSlopesApart<IN>) return launch_slopes<IN, OUT, COMPLEX>(q, stream);
        if (p.groups) return launch_steps<IN, OUT, COMPLEX, GRAD, SLOPES>(q, p.nt, held ? held_for(steps) : 0, p.block_rows, lds, stream);
    }
    if (tiles16 == 1 || tiles * tiles16 <= 1024) return launch_direct<IN, OUT, COMPLEX, GRAD, SLOPES, 1, false, false>(q, stream);
    if constexpr (SLOPES)
        if (tiles * tiles16 > kFewTiles && tiles16 > 4 * (kSlopesApart<IN> - 1)) return launch_slopes<IN, OUT, COMPLEX>(q, stream);
    if constexpr (!(SLOPES && IN == kIn32 && !COMPLEX))     // two steps of gy and of z leave no registers for 64 rows of sums there
        if (tiles16 > 2 && tiles * tiles16 > 2048) return launch_direct<IN, OUT, COMPLEX, GRAD, SLOPES, 4, false, false>(q, stream);
    return launch_direct<IN, OUT, COMPLEX, GRAD, SLOPES, 2, false, false>(q, stream);
}

}  // namespace tfno
