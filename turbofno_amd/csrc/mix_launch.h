// Launch of the channel product: which kernel runs for which sizes
#pragma once
#include "kernels.h"
#include "mix_kernel.h"
#include <algorithm>

namespace tfno {

template <int IN, int OUT, bool COMPLEX, bool GRAD, int NT, bool RAGGED, bool FEW> hipError_t launch_direct(const MixParams& q, hipStream_t stream)
{
    const long tiles = (q.columns + kColumns - 1) / kColumns;
    const int groups = (q.rows + 16 * NT - 1) / (16 * NT);
    const long blocks = (tiles * groups + 3) / 4;
    hipLaunchKernelGGL((mix_direct_kernel<IN, OUT, COMPLEX, GRAD, NT, RAGGED, FEW>), dim3((unsigned)blocks), dim3(256), 0, stream, q, groups);
    return hipGetLastError();
}

constexpr size_t kResidentLds = 152 << 10, kResidentBias = 8 << 10;    // operands of A; bias and scales of up to 640 complex rows

template <int IN, int OUT, bool COMPLEX, bool GRAD, int NT, int HELD> hipError_t launch_resident(const MixParams& q, int block_rows, size_t lds, hipStream_t stream)
{
    static std::atomic<unsigned long long> served{ 0 };
    if (hipError_t e = allow_dynamic_lds(reinterpret_cast<const void*>(mix_resident_kernel<IN, OUT, COMPLEX, GRAD, NT, HELD>), kResidentLds + kResidentBias, served); e != hipSuccess)
        return e;
    const long tiles = (q.columns + kColumns - 1) / kColumns;
    const int chunks = (q.rows + block_rows - 1) / block_rows;
    int threads = lds > (kResidentLds / 2) ? 512 : 256;
    const long most = cu_count() * (512 / threads) / chunks, want = (tiles + threads / 64 - 1) / (threads / 64);
    const long blocks = want < most ? want : most > 0 ? most : 1;
    hipLaunchKernelGGL((mix_resident_kernel<IN, OUT, COMPLEX, GRAD, NT, HELD>), dim3((unsigned)blocks, (unsigned)chunks), dim3(threads), lds, stream, q,
                       block_rows, (int)tiles);
    return hipGetLastError();
}

// Up to this many tiles of 64 columns x 16 rows a wave of the direct kernel takes one of them: the resident one would form its operands of A on few CUs
// first. complex64, gelu, residual: 64 to 64 channels at 200 ... 4096 positions 7.4 ... 7.7 us, 12.2 ... 12.6 in the resident one; 128 to 128 at
// 4096 13.2 and 14.2; bf16, 256 to 256 at 4096 11.4 and 13.7. Above, the operands are formed once for all tiles of a block.
constexpr long kFewTiles = 1024;
// Fewer tiles than this number of waves (of 256 CUs): the rows of A are divided too
constexpr long kWaves = 2048;

// steps that registers hold, and beyond how many of them the sums of 64 rows find no room beside them
template <int IN, bool COMPLEX> constexpr int kMostSteps = IN == kIn32 && !COMPLEX ? 4 : 8;
template <int IN, int OUT, bool COMPLEX> constexpr int kMostWideSteps = IN == kIn32 ? (COMPLEX ? 4 : 2) : OUT == kIn32 ? 4 : 8;

template <int IN, int OUT, bool COMPLEX, bool GRAD, int HELD = kMostSteps<IN, COMPLEX>>
hipError_t launch_steps(const MixParams& q, int nt, int held, int block_rows, size_t lds, hipStream_t stream)
{
    if constexpr (HELD != held_for(HELD)) return launch_steps<IN, OUT, COMPLEX, GRAD, HELD - 1>(q, nt, held, block_rows, lds, stream);
    else {
        if (held == HELD) {
            if constexpr (HELD <= kMostWideSteps<IN, OUT, COMPLEX>)
                if (nt == 4) return launch_resident<IN, OUT, COMPLEX, GRAD, 4, HELD>(q, block_rows, lds, stream);
            return launch_resident<IN, OUT, COMPLEX, GRAD, 2, HELD>(q, block_rows, lds, stream);
        }
        if constexpr (HELD > 0) return launch_steps<IN, OUT, COMPLEX, GRAD, HELD - 1>(q, nt, held, block_rows, lds, stream);
        else return hipErrorInvalidValue;
    }
}

template <int IN, int OUT, bool COMPLEX, bool GRAD> hipError_t launch_mix(const MixParams& q, hipStream_t stream)
{
    if (q.columns == 0) return hipSuccess;
    // Columns that do not fill a tile: the last tile ends with them, among columns of the one before it. Where those may be results by then (the residuals
    // are in their place), and where there are no others, a kernel takes them one by one
    const long last = q.columns % kColumns, head = q.columns - last;
    if (last && head == 0) return launch_direct<IN, OUT, COMPLEX, GRAD, 1, true, !GRAD>(q, stream);
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
        if (hipError_t e = launch_mix<IN, OUT, COMPLEX, GRAD>(whole, stream); e != hipSuccess) return e;
        return launch_direct<IN, OUT, COMPLEX, GRAD, 1, true, !GRAD>(rest, stream);
    }
    if constexpr (!GRAD)        // weights that cannot be read by eight
        if (((long)(q.rows - 1) * q.ldw + q.contraction) * (COMPLEX ? 2 : 1) < 8) return launch_direct<IN, OUT, COMPLEX, GRAD, 1, false, true>(q, stream);
    constexpr int CHANNELS = COMPLEX ? 16 : 32;
    const long tiles = (q.columns + kColumns - 1) / kColumns;
    const int tiles16 = (q.rows + 15) / 16, steps = (q.contraction + CHANNELS - 1) / CHANNELS;
    // gradients of 32-bit real rows with three or four steps are streamed in 64 rows instead of held in 32: the slopes are formed half as often
    // (128 to 128 channels at 262144 positions, both gradients: 252 us, 264 held; 256 to 120 at 65536: 104 and 124)
    const bool held = steps <= kMostSteps<IN, COMPLEX> && !(GRAD && IN == kIn32 && !COMPLEX && steps > 2);
    const size_t lds16 = (size_t)(held ? held_for(steps) : steps) * kWaveParts(IN) * 1024;     // of 16 rows
    const int nt = tiles16 <= 2 || (held && steps > kMostWideSteps<IN, OUT, COMPLEX>) ? 2 : 4;
    // the lane's part of an address, up to 24 rows of the input or 12 of the results, in 32 bits
    const long widest = std::max(std::max(std::max(q.ldx, q.ldzin), q.ldr), std::max(q.ldy, q.ldz));
    const bool near = widest < (1L << 24) && tiles < (1L << 30);
    if (near && tiles * tiles16 > kFewTiles && nt * lds16 <= kResidentLds) {
        const int groups = (tiles16 + nt - 1) / nt, fit = std::min((int)(kResidentLds / (nt * lds16)), 640 / (16 * nt));
        int chunks = (groups + fit - 1) / fit;
        while (chunks < groups && tiles * chunks < kWaves) ++chunks;
        if (GRAD && IN == kIn32) chunks = groups;       // the kernel walks 64 rows: what it made of gy and z is gone after them
        const int block_groups = (groups + chunks - 1) / chunks, block_rows = block_groups * nt * 16;
        const size_t lds = block_groups * nt * lds16 + block_rows * ((COMPLEX ? 8 : 4) + (IN == kIn8 ? 4 : 0));
        return launch_steps<IN, OUT, COMPLEX, GRAD>(q, nt, held ? held_for(steps) : 0, block_rows, lds, stream);
    }
    if (tiles16 == 1 || tiles * tiles16 <= 1024) return launch_direct<IN, OUT, COMPLEX, GRAD, 1, false, false>(q, stream);
    if (tiles16 == 2 || tiles * tiles16 <= 2048) return launch_direct<IN, OUT, COMPLEX, GRAD, 2, false, false>(q, stream);
    return launch_direct<IN, OUT, COMPLEX, GRAD, 4, false, false>(q, stream);
}

}  // namespace tfno
