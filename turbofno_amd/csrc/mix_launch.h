// Launch of the channel product: which kernel runs for which sizes
#pragma once
#include "kernels.h"
#include "mix_kernel.h"
#include <algorithm>

namespace tfno {

template <int IN, int OUT, bool COMPLEX, bool GRAD, int NT> hipError_t launch_direct(const MixParams& q, hipStream_t stream)
{
    const long tiles = (q.columns + kColumns - 1) / kColumns;
    const int groups = (q.rows + 16 * NT - 1) / (16 * NT);
    const long blocks = (tiles * groups + 3) / 4;
    hipLaunchKernelGGL((mix_direct_kernel<IN, OUT, COMPLEX, GRAD, NT>), dim3((unsigned)blocks), dim3(256), 0, stream, q, groups);
    return hipGetLastError();
}

constexpr size_t kResidentLds = 152 << 10, kResidentBias = 8 << 10;    // operands of A; a bias of up to 1024 complex rows

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

template <int IN, int OUT, bool COMPLEX, bool GRAD> hipError_t launch_mix(const MixParams& q, hipStream_t stream)
{
    if (q.columns == 0) return hipSuccess;
    constexpr int CHANNELS = COMPLEX ? 16 : 32;
    const long tiles = (q.columns + kColumns - 1) / kColumns;
    const int tiles16 = (q.rows + 15) / 16, steps = (q.contraction + CHANNELS - 1) / CHANNELS;
    const size_t lds16 = (size_t)steps * kWaveParts(IN) * 1024;         // of 16 rows
    constexpr int MOST = IN == kIn32 && !COMPLEX ? 4 : 8;               // steps that registers hold
    // 32 rows at a time where 64 are too many, or where the held steps leave no registers for the sums of 64
    const bool narrow = IN == kIn32 && steps > MOST / 2 && steps <= MOST;
    const int nt = tiles16 <= 2 || narrow ? 2 : 4;
    // the lane's part of an address, up to 24 rows of the input or 12 of the results, in 32 bits
    const long widest = std::max(std::max(std::max(q.ldx, q.ldzin), q.ldr), std::max(q.ldy, q.ldz));
    const bool near = widest < (1L << 24) && tiles < (1L << 30);
    if (near && q.columns >= kColumns && tiles * tiles16 > 4096 && nt * lds16 <= kResidentLds) {
        const int groups = (tiles16 + nt - 1) / nt, fit = (int)(kResidentLds / (nt * lds16)), chunks = (groups + fit - 1) / fit;
        const int block_groups = (groups + chunks - 1) / chunks, block_rows = block_groups * nt * 16;
        const size_t lds = block_groups * nt * lds16 + block_rows * (COMPLEX ? 8 : 4);
        const long last = q.columns % kColumns;
        if (last && q.residual && (q.residual == q.y || q.residual == q.z)) {
            // the last tile would start among columns of the one before it, whose residuals may be results by then: it goes to the direct kernel
            constexpr size_t SIZE = sizeof(typename Columns<OUT>::Value);
            MixParams whole = q, rest = q;
            whole.columns = q.columns - last;
            rest.columns = last;
            auto ahead = [&](auto* p, size_t size) { return p ? decltype(p)((size_t)p + whole.columns * size) : p; };
            rest.x = ahead(q.x, sizeof(typename Columns<IN>::Value));
            rest.residual = ahead(q.residual, SIZE);
            rest.y = ahead(q.y, SIZE);
            rest.z = ahead(q.z, SIZE);
            if (q.xscale) rest.xscale = q.xscale + whole.columns / (COMPLEX ? 2 : 1);
            if (hipError_t e = launch_mix<IN, OUT, COMPLEX, GRAD>(whole, stream); e != hipSuccess) return e;
            return launch_direct<IN, OUT, COMPLEX, GRAD, 1>(rest, stream);
        }
#define TFNO_RESIDENT(NT, HELD) launch_resident<IN, OUT, COMPLEX, GRAD, NT, HELD>(q, block_rows, lds, stream)
        if (steps > MOST) return nt == 2 ? TFNO_RESIDENT(2, 0) : TFNO_RESIDENT(4, 0);
        if (steps <= 2) return nt == 2 ? TFNO_RESIDENT(2, 2) : TFNO_RESIDENT(4, 2);
        if constexpr (MOST == 8) {
            if (steps <= 4) return nt == 2 ? TFNO_RESIDENT(2, 4) : TFNO_RESIDENT(4, 4);
            if constexpr (IN == kIn32) return TFNO_RESIDENT(2, 8);
            else return nt == 2 ? TFNO_RESIDENT(2, 8) : TFNO_RESIDENT(4, 8);
        } else return TFNO_RESIDENT(2, 4);
#undef TFNO_RESIDENT
    }
    if (tiles16 == 1 || tiles * tiles16 <= 1024) return launch_direct<IN, OUT, COMPLEX, GRAD, 1>(q, stream);
    if (tiles16 == 2 || tiles * tiles16 <= 2048) return launch_direct<IN, OUT, COMPLEX, GRAD, 2>(q, stream);
    return launch_direct<IN, OUT, COMPLEX, GRAD, 4>(q, stream);
}

}  // namespace tfno
