// Launch of the channel product: which kernel runs for which sizes
#pragma once
#include "mix_kernel.h"

namespace tfno {

template <int IN, int OUT, bool COMPLEX, bool GRAD, int NT> hipError_t launch_direct(const MixParams& q, hipStream_t stream)
{
    const long tiles = (q.columns + kColumns - 1) / kColumns;
    const int groups = (q.rows + 16 * NT - 1) / (16 * NT);
    const long blocks = (tiles * groups + 3) / 4;
    hipLaunchKernelGGL((mix_direct_kernel<IN, OUT, COMPLEX, GRAD, NT>), dim3((unsigned)blocks), dim3(256), 0, stream, q, groups);
    return hipGetLastError();
}

template <int IN, int OUT, bool COMPLEX, bool GRAD> hipError_t launch_mix(const MixParams& q, hipStream_t stream)
{
    if (q.columns == 0) return hipSuccess;
    const long tiles = (q.columns + kColumns - 1) / kColumns;
    const int tiles16 = (q.rows + 15) / 16;
    if (tiles16 == 1 || tiles * tiles16 <= 1024) return launch_direct<IN, OUT, COMPLEX, GRAD, 1>(q, stream);
    if (tiles16 == 2 || tiles * tiles16 <= 2048) return launch_direct<IN, OUT, COMPLEX, GRAD, 2>(q, stream);
    return launch_direct<IN, OUT, COMPLEX, GRAD, 4>(q, stream);
}

}  // namespace tfno
