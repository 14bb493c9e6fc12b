#include "mix_launch.h"

namespace tfno {

hipError_t launch_mix_c64(const MixParams& q, bool grad, hipStream_t stream)
{
    if (!grad) return launch_mix<kIn32, kIn32, true, false, false>(q, stream);
    return q.act == kActNone ? launch_mix<kIn32, kIn32, true, true, false>(q, stream) : launch_mix<kIn32, kIn32, true, true, true>(q, stream);
}

}  // namespace tfno
