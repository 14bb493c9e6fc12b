#include "mix_launch.h"

namespace tfno {

hipError_t launch_mix_c64(const MixParams& q, bool grad, hipStream_t stream)
{
    return grad ? launch_mix<kIn32, kIn32, true, true>(q, stream) : launch_mix<kIn32, kIn32, true, false>(q, stream);
}

}  // namespace tfno
