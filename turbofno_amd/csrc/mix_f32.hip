#include "mix_launch.h"

namespace tfno {

hipError_t launch_mix_f32(const MixParams& q, bool grad, hipStream_t stream)
{
    return grad ? launch_mix<kIn32, kIn32, false, true>(q, stream) : launch_mix<kIn32, kIn32, false, false>(q, stream);
}

}  // namespace tfno
