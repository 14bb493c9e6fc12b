#include "mix_launch.h"

namespace tfno {

// type: of the result and the residual
hipError_t launch_mix_8bit(const MixParams& q, int type, hipStream_t stream)
{
    switch (type) {
    case kC64: return launch_mix<kIn8, kIn32, true, false, false>(q, stream);
    case kF32: return launch_mix<kIn8, kIn32, false, false, false>(q, stream);
    default: return launch_mix<kIn8, kIn16, false, false, false>(q, stream);
    }
}

}  // namespace tfno
