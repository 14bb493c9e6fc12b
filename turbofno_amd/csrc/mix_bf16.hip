#include "mix_launch.h"

namespace tfno {

hipError_t launch_mix_bf16(const MixParams& q, bool grad, hipStream_t stream)
{
    return grad ? launch_mix<kIn16, kIn16, false, true>(q, stream) : launch_mix<kIn16, kIn16, false, false>(q, stream);
}

}  // namespace tfno
