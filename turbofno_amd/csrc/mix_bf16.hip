#include "mix_launch.h"

namespace tfno {

hipError_t launch_mix_bf16(const MixParams& q, bool grad, hipStream_t stream)
{
    if (!grad) return launch_mix<kIn16, kIn16, false, false, false>(q, stream);
    return q.act == kActNone ? launch_mix<kIn16, kIn16, false, true, false>(q, stream) : launch_mix<kIn16, kIn16, false, true, true>(q, stream);
}

}  // namespace tfno
