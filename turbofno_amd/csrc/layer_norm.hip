// Layer norm (turbofno_layer_norm): which form a call takes, and the one without dropout. The kernel is in layer_norm_strip.h.
#include "layer_norm_strip.h"

namespace tfno {

hipError_t launch_layer_norm(const LayerNormParams& q, int type, bool eight_bits, hipStream_t stream)
{
    if (q.columns == 0) return hipSuccess;
    if (eight_bits) return launch_layer_norm_8bit(q, type, stream);
    return q.drop.rng ? launch_layer_norm_dropout(q, type, stream) : launch<false, false>(q, type, stream);
}

}  // namespace tfno
