// Layer norm with its result in 8 bits (turbofno_layer_norm_8bit). The kernel is in layer_norm_strip.h.
#include "layer_norm_strip.h"

namespace tfno {

hipError_t launch_layer_norm_8bit(const LayerNormParams& q, int type, hipStream_t stream)
{
    return launch<false, true>(q, type, stream);
}

}  // namespace tfno
