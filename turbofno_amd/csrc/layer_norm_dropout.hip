// Layer norm with dropout of x. The kernel is in layer_norm_strip.h.
#include "layer_norm_strip.h"

namespace tfno {

hipError_t launch_layer_norm_dropout(const LayerNormParams& q, int type, hipStream_t stream)
{
    return launch<true, false>(q, type, stream);
}

}  // namespace tfno
