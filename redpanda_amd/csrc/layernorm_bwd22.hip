// Instantiations of layernorm_rows.h: backward, x of 2 bytes an element, gradients of 2.
#include "layernorm_rows.h"
namespace rp {
hipError_t launch_norm_bwd22(const LayerNormParams& p, const LayerNormGrad& g, unsigned wg,
                             hipStream_t st) {
  return launch_norm_bwd_rows<2, 2>(p, g, wg, st);
}
}  // namespace rp
