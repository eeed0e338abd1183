// Instantiations of layernorm_rows.h: backward, x of 2 bytes an element, gradients of 4.
#include "layernorm_rows.h"
namespace rp {
hipError_t launch_norm_bwd24(const LayerNormParams& p, const LayerNormGrad& g, unsigned wg,
                             hipStream_t st) {
  return launch_norm_bwd_rows<2, 4>(p, g, wg, st);
}
}  // namespace rp
