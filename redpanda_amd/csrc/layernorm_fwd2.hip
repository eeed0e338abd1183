// Instantiations of layernorm_rows.h: forward, elements of 2 bytes.
#include "layernorm_rows.h"
namespace rp {
hipError_t launch_norm_fwd2(const LayerNormParams& p, unsigned wg, hipStream_t st) {
  return launch_norm_fwd_rows<2>(p, wg, st);
}
}  // namespace rp
