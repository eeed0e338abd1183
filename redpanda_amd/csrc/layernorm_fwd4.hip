// Instantiations of layernorm_rows.h: forward, elements of 4 bytes.
#include "layernorm_rows.h"
namespace rp {
hipError_t launch_norm_fwd4(const LayerNormParams& p, unsigned wg, hipStream_t st) {
  return launch_norm_fwd_rows<4>(p, wg, st);
}
}  // namespace rp
