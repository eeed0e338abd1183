// Instantiations of addnorm_rows.h: backward, rows in 8 bits, gradients of 4 and (the sum's) 2 bytes.
#include "addnorm_rows.h"
namespace rp {
RP_ADDNORM_BWD(1, 4, 2) { return launch_addnorm_bwd_rows<1, 4, 2>(p, g, wg, st); }
}  // namespace rp
