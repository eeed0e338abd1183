// Instantiations of addnorm_rows.h: backward, rows in 8 bits, gradients of 2 and (the sum's) 4 bytes.
#include "addnorm_rows.h"
namespace rp {
RP_ADDNORM_BWD(1, 2, 4) { return launch_addnorm_bwd_rows<1, 2, 4>(p, g, wg, st); }
}  // namespace rp
