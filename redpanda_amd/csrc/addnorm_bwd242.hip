// Instantiations of addnorm_rows.h: backward, rows of 2 bytes an element, gradients of 4.
#include "addnorm_rows.h"
namespace rp {
RP_ADDNORM_BWD(2, 4, 2) { return launch_addnorm_bwd_rows<2, 4, 2>(p, g, wg, st); }
}  // namespace rp
