// Instantiations of addnorm_rows.h: backward, rows of 4 bytes an element, gradients of 4.
#include "addnorm_rows.h"
namespace rp {
RP_ADDNORM_BWD(4, 4, 4) { return launch_addnorm_bwd_rows<4, 4, 4>(p, g, wg, st); }
}  // namespace rp
