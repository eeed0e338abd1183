// Instantiations of addnorm_rows.h: forward, rows of 2 bytes an element, add of 4.
#include "addnorm_rows.h"
namespace rp {
RP_ADDNORM_FWD(2, 4) { return launch_addnorm_fwd_rows<2, 4>(p, wg, st); }
}  // namespace rp
