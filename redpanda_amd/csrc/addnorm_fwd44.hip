// Instantiations of addnorm_rows.h: forward, rows of 4 bytes an element, add of 4.
#include "addnorm_rows.h"
namespace rp {
RP_ADDNORM_FWD(4, 4) { return launch_addnorm_fwd_rows<4, 4>(p, wg, st); }
}  // namespace rp
