// Instantiations of addnorm_rows.h: forward, rows of 4 byte(s) an element.
#include "addnorm_rows.h"
namespace rp {
RP_ADDNORM_FWD(4) { return launch_addnorm_fwd_rows<4>(p, wg, st); }
}  // namespace rp
