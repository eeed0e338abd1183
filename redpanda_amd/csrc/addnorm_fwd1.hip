// Instantiations of addnorm_rows.h: forward, rows of 1 byte(s) an element.
#include "addnorm_rows.h"
namespace rp {
RP_ADDNORM_FWD(1) { return launch_addnorm_fwd_rows<1>(p, wg, st); }
}  // namespace rp
