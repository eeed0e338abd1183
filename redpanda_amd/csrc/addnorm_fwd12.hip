// Instantiations of addnorm_rows.h: forward, rows in 8 bits.
#include "addnorm_rows.h"
namespace rp {
RP_ADDNORM_FWD(1, 2) { return launch_addnorm_fwd_rows<1, 2>(p, wg, st); }
}  // namespace rp
