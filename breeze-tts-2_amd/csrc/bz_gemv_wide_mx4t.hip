// Instances of the several-block streaming GEMV for one weight format (WF_MX4T).
#include "bz_gemv_wide.h"

namespace bz {
int launch_wide_mx4t(const StreamParams& p, const WideLaunch& l, int nblk, hipStream_t st) {
    return launch_wide_wf<WF_MX4T>(p, l, nblk, st);
}
}  // namespace bz
