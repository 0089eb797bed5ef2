// Instances of the tiled streaming GEMV for one weight format (WF_MX4TP).
#include "bz_gemv_stream.h"

namespace bz {
int launch_stream_mx4tp(const StreamParams& p, const StreamLaunch& l, hipStream_t st) {
    return launch_stream_wf<WF_MX4TP>(p, l, st);
}
}  // namespace bz
