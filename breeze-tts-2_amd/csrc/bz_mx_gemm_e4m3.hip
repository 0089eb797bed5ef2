// Instances of the product of microscaled rows (e4m3 elements).
#include "bz_mx_gemm.h"

namespace bz {
int launch_mx_gemm_e4m3(const MxGemmParams& p, const MxGemmLaunch& l, hipStream_t st) {
    return launch_mx_gemm_elem<BZ_MX_E4M3>(p, l, st);
}
}  // namespace bz
