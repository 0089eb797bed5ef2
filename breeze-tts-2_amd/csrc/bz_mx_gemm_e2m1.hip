// Instances of the product of microscaled rows (e2m1 elements).
#include "bz_mx_gemm.h"

namespace bz {
int launch_mx_gemm_e2m1(const MxGemmParams& p, const MxGemmLaunch& l, hipStream_t st) {
    return launch_mx_gemm_elem<BZ_MX_E2M1>(p, l, st);
}
}  // namespace bz
