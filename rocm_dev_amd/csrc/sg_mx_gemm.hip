// Launches of the products with MXFP4 weights.
#include <limits.h>

#include <type_traits>

#include "sg_mx_kernel.h"

namespace sg {

template <bool FP4, int NF, int MF>
static int launch_small(MxArgs& a, int waves, hipStream_t stream) {
    a.n_groups = (a.tiles + NF - 1) / NF;
    a.m_groups = (int)(((unsigned)a.m + 16 * MF - 1) / (16 * MF));
    const long long grid = (long long)a.n_groups * a.m_groups;
    if (grid > INT_MAX) return SG_BAD_ARGUMENT;
    const size_t lds = waves > 1 ? (size_t)waves * NF * MF * 1024 : 0;
    static LdsGranted granted;
    if (int rc = request_dynamic_lds(reinterpret_cast<const void*>(mx_gemm_kernel<FP4, NF, MF>), lds, granted)) return rc;
    mx_gemm_kernel<FP4, NF, MF><<<(unsigned)grid, 64 * waves, lds, stream>>>(a);
    return report_hip("mx_gemm launch", hipGetLastError()) == hipSuccess ? SG_SUCCESS : SG_LAUNCH_FAILED;
}

template <bool FP4>
static int launch_any(MxArgs& a, int cu_count, hipStream_t stream) {
    const int most = a.quads < 8 ? a.quads : 8;      // waves that have a share of K
    if (a.m <= 16) return launch_small<FP4, 1, 1>(a, most, stream);
    return launch_small<FP4, 2, 2>(a, most, stream);
}

int launch_mx_gemm(bool fp4, MxArgs& a, int cu_count, hipStream_t stream) {
    return fp4 ? launch_any<true>(a, cu_count, stream) : launch_any<false>(a, cu_count, stream);
}

}  // namespace sg
