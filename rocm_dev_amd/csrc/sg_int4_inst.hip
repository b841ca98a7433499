// Launches of the products with 4-bit integer weights, SG_GPS groups a step of 128 columns.
#include <limits.h>

#include <type_traits>

#include "sg_int4_kernel.h"

namespace sg {

template <int FLAGS, int NF, int MF, int DEPTH>
static int launch_build(Int4Args& a, int waves, hipStream_t stream) {
    a.n_groups = (a.tiles - 1) / NF + 1;
    a.m_groups = (a.m - 1) / (16 * MF) + 1;
    const long long grid = (long long)a.n_groups * a.m_groups;
    if (grid > INT_MAX) return SG_BAD_ARGUMENT;
    const size_t lds = waves > 1 ? (size_t)waves * NF * MF * 1024 : 0;
    auto* const kernel = int4_gemm_kernel<SG_GPS, FLAGS, NF, MF, DEPTH>;
    static LdsGranted granted;
    if (int rc = request_dynamic_lds(reinterpret_cast<const void*>(kernel), lds, granted)) return rc;
    kernel<<<(unsigned)grid, 64 * waves, lds, stream>>>(a);
    return report_hip("int4_gemm launch", hipGetLastError()) == hipSuccess ? SG_SUCCESS : SG_LAUNCH_FAILED;
}

template <int FLAGS>
static int launch_flags(Int4Args& a, int cu_count, hipStream_t stream) {
    (void)cu_count;
    const int waves = a.steps >= 16 ? 8 : a.steps >= 8 ? 4 : a.steps >= 4 ? 2 : 1;
    if (a.m <= 16) return launch_build<FLAGS, 2, 1, 2>(a, waves, stream);
    if (a.m <= 32) return launch_build<FLAGS, 2, 2, 2>(a, waves, stream);
    return launch_build<FLAGS, 2, 4, 1>(a, waves, stream);
}

#define SG_INT4_CAT_(a, b) a##b
#define SG_INT4_CAT(a, b) SG_INT4_CAT_(a, b)
int SG_INT4_CAT(launch_int4_, SG_GPS)(Int4Args& a, int flags, int cu_count, hipStream_t stream) {
    switch (flags) {
        case 0: return launch_flags<0>(a, cu_count, stream);
        case 1: return launch_flags<1>(a, cu_count, stream);
        case 2: return launch_flags<2>(a, cu_count, stream);
        default: return launch_flags<3>(a, cu_count, stream);
    }
}

}  // namespace sg
