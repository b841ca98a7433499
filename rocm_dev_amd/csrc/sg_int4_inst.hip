// Launches of the products with 4-bit integer weights, SG_GPS groups a step of 128 columns.
#include <limits.h>

#include "sg_int4_kernel.h"

namespace sg {

// kw groups of NW waves share K
template <int FLAGS, int NF, int XU, int NW>
static int launch_build(Int4Args& a, int kw, hipStream_t stream) {
    a.n_groups = (a.tiles - 1) / (NF * NW) + 1;
    a.m_groups = (a.m - 1) / (4 * XU) + 1;
    const long long grid = (long long)a.n_groups * a.m_groups;
    if (grid > INT_MAX) return SG_BAD_ARGUMENT;
    constexpr int MF = XU < 4 ? 1 : XU / 4;
    const size_t acts = (size_t)kw * (NW > 1 ? 2 : 1) * int4_buffer(SG_GPS, XU, NW), sums = kw > 1 ? (size_t)kw * NW * NF * MF * 1024 : 0;
    const size_t lds = acts > sums ? acts : sums;
    auto* const kernel = int4_gemm_kernel<SG_GPS, FLAGS, NF, XU, NW, XU / NW <= 2 ? 4 : 2>;     // activations: 4 or 2 steps in flight
    static LdsGranted granted;
    if (int rc = request_dynamic_lds(reinterpret_cast<const void*>(kernel), lds, granted)) return rc;
    kernel<<<(unsigned)grid, 64 * kw * NW, lds, stream>>>(a);
    return report_hip("int4_gemm launch", hipGetLastError()) == hipSuccess ? SG_SUCCESS : SG_LAUNCH_FAILED;
}

template <int FLAGS>
static int launch_flags(Int4Args& a, int cu_count, hipStream_t stream) {
#ifdef SG_SWEEP
    {
        const int nf = atoi(getenv("SW_NF")), nw = atoi(getenv("SW_NW")), kw = atoi(getenv("SW_KW"));
        const int xu = a.m <= 4 ? 1 : a.m <= 8 ? 2 : a.m <= 16 ? 4 : a.m <= 32 ? 8 : 16;
#define SW(NF, XU, NW) if (nf == NF && xu == XU && nw == NW) return launch_build<FLAGS, NF, XU, NW>(a, kw, stream);
        SW(1, 1, 1) SW(2, 1, 1)  SW(1, 2, 1) SW(2, 2, 1)  SW(1, 4, 1) SW(2, 4, 1)  SW(1, 4, 2) SW(2, 4, 2) SW(1, 4, 4) SW(2, 4, 4) SW(1, 8, 2) SW(2, 8, 2) SW(1, 8, 4) SW(2, 8, 4) SW(1, 16, 2) SW(2, 16, 2) SW(1, 16, 4) SW(2, 16, 4) SW(1, 16, 8) SW(2, 16, 8) SW(1, 8, 8) SW(2, 8, 8)
        return SG_INVALID_CONFIG;
    }
#endif
    const int share = a.steps >= 16 ? 8 : a.steps >= 8 ? 4 : a.steps >= 4 ? 2 : 1;
    if (a.m <= 4) return a.tiles >= 4 * cu_count ? launch_build<FLAGS, 2, 1, 1>(a, share, stream) : launch_build<FLAGS, 1, 1, 1>(a, share, stream);
    if (a.m <= 8) return a.tiles >= 4 * cu_count ? launch_build<FLAGS, 2, 2, 1>(a, share, stream) : launch_build<FLAGS, 1, 2, 1>(a, share, stream);
    if (a.m <= 16) return a.tiles >= 4 * cu_count ? launch_build<FLAGS, 2, 4, 1>(a, share, stream) : launch_build<FLAGS, 1, 4, 1>(a, share, stream);
    if (a.m <= 32) return a.tiles >= 4 * cu_count ? launch_build<FLAGS, 2, 8, 4>(a, share < 2 ? share : 2, stream) : launch_build<FLAGS, 2, 8, 2>(a, share < 4 ? share : 4, stream);
    return a.tiles >= 4 * cu_count ? launch_build<FLAGS, 2, 16, 4>(a, share < 2 ? share : 2, stream) : launch_build<FLAGS, 2, 16, 2>(a, share < 4 ? share : 4, stream);
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
