// Launches of the products with 4-bit integer weights, SG_GPS groups a step of 128 columns.
#include <limits.h>

#include "sg_int4_kernel.h"

namespace sg {

template <int FLAGS, int NF, int XU, int NW, int DW, int MAXW, int MINB>
static int launch_build(Int4Args& a, const Int4Plan& plan, hipStream_t stream) {
    const int kw = plan.kw;
    if (kw * NW > MAXW) return SG_INVALID_CONFIG;
    a.n_groups = (a.tiles - 1) / (NF * NW) + 1;
    a.m_groups = (a.m - 1) / (4 * XU) + 1;
    const long long grid = (long long)a.n_groups * a.m_groups * a.splits;
    if (grid > INT_MAX) return SG_BAD_ARGUMENT;
    constexpr int MF = XU < 4 ? 1 : XU / 4, DX = XU / NW <= 2 && DW == 4 ? 4 : 2;      // activations: DX steps in flight
    const size_t acts = (size_t)kw * (2 * int4_buffer(SG_GPS, XU, NW) + NW * NF * 256), sums = kw > 1 ? (size_t)kw * NW * NF * MF * 1024 : 0;
    const size_t lds = acts > sums ? acts : sums;
    auto* const kernel = int4_gemm_kernel<SG_GPS, FLAGS, NF, XU, NW, DW, DX, MAXW, MINB>;
    static LdsGranted granted;
    if (int rc = request_dynamic_lds(reinterpret_cast<const void*>(kernel), lds, granted)) return rc;
    kernel<<<(unsigned)grid, 64 * kw * NW, lds, stream>>>(a);
    return report_hip("int4_gemm launch", hipGetLastError()) == hipSuccess ? SG_SUCCESS : SG_LAUNCH_FAILED;
}

// Up to 16 rows a wave has the activations to itself: one tile on up to eight waves (sixteen with four rows), or two on up to eight; four waves of
// two tiles share them where there are many tiles, in groups of 64 and 128.  Beyond, waves share them: two or four waves of a tile each, eight of one (two such
// workgroups a CU, but for 64 rows in groups of 32, which take too many registers) or two.
template <int FLAGS>
static int launch_flags(Int4Args& a, const Int4Plan& p, hipStream_t stream) {
    switch (p.xu * 100 + p.nw * 10 + p.nf) {
#define SG_ROWS(XU)                                                                    \
    case XU * 100 + 11: return launch_build<FLAGS, 1, XU, 1, 2, XU == 1 ? 16 : 8, 1>(a, p, stream); \
    case XU * 100 + 12: return launch_build<FLAGS, 2, XU, 1, 2, 8, 1>(a, p, stream);
        SG_ROWS(1) SG_ROWS(2) SG_ROWS(4)
#undef SG_ROWS
#if SG_GPS < 4
        case 442: return launch_build<FLAGS, 2, 4, 4, 4, 8, 1>(a, p, stream);
#endif
#define SG_ROWS(XU)                                                                    \
    case XU * 100 + 21: return launch_build<FLAGS, 1, XU, 2, 4, 8, 1>(a, p, stream);   \
    case XU * 100 + 41: return launch_build<FLAGS, 1, XU, 4, 4, 8, 1>(a, p, stream);   \
    case XU * 100 + 81: return launch_build<FLAGS, 1, XU, 8, 2, 8, SG_GPS == 4 && XU == 16 ? 1 : 4>(a, p, stream); \
    case XU * 100 + 82: return launch_build<FLAGS, 2, XU, 8, 4, 8, 1>(a, p, stream);
        SG_ROWS(8) SG_ROWS(16)
#undef SG_ROWS
        default: return SG_INVALID_CONFIG;
    }
}

#define SG_INT4_CAT_(a, b) a##b
#define SG_INT4_CAT(a, b) SG_INT4_CAT_(a, b)
int SG_INT4_CAT(launch_int4_, SG_GPS)(Int4Args& a, int flags, const Int4Plan& plan, hipStream_t stream) {
    switch (flags) {
        case 0: return launch_flags<0>(a, plan, stream);
        case 1: return launch_flags<1>(a, plan, stream);
        case 2: return launch_flags<2>(a, plan, stream);
        default: return launch_flags<3>(a, plan, stream);
    }
}

#if SG_GPS == 1
// The second launch of a K split: a wave adds the parts of one fragment, in their order.
__global__ void __launch_bounds__(256) int4_sum_kernel(const Int4Args a) {
    const int lane = lane_id(), m_frags = (a.m - 1) / 16 + 1;
    const size_t frags = (size_t)m_frags * a.tiles, f = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (f >= frags) return;
    const f32x4* const p = reinterpret_cast<const f32x4*>(a.ws) + f * 64 + lane;
    f32x4 t[kInt4Splits], v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < kInt4Splits; s++) t[s] = p[(size_t)(s < a.splits ? s : 0) * frags * 64];        // all in flight
#pragma unroll
    for (int s = 0; s < kInt4Splits; s++)
        if (s < a.splits) v += t[s];
    const int m_frag = (int)(f / a.tiles), tile = (int)(f - (size_t)m_frag * a.tiles);
    const int m_idx = m_frag * 16 + (lane & 15), n_idx = tile * 16 + 4 * (lane >> 4);
    if (m_idx < a.m && n_idx < a.n) int4_store4(a, m_idx, n_idx, v * kInt4OutOfUnits);
}

int launch_int4_sum(const Int4Args& a, hipStream_t stream) {
    const size_t frags = (size_t)((a.m - 1) / 16 + 1) * a.tiles;
    int4_sum_kernel<<<(unsigned)((frags + 3) / 4), 256, 0, stream>>>(a);
    return report_hip("int4_sum launch", hipGetLastError()) == hipSuccess ? SG_SUCCESS : SG_LAUNCH_FAILED;
}
#endif

}  // namespace sg
