// Launches of the products with MXFP4 weights.
#include <limits.h>

#include <type_traits>

#include "sg_mx_choice.h"
#include "sg_mx_wide_kernel.h"

namespace sg {

// Workgroup tiles of bn x bm rows, times the K splits; 0 where the grid would be too large.
static unsigned mx_grid(MxArgs& a, int bn, int bm) {
    a.n_groups = (a.tiles - 1) / (bn / 16) + 1;
    a.m_groups = (a.m - 1) / bm + 1;
    const long long grid = (long long)a.n_groups * a.m_groups * a.splits;
    return grid > INT_MAX ? 0 : (unsigned)grid;
}

template <bool FP4, int NF, int MF>
static int launch_small(MxArgs& a, int waves, hipStream_t stream) {
    const unsigned grid = mx_grid(a, 16 * NF, 16 * MF);
    if (!grid) return SG_BAD_ARGUMENT;
    const size_t lds = waves > 1 ? (size_t)waves * NF * MF * 1024 : 0;
    static LdsGranted granted;
    if (int rc = request_dynamic_lds(reinterpret_cast<const void*>(mx_gemm_kernel<FP4, NF, MF>), lds, granted)) return rc;
    mx_gemm_kernel<FP4, NF, MF><<<grid, 64 * waves, lds, stream>>>(a);
    return report_hip("mx_gemm launch", hipGetLastError()) == hipSuccess ? SG_SUCCESS : SG_LAUNCH_FAILED;
}

template <bool FP4, int NF, int MF, int WN, int WM, int WR, int XR>
static int launch_tile(MxArgs& a, hipStream_t stream) {
    const unsigned grid = mx_grid(a, 16 * NF * WN, 16 * MF * WM);
    if (!grid) return SG_BAD_ARGUMENT;
    mx_tile_kernel<FP4, NF, MF, WN, WM, WR, XR><<<grid, 64 * WN * WM, 0, stream>>>(a);
    return report_hip("mx_tile launch", hipGetLastError()) == hipSuccess ? SG_SUCCESS : SG_LAUNCH_FAILED;
}

// The wide kernel addresses rows of its tile with 32 bits.
static bool wide_takes(const MxArgs& a) { return a.k <= 1 << 22; }
// ... and reads the scales of MXFP4 activations from rows of whole groups of four steps.
static bool scales_lie_right(const MxArgs& a) { return a.k % 512 == 0 && (reinterpret_cast<uintptr_t>(a.SA) & 15u) == 0; }

template <bool FP4, int RGW, int MH, int DW, int DX>
static int launch_mx_wide(MxArgs& a, hipStream_t stream) {
    if (!wide_takes(a)) return SG_INVALID_CONFIG;
    const unsigned grid = mx_grid(a, 32 * RGW, 32 * MH);
    if (!grid) return SG_BAD_ARGUMENT;
    constexpr size_t lds = mx_wide_lds(FP4, RGW, MH, DW, DX);
    static_assert(lds <= 160 * 1024, "LDS");
    static LdsGranted granted;
    if (int rc = request_dynamic_lds(reinterpret_cast<const void*>(mx_wide_kernel<FP4, RGW, MH, DW, DX>), lds, granted)) return rc;
    mx_wide_kernel<FP4, RGW, MH, DW, DX><<<grid, 256, lds, stream>>>(a);
    return report_hip("mx_wide launch", hipGetLastError()) == hipSuccess ? SG_SUCCESS : SG_LAUNCH_FAILED;
}

// Every build, by number (include/sgemm_debug.h).
template <bool FP4>
static int launch_build(int build, MxArgs& a, hipStream_t stream) {
    const int waves = build % 100;
    if (build < 2000 && (waves < 1 || waves > 8)) return SG_INVALID_CONFIG;
    switch (build < 2000 ? build / 100 : build) {
        case 11: return launch_small<FP4, 1, 1>(a, waves, stream);   // 16 weight rows x 16 activation rows
        case 12: return launch_small<FP4, 2, 1>(a, waves, stream);   // 32 x 16
        case 13: return launch_small<FP4, 2, 2>(a, waves, stream);   // 32 x 32
        case 14: return launch_small<FP4, 1, 2>(a, waves, stream);   // 16 x 32
        case 16: return launch_small<FP4, 2, 4>(a, waves, stream);   // 32 x 64
        case 17: return launch_small<FP4, 4, 1>(a, waves, stream);   // 64 x 16
        case 2001: return launch_tile<FP4, 2, 4, 4, 2, 2, 1>(a, stream);   // 128 x 128, eight waves
        case 2005: return launch_tile<FP4, 2, 8, 4, 1, 2, 1>(a, stream);   // 128 x 128, four
        case 2010: return launch_tile<FP4, 2, 4, 4, 1, 2, 1>(a, stream);   // 128 x 64
        case 2011: return launch_tile<FP4, 2, 4, 4, 1, 4, 2>(a, stream);   // 128 x 64, deep rings (and below)
        case 2012: return launch_tile<FP4, 1, 2, 4, 1, 4, 2>(a, stream);   //  64 x 32
        case 2013: return launch_tile<FP4, 1, 4, 4, 1, 4, 2>(a, stream);   //  64 x 64
        case 2015: return launch_tile<FP4, 2, 2, 4, 1, 4, 2>(a, stream);   // 128 x 32
        case 3001: return launch_mx_wide<FP4, 8, 8, FP4 ? 2 : 3, FP4 ? 2 : 3>(a, stream);   // 256 x 256
        case 3002: return launch_mx_wide<FP4, 6, 4, 3, 3>(a, stream);                       // 192 x 128
        case 3003: return launch_mx_wide<FP4, 8, 4, 3, 3>(a, stream);                       // 256 x 128
        case 3004: return launch_mx_wide<FP4, 6, 8, 3, 2>(a, stream);                       // 192 x 256
        case 3006: return launch_mx_wide<FP4, 4, 4, 3, 3>(a, stream);                       // 128 x 128
        case 3007: return launch_mx_wide<FP4, 4, 4, 2, 2>(a, stream);                       // 128 x 128, two workgroups a CU
        default: return SG_INVALID_CONFIG;
    }
}

// The build that a call without one runs.  The search takes 0.2 to 0.9 us of host time, so a thread keeps the answers of its last
// 16 shapes - a function of the shape, of nothing else - and looks through all of them, a few ns: the shapes of a layer's projections are
// too much alike (multiples of powers of two) for a place by their value to keep them apart.
static thread_local int t_searches = 0;
int mx_searches() { return t_searches; }

static int pick_mx(bool fp4, const MxArgs& a, int cu_count, bool workspace) {
    struct Kept {
        int m, n, k, flags, build;
    };
    constexpr unsigned kKept = 16;
    static thread_local Kept kept[kKept];
    static thread_local unsigned oldest = 0;
    const bool copy = fp4 && !scales_lie_right(a);
    const int flags = 1 | (fp4 ? 2 : 0) | (copy ? 4 : 0) | (workspace ? 8 : 0) | cu_count << 4;      // (0: a place not yet taken)
    for (const Kept& e : kept)
        if (e.m == a.m && e.n == a.n && e.k == a.k && e.flags == flags) return e.build;
    t_searches++;
    Kept& e = kept[oldest++ % kKept];
    e = Kept{a.m, a.n, a.k, flags, mx_choose(fp4, a.m, a.n, a.k, cu_count, workspace, copy)};
    return e.build;
}

int mx_choice(bool fp4, int m, int n, int k, int cu_count, bool workspace) {
    return mx_choose(fp4, m, n, k, cu_count, workspace, fp4 && k % 512 != 0);
}

static int launch_mx(bool fp4, int build, MxArgs& a, hipStream_t stream);

int launch_mx_gemm(bool fp4, int build, MxArgs& a, int cu_count, hipStream_t stream) {
    if (build) return launch_mx(fp4, build, a, stream);
    build = pick_mx(fp4, a, cu_count, true);
    // A recorded launch uses no memory of the library's, so that graphs may replay side by side; a launch without device
    // memory for it runs what needs none.
    const bool shares = build >= 10000 || (fp4 && build >= 3000 && !scales_lie_right(a));
    if (shares && stream_is_capturing(stream)) return launch_mx(fp4, pick_mx(fp4, a, cu_count, false), a, stream);
    const int rc = launch_mx(fp4, build, a, stream);
    if (shares && (rc == SG_NO_DEVICE || rc == SG_WORKSPACE_TOO_SMALL)) return launch_mx(fp4, pick_mx(fp4, a, cu_count, false), a, stream);
    return rc;
}

static int launch_mx(bool fp4, int build, MxArgs& a, hipStream_t stream) {
    a.splits = 1;
    const int splits = build / 10000 < 1 ? 1 : build / 10000;
    build %= 10000;
    if (splits > a.quads) return SG_INVALID_CONFIG;
    a.SX = a.SA;
    const bool copy_scales = fp4 && build >= 3000 && !scales_lie_right(a);
    if (splits == 1 && !copy_scales) return fp4 ? launch_build<true>(build, a, stream) : launch_build<false>(build, a, stream);

    // More than one launch: the copied scales, then the partial sums, in the stream's workspace.
    std::lock_guard<std::recursive_mutex> turn(stream_turn(stream));
    const size_t frags = (size_t)((a.m - 1) / 16 + 1) * a.tiles;
    const size_t sum_grid = (frags + 3) / 4;
    const size_t pieces = copy_scales ? (size_t)a.m * a.quads : 0;
    if (sum_grid > INT_MAX || pieces > INT_MAX) return SG_BAD_ARGUMENT;
    const size_t scale_bytes = (pieces * 16 + 255) / 256 * 256;
    Workspace w;
    if (int rc = get_workspace(stream, scale_bytes + (splits > 1 ? frags * splits * 1024 : 0), 0, &w)) return rc;
    if (copy_scales) {
        uint8_t* const copy = reinterpret_cast<uint8_t*>(w.partials);
        if (int rc = launch_mx_scale_rows(a.SA, copy, a.m, a.k, a.quads, stream)) return rc;
        a.SX = copy;
    }
    a.splits = splits;
    a.ws = w.partials + scale_bytes / 4;
    if (int rc = fp4 ? launch_build<true>(build, a, stream) : launch_build<false>(build, a, stream)) return rc;
    if (splits == 1) return SG_SUCCESS;
    mx_sum_kernel<<<(unsigned)sum_grid, 256, 0, stream>>>(a);
    return report_hip("mx_sum launch", hipGetLastError()) == hipSuccess ? SG_SUCCESS : SG_LAUNCH_FAILED;
}

}  // namespace sg
