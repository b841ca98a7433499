// 4-bit integer weights with group scales: packing, launches and C entry points (include/sgemm.h).
#include "sg_int4.h"

namespace sg {

struct Int4PackArgs {
    const uint8_t* B;
    const uint16_t* scales;
    const uint8_t* zeros;            // or NULL
    uint8_t* P;
    uint16_t* PS;
    uint8_t* PZ;
    int n, k, group, b_stride;
    int tiles, steps, gps;
};

// A thread a lane of a step of a tile: its four dwords, and the scales and zeros of one of the tile's groups each for the first 16 * gps lanes.
__global__ void __launch_bounds__(256) int4_pack_kernel(const Int4PackArgs a) {
    const size_t at = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (at >= (size_t)a.tiles * a.steps) return;
    const int tile = (int)(at / a.steps), step = (int)(at - (size_t)tile * a.steps);
    const int lane = lane_id(), row = tile * 16 + (lane & 15), g = lane >> 4;
    u32x4 out = {0, 0, 0, 0};
    if (row < a.n) {
        const uint8_t* const b = a.B + (size_t)row * a.b_stride;
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const int col = 128 * step + 32 * t + 8 * g;
            if (col >= a.k) continue;                                  // (k is a multiple of 32)
            const uint32_t d = *reinterpret_cast<const uint32_t*>(b + col / 2);
            uint32_t o = 0;
#pragma unroll
            for (int p = 0; p < 4; p++) {
                const uint32_t lo = (d >> (8 * p)) & 15u, hi = (d >> (8 * p + 4)) & 15u;
                o |= lo << (3 + 4 * p);
                o |= p < 3 ? hi << (19 + 4 * p) : hi << 31 | hi >> 1;
            }
            out[t] = o;
        }
    }
    reinterpret_cast<u32x4*>(a.P)[at * 64 + lane] = out;
    const int gps = a.gps;
    if (lane >= 16 * gps) return;
    // group q of the step, row `in` of the tile: [4][gps][4]
    const int q = lane >> 4, in = lane & 15, groups = a.k / a.group;
    const int n_idx = tile * 16 + in, group = step * gps + q;
    const bool inside = n_idx < a.n && group < groups;
    const size_t to = (at * 4 + (in >> 2)) * gps * 4 + q * 4 + (in & 3), from = (size_t)n_idx * groups + group;
    a.PS[to] = inside ? a.scales[from] : (uint16_t)0;
    if (a.zeros) a.PZ[to] = inside ? a.zeros[from] : (uint8_t)0;
}

// The build, its waves and its K splits by the shape; us below are of one MI355X, medians of graph replays on cold weights.
//
// Up to 16 rows: one tile a wave where there are at most as many tiles as CUs (13 rows of 3712 x 10944, groups of 32, 11.4; two tiles 14.7), or up to
// three times as many and at most eight rows (1 x 11008 x 4096 7.5, two 8.0; 13 rows 11.4, 9.9), two elsewhere (5 x 28672 x 4096 15.1,
// one 15.6), on as many waves as leave each a few steps: 1 x 3712 x 10944, groups of 64, sixteen 8.1, eight 9.8; 1 x 6144 x 4096 eight
// 5.8, four 6.6, two 9.5; 1 x 28672 x 4096 two 13.9, four 14.8, eight 15.7, in groups of 32 19.2, 17.9, 19.5.  With more than eight rows and
// many tiles the activations are what goes to a CU most: four waves share them (13 x 28672 x 4096 14.6, each its own 16.3), but not
// in groups of 32 (19.3 and 19.8, 57344 x 8192 67.5 and 63.1).  K splits where idle CUs can take them and the steps that a
// wave has left outweigh the second launch: 1 x 1024 x 32768 14.3 -> 9.8, 8 x 512 x 16384 10.9 -> 7.3.
//
// Beyond, the waves' vector and matrix units bound what a workgroup does, so that its time is its steps times that of one, and a product's
// that of its rounds of workgroups.  The four ways - two or four waves of one tile and groups of them that share K, eight of one tile, eight
// of two - and their K splits are compared by that.  64 rows, groups of 64: 57344 x 8192 101 (two tiles on eight waves; twice that on two waves of one),
// 10240 x 8192 32 with the splits' second launch (the same, six splits; unsplit 38 on four waves), 8192 x 8192 26 (30), 8192 x 28672 54
// (eight splits; unsplit 91).
Int4Plan int4_plan(const Int4Args& a, int group, int cu_count, bool workspace) {
    Int4Plan p{1, a.m <= 4 ? 1 : a.m <= 8 ? 2 : a.m <= 16 ? 4 : a.m <= 32 ? 8 : 16, 1, 1, 1};
    if (p.xu <= 4) {
        p.nf = a.tiles <= cu_count || (p.xu < 4 && a.tiles > 2 * cu_count && a.tiles <= 3 * cu_count) ? 1 : 2;
        const int groups = (a.tiles - 1) / p.nf + 1;
        if (groups <= cu_count) p.kw = p.nf == 1 && p.xu == 1 && a.steps >= 32 ? 16 : 8;
        else if (p.nf == 1 || groups <= 2 * cu_count) p.kw = 4;
        else if (p.xu == 4 && group >= 64) p.nw = 4, p.kw = 2;
        else p.kw = a.steps >= 48 || (group == 32 && p.xu < 4) ? 4 : 2;
        while (p.kw > a.steps) p.kw /= 2;
        if (!workspace || 2 * groups > cu_count) return p;
        const int splits = cu_count / groups < kInt4Splits ? cu_count / groups : kInt4Splits;
        const float left = (float)a.steps / p.kw, a_step = p.xu == 4 ? 0.7f : 0.45f;
        if (left * a_step * (1.0f - 1.0f / splits) > 3.5f) p.splits = splits;
        return p;
    }
    struct Way {
        int nf, nw, kw, at_once;     // workgroups a CU
        float a_step[2];             // us of a step of a workgroup, up to 32 and up to 64 rows, with all of a CU's
    };
    static constexpr Way ways[] = {{1, 2, 4, 1, {1.28f, 2.0f}}, {1, 4, 2, 1, {0.84f, 1.2f}}, {1, 8, 1, 2, {1.14f, 1.64f}}, {2, 8, 1, 1, {1.1f, 1.53f}}};
    const int m_groups = (a.m - 1) / (4 * p.xu) + 1;
    float best = 0.0f;
    for (const Way& w : ways) {
        const long long groups = (long long)((a.tiles - 1) / (w.nf * w.nw) + 1) * m_groups;
        const int at_once = group == 32 && p.xu == 16 ? 1 : w.at_once;
        int kw = w.kw;
        while (kw > a.steps) kw /= 2;
        for (int splits = 1; splits <= (workspace ? kInt4Splits : 1) && splits * kw <= a.steps; splits++) {
            const long long all = groups * splits, slots = (long long)at_once * cu_count;
            // a workgroup alone on its CU is through sooner than two
            const float a_step = w.a_step[p.xu == 16] * (w.at_once == 2 && (at_once == 1 || all <= cu_count) ? 0.6f : 1.0f);
            const float rounds = (float)((all + slots - 1) / slots), turns = (float)((a.steps - 1) / (splits * kw) + 1);
            const float parts = splits > 1 ? 2.5f + (float)splits * ((a.m - 1) / 16 + 1) * a.tiles * 1024 * 2 / 3.5e6f : 0.0f;
            const float us = rounds * (turns * a_step + 1.5f) + parts;
            if (best == 0.0f || us < best) best = us, p.nf = w.nf, p.nw = w.nw, p.kw = kw, p.splits = splits;
        }
    }
    return p;
}

static int launch(Int4Args& a, int group, int flags, const Int4Plan& plan, hipStream_t stream) {
    a.splits = plan.splits;
    return group == 128 ? launch_int4_1(a, flags, plan, stream) : group == 64 ? launch_int4_2(a, flags, plan, stream) : launch_int4_4(a, flags, plan, stream);
}

// A K split adds its parts up in the stream's workspace by a second launch.  A recorded launch uses no memory of the library's, so that
// graphs may replay side by side, and a call that can get no device memory does without too.
static int launch_gemm(Int4Args& a, int group, int flags, int cu_count, hipStream_t stream) {
    const Int4Plan plan = int4_plan(a, group, cu_count, true);
    // A launch has fewer than 2^32 threads: beyond, half of the rows at a time.
    const long long groups = (long long)((a.tiles - 1) / (plan.nf * plan.nw) + 1) * ((a.m - 1) / (4 * plan.xu) + 1) * plan.splits;
    if (groups * 64 * plan.kw * plan.nw >= 1ll << 32 && a.m > 64) {
        const int half = (a.m / 2 + 63) / 64 * 64;
        Int4Args first = a;
        first.m = half;
        if (int rc = launch_gemm(first, group, flags, cu_count, stream)) return rc;
        a.A += (size_t)half * a.k;
        a.D += (size_t)half * a.n;
        a.m -= half;
        return launch_gemm(a, group, flags, cu_count, stream);
    }
    if (plan.splits == 1) return launch(a, group, flags, plan, stream);
    if (!stream_is_capturing(stream)) {
        std::lock_guard<std::recursive_mutex> turn(stream_turn(stream));
        Workspace w;
        const int rc = get_workspace(stream, (size_t)((a.m - 1) / 16 + 1) * a.tiles * plan.splits * 1024, 0, &w);
        if (rc == SG_SUCCESS) {
            a.ws = w.partials;
            if (int failed = launch(a, group, flags, plan, stream)) return failed;
            return launch_int4_sum(a, stream);
        }
        if (rc != SG_NO_DEVICE && rc != SG_WORKSPACE_TOO_SMALL) return rc;
    }
    return launch(a, group, flags, int4_plan(a, group, cu_count, false), stream);
}

}  // namespace sg

using namespace sg;

namespace {
bool off(const void* p, unsigned bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }
}  // namespace

extern "C" {

size_t sg_int4_packed_bytes(int n, int k, int group, int flags) {
    return int4_takes(n, k, group, flags) ? int4_layout(n, k, group, flags).bytes : 0;
}

int sg_int4_pack(const uint8_t* B, const void* scales, const uint8_t* zeros, uint8_t* P, int n, int k, int group, int flags, int b_stride,
                 void* stream) {
    if (!B || !scales || !P || (flags & SG_INT4_ZEROS ? !zeros : zeros != nullptr) || !int4_takes(n, k, group, flags) || b_stride < k / 2)
        return SG_BAD_ARGUMENT;
    if (off(B, 16) || b_stride % 16 || off(P, 16) || off(scales, 2)) return SG_BAD_ALIGNMENT;
    DeviceInfo* dev;
    if (int rc = get_device_info(&dev)) return rc;
    const Int4Layout l = int4_layout(n, k, group, flags);
    Int4PackArgs a{B, static_cast<const uint16_t*>(scales), zeros, P, reinterpret_cast<uint16_t*>(P + l.scales_at), P + l.zeros_at,
                   n, k, group, b_stride, l.tiles, l.steps, l.gps};
    const int most = ((1 << 26) - 4) / l.steps;      // tiles: a launch has fewer than 2^32 threads
    for (int left = l.tiles;; left -= most) {
        a.tiles = left < most ? left : most;
        const size_t grid = ((size_t)a.tiles * l.steps + 3) / 4;
        int4_pack_kernel<<<(unsigned)grid, 256, 0, static_cast<hipStream_t>(stream)>>>(a);
        if (report_hip("int4_pack launch", hipGetLastError()) != hipSuccess) return SG_LAUNCH_FAILED;
        if (left <= most) return SG_SUCCESS;
        const size_t rows = (size_t)most * 16, at = (size_t)most * l.steps, groups = k / group;
        a.B += rows * b_stride;
        a.scales += rows * groups;
        if (a.zeros) a.zeros += rows * groups;
        a.n -= (int)rows;
        a.P += at * 1024;
        a.PS += at * l.gps * 16;
        a.PZ += at * l.gps * 16;
    }
}

int sg_int4_gemm(const void* A, const uint8_t* P, void* D, int m, int n, int k, int group, int flags, void* stream) {
    if (!A || !P || !D || m <= 0 || !int4_takes(n, k, group, flags)) return SG_BAD_ARGUMENT;
    if (off(A, 16) || off(P, 16) || off(D, 8)) return SG_BAD_ALIGNMENT;
    DeviceInfo* dev;
    if (int rc = get_device_info(&dev)) return rc;
    const Int4Layout l = int4_layout(n, k, group, flags);
    Int4Args a{};
    a.A = static_cast<const uint16_t*>(A);
    a.P = P;
    a.PS = P + l.scales_at;
    a.PZ = flags & SG_INT4_ZEROS ? P + l.zeros_at : nullptr;
    a.D = static_cast<uint16_t*>(D);
    a.m = m;
    a.n = n;
    a.k = k;
    a.tiles = l.tiles;
    a.steps = l.steps;
    return launch_gemm(a, group, flags, dev->cu_count, static_cast<hipStream_t>(stream));
}

}  // extern "C"
