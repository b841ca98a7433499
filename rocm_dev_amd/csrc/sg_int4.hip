// 4-bit integer weights with group scales: packing, launches and C entry points (include/sgemm.h).
#include <limits.h>

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
    const size_t grid = ((size_t)l.tiles * l.steps + 3) / 4;
    if (grid > INT_MAX) return SG_BAD_ARGUMENT;
    const Int4PackArgs a{B, static_cast<const uint16_t*>(scales), zeros, P, reinterpret_cast<uint16_t*>(P + l.scales_at), P + l.zeros_at,
                         n, k, group, b_stride, l.tiles, l.steps, l.gps};
    int4_pack_kernel<<<(unsigned)grid, 256, 0, static_cast<hipStream_t>(stream)>>>(a);
    return report_hip("int4_pack launch", hipGetLastError()) == hipSuccess ? SG_SUCCESS : SG_LAUNCH_FAILED;
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
    auto* const launch = group == 128 ? launch_int4_1 : group == 64 ? launch_int4_2 : launch_int4_4;
    return launch(a, flags, dev->cu_count, static_cast<hipStream_t>(stream));
}

}  // extern "C"
