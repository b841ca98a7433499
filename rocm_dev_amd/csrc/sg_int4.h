// 4-bit integer weights with group scales: what its translation units share.
//
// A weight is (q - z) * s, q a code 0..15, s and z its group's: 32, 64 or 128 neighbouring columns of a row.  Weights are multiplied
// from a packed buffer, laid out once when a program loads them, as v_mfma_f32_16x16x32_bf16 takes them after an unpacking
// of one bit operation a pair.  A tile is 16 rows, a step 128 columns = four instructions:
//     codes   [n / 16][k / 128][64 lanes][4 dwords]         lane (row r = l % 16, g = l / 16), dword t: columns 32 t + 8 g .. + 7
//     scales  [n / 16][k / 128][4][groups][4 rows]  16 bits  the four rows 4 g .. 4 g + 3 that a lane of the result holds
//     zeros   [n / 16][k / 128][4][groups][4 rows]   8 bits  (with SG_INT4_ZEROS)
// with n, k rounded up; what is beyond the matrix holds code 0 and scale 0.  Within a dword, code 2 p (the pair's low half) lies at
// bit 3 + 4 p and code 2 p + 1 at bit 19 + 4 p (mod 32): rotated right by 4 p and masked with 0x00780078 the pair lies in the
// mantissas of two bf16, and with a power of two in each half it is that times 1 + q / 16, exactly.
#pragma once

#include "sg_device.h"
#include "sg_host.h"

namespace sg {

struct Int4Layout {
    int tiles, steps, gps;           // 16-row tiles, 128-column steps, groups of a step
    size_t scales_at, zeros_at, bytes;
};
inline bool int4_takes(int n, int k, int group, int flags) {
    return n > 0 && k > 0 && k <= 1 << 24 && (group == 32 || group == 64 || group == 128) && k % group == 0 && !(flags & ~(SG_INT4_ZEROS | SG_INT4_F16_SCALES));
}
inline Int4Layout int4_layout(int n, int k, int group, int flags) {
    Int4Layout l;
    l.tiles = (int)(((unsigned)n + 15) / 16);
    l.steps = (int)(((unsigned)k + 127) / 128);
    l.gps = 128 / group;
    const size_t all = (size_t)l.tiles * l.steps;
    l.scales_at = all * 1024;
    l.zeros_at = l.scales_at + all * l.gps * 32;
    l.bytes = l.zeros_at + (flags & SG_INT4_ZEROS ? all * l.gps * 16 : 0);
    return l;
}

struct Int4Args {
    const uint16_t* A;               // [m][k] bf16
    const uint8_t* P;                // codes
    const uint8_t* PS;               // scales
    const uint8_t* PZ;               // zeros, or NULL: 8
    uint16_t* D;                     // [m][n] bf16
    int m, n, k;
    int tiles, steps;
    int n_groups, m_groups;          // workgroup tiles along n and m
    int splits;                      // workgroups that share K of a tile
    float* ws;                       // splits > 1: their sums, [split][m / 16][n / 16][64 lanes][4], added by a second launch
};

constexpr int kInt4Splits = 8;       // at most

// How a product is carried out: workgroups of kw * nw waves, nw of them with nf weight tiles each, on 4 * xu activation rows.
struct Int4Plan {
    int nf, xu, nw, kw, splits;
};
Int4Plan int4_plan(const Int4Args& a, int group, int cu_count, bool workspace);

// one build of kernels for each number of groups a step (sg_int4_inst.hip)
int launch_int4_1(Int4Args& a, int flags, const Int4Plan& plan, hipStream_t stream);
int launch_int4_2(Int4Args& a, int flags, const Int4Plan& plan, hipStream_t stream);
int launch_int4_4(Int4Args& a, int flags, const Int4Plan& plan, hipStream_t stream);
int launch_int4_sum(const Int4Args& a, hipStream_t stream);

}  // namespace sg
