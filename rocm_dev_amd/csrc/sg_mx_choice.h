// Which build of the MXFP4 products a shape runs on, and into how many parts its K is split.
//
// A model of the time of a launch, in microseconds, for every build:
//     steps = ceil(k / 128) / splits,  w = workgroups / (256 CUs), at least 1
//     streaming builds   a + max(steps / waves * lat, w * (e + steps * thr))     latency of one workgroup, or the CUs' throughput
//     wide builds        a + ceil(w / workgroups a CU holds) * (e + steps * lat)   whole rounds
//     both               at least bytes / 6.3 TB/s + 2.4;  2.4 more where the scales are copied first;  with a K split
//                        s0 + KB of partial sums * s1 more
// The constants are fitted to 34522 measured launches on 1000 random shapes (1..2048 rows, 128..65536 x 256..32768, cold weights,
// every build and split there is room for); picking the least on those costs 3 % over the best of them in the geometric mean.
#pragma once

#include "sg_mx.h"

namespace sg {

struct MxTimes {
    float a, lat, thr, e, s0, s1;
};
struct MxBuild {
    int number, bn, bm, waves, wide;     // wide: workgroups of a wide build that a CU holds
    MxTimes fp8, fp4;
};
// up to 16 activation rows
constexpr MxBuild kDecode[] = {
    {1101, 16, 16, 1, 0, {1.97f, 0.149f, 0.000f, 0.06f, 2.65f, 0.001880f}, {1.91f, 0.152f, 0.000f, 0.15f, 2.72f, 0.002166f}},
    {1104, 16, 16, 4, 0, {2.95f, 0.051f, 0.054f, 0.01f, 2.41f, 0.001149f}, {2.94f, 0.196f, 0.051f, 0.03f, 2.49f, 0.001230f}},
    {1108, 16, 16, 8, 0, {2.81f, 0.170f, 0.049f, 0.24f, 2.38f, 0.001753f}, {2.95f, 0.353f, 0.045f, 0.14f, 2.17f, 0.002376f}},
    {1201, 32, 16, 1, 0, {2.46f, 0.175f, 0.093f, 0.11f, 2.35f, 0.000816f}, {2.47f, 0.161f, 0.089f, 0.14f, 2.40f, 0.000919f}},
    {1204, 32, 16, 4, 0, {2.59f, 0.000f, 0.066f, 0.39f, 2.45f, 0.001277f}, {2.67f, 0.221f, 0.056f, 0.44f, 2.49f, 0.001476f}},
    {1208, 32, 16, 8, 0, {1.96f, 0.481f, 0.064f, 1.15f, 2.44f, 0.001765f}, {2.52f, 0.252f, 0.052f, 0.97f, 2.23f, 0.002166f}},
    {1702, 64, 16, 2, 0, {3.13f, 0.229f, 0.018f, 0.34f, 2.42f, 0.001173f}, {3.19f, 0.213f, 0.107f, 0.00f, 2.48f, 0.001071f}},
};
// more
constexpr MxBuild kMore[] = {
    {1301, 32, 32, 1, 0, {2.69f, 0.236f, 0.143f, 0.13f, 2.35f, 0.000533f}, {2.77f, 0.189f, 0.122f, 0.15f, 2.43f, 0.000467f}},
    {1304, 32, 32, 4, 0, {2.65f, 0.001f, 0.143f, 0.08f, 2.25f, 0.000798f}, {2.98f, 0.327f, 0.127f, 0.06f, 2.36f, 0.000600f}},
    {1404, 16, 32, 4, 0, {2.79f, 0.422f, 0.120f, 0.05f, 2.34f, 0.000792f}, {2.95f, 0.000f, 0.103f, 0.00f, 2.48f, 0.000656f}},
    {1604, 32, 64, 4, 0, {2.65f, 0.559f, 0.226f, 0.67f, 1.77f, 0.000871f}, {2.72f, 0.813f, 0.202f, 0.53f, 1.93f, 0.000778f}},
    {1702, 64, 16, 2, 0, {2.92f, 0.105f, 0.136f, 0.18f, 2.48f, 0.000423f}, {2.88f, 0.002f, 0.133f, 0.31f, 2.40f, 0.000313f}},
    {2005, 128, 128, 1, 0, {6.10f, 0.835f, 0.583f, 1.01f, 0.62f, 0.000357f}, {5.45f, 0.468f, 0.428f, 1.38f, 0.52f, 0.000397f}},
    {2006, 64, 32, 1, 0, {2.50f, 0.365f, 0.125f, 0.36f, 1.81f, 0.000868f}, {3.18f, 0.219f, 0.114f, 0.30f, 1.87f, 0.000727f}},
    {2010, 128, 64, 1, 0, {3.95f, 0.555f, 0.320f, 1.01f, 1.65f, 0.000404f}, {3.82f, 0.304f, 0.257f, 1.05f, 1.65f, 0.000450f}},
    {3001, 256, 256, 1, 1, {4.13f, 1.219f, 0.000f, 4.90f, 0.00f, 0.000312f}, {1.80f, 0.964f, 0.000f, 7.10f, 0.00f, 0.000347f}},
    {3002, 192, 128, 1, 1, {2.51f, 0.603f, 0.000f, 3.89f, 0.48f, 0.000384f}, {2.20f, 0.461f, 0.000f, 4.70f, 0.20f, 0.000437f}},
    {3003, 256, 128, 1, 1, {3.12f, 0.742f, 0.000f, 3.46f, 0.56f, 0.000377f}, {2.04f, 0.530f, 0.000f, 5.55f, 0.25f, 0.000409f}},
    {3004, 192, 256, 1, 1, {3.46f, 0.949f, 0.000f, 5.14f, 0.00f, 0.000322f}, {1.73f, 0.674f, 0.000f, 7.11f, 0.00f, 0.000367f}},
    {3006, 128, 128, 1, 1, {4.34f, 0.491f, 0.000f, 0.59f, 1.69f, 0.000390f}, {1.25f, 0.363f, 0.000f, 4.07f, 1.38f, 0.000466f}},
    {3007, 128, 128, 1, 2, {0.00f, 0.940f, 0.000f, 4.31f, 1.18f, 0.000510f}, {0.00f, 0.594f, 0.000f, 4.82f, 0.94f, 0.000593f}},
};
// build + 10000 * splits (splits > 1).  workspace: the launch may use the stream's (a K split, copied scales); copy: the wide
// kernel would need the scales copied.
inline int mx_choose(bool fp4, int m, int n, int k, int cu_count, bool workspace, bool copy) {
    const int tiles = (n - 1) / 16 + 1, steps = (k - 1) / 128 + 1, quads = (steps + 3) / 4;
    const float frags = (float)tiles * (float)((m - 1) / 16 + 1);
    const float bytes = (float)n * k * (17.f / 32) + (float)m * k * (fp4 ? 17.f / 32 : 1.f) + 2.f * m * n;
    const float least = bytes / 6.3e6f + 2.4f;
    const MxBuild* const table = m <= 16 ? kDecode : kMore;
    const int count = m <= 16 ? (int)(sizeof kDecode / sizeof *kDecode) : (int)(sizeof kMore / sizeof *kMore);
    int best = table[0].number;
    float best_us = 1e30f;
    static constexpr int kSplits[] = {1, 2, 3, 4, 6, 8, 12, 16};
    for (int b = 0; b < count; b++) {
        const MxBuild& c = table[b];
        if (c.wide && (k > 1 << 22 || (copy && !workspace))) continue;
        const MxTimes& t = fp4 ? c.fp4 : c.fp8;
        const float groups = (float)((n - 1) / c.bn + 1) * (float)((m - 1) / c.bm + 1);
        for (int splits : kSplits) {
            if (splits > quads || (splits > 1 && !workspace)) break;
            const float grid = groups * splits;
            if (splits > 1 && (grid > (c.wide ? 520 : 1100) * (cu_count / 256.f) || frags * splits > 262144.f || quads / splits < c.waves / 2)) break;
            const int part = (quads + splits - 1) / splits * 4, s = part < steps ? part : steps;
            float us, w = grid / cu_count;
            if (c.wide) {
                w /= c.wide;
                us = t.a + __builtin_ceilf(w) * (t.e + s * t.lat);
            } else {
                const float one = s * t.lat / c.waves, all = (w > 1.f ? w : 1.f) * (t.e + s * t.thr);
                us = t.a + (one > all ? one : all);
            }
            if (us < least) us = least;
            if (c.wide && copy) us += 2.4f;
            if (splits > 1) us += t.s0 + frags * splits * t.s1;
            if (us < best_us) {
                best_us = us;
                best = c.number + (splits > 1 ? 10000 * splits : 0);
            }
        }
    }
    return best;
}

}  // namespace sg
