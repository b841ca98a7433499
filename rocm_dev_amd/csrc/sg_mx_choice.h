// Which build of the MXFP4 products a shape runs on, and into how many parts its K is split.
//
// A model of the time of a launch, in microseconds, for every build:
//     steps = ceil(k / 128) / splits,  w = workgroups / (256 CUs), at least 1
//     streaming builds   a + max(steps / waves * lat, w * (e + steps * thr))     latency of one workgroup, or the CUs' throughput
//     wide builds        a + ceil(w / workgroups a CU holds) * (e + steps * lat)   whole rounds
//     both               at least bytes / 6.3 TB/s + 2.4;  2.4 more where the scales are copied first;  with a K split
//                        s0 + KB of partial sums * s1 more
// The constants are fitted to 53727 measured launches on 1200 random shapes (1..2048 rows, 128..65536 x 256..32768, cold weights,
// every build and split there is room for); picking the least on those costs 3 to 4 % over the best of them in the geometric mean.
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
    {1101, 16, 16, 1, 0, {1.98f, 0.148f, 0.051f, 0.11f, 2.64f, 0.002020f}, {1.88f, 0.150f, 0.050f, 0.11f, 2.81f, 0.001640f}},
    {1104, 16, 16, 4, 0, {2.90f, 0.202f, 0.053f, 0.05f, 2.43f, 0.001460f}, {2.90f, 0.193f, 0.052f, 0.02f, 2.46f, 0.001025f}},
    {1108, 16, 16, 8, 0, {2.77f, 0.364f, 0.048f, 0.18f, 2.34f, 0.002378f}, {2.66f, 0.322f, 0.045f, 0.25f, 2.43f, 0.001672f}},
    {1201, 32, 16, 1, 0, {2.52f, 0.175f, 0.030f, 0.35f, 2.17f, 0.001508f}, {2.48f, 0.162f, 0.007f, 0.34f, 2.22f, 0.001464f}},
    {1204, 32, 16, 4, 0, {2.73f, 0.259f, 0.000f, 0.78f, 2.65f, 0.001788f}, {2.71f, 0.053f, 0.055f, 0.34f, 2.48f, 0.001395f}},
    {1208, 32, 16, 8, 0, {2.12f, 0.011f, 0.063f, 0.86f, 2.45f, 0.002383f}, {2.22f, 0.314f, 0.051f, 1.10f, 2.34f, 0.002161f}},
    {1702, 64, 16, 2, 0, {2.96f, 0.191f, 0.112f, 0.26f, 2.44f, 0.001139f}, {3.16f, 0.216f, 0.000f, 0.38f, 2.42f, 0.001178f}},
    {1704, 64, 16, 4, 0, {2.82f, 0.397f, 0.000f, 1.22f, 2.78f, 0.001283f}, {2.76f, 0.358f, 0.090f, 0.46f, 2.47f, 0.001227f}},
    {2012, 64, 32, 1, 0, {2.96f, 0.264f, 0.019f, 0.11f, 1.78f, 0.001560f}, {3.29f, 0.000f, 0.186f, 0.00f, 1.94f, 0.001070f}},
    {2015, 128, 32, 1, 0, {2.59f, 0.324f, 0.000f, 0.79f, 2.23f, 0.001116f}, {3.33f, 0.208f, 0.092f, 0.23f, 2.19f, 0.001330f}},
};
// more
constexpr MxBuild kMore[] = {
    {1301, 32, 32, 1, 0, {2.58f, 0.241f, 0.140f, 0.10f, 2.39f, 0.000525f}, {2.83f, 0.188f, 0.127f, 0.05f, 2.34f, 0.000482f}},
    {1304, 32, 32, 4, 0, {2.80f, 0.016f, 0.142f, 0.03f, 2.15f, 0.000742f}, {3.06f, 0.077f, 0.127f, 0.04f, 2.25f, 0.000630f}},
    {1404, 16, 32, 4, 0, {2.83f, 0.360f, 0.119f, 0.04f, 2.35f, 0.000703f}, {2.91f, 0.106f, 0.104f, 0.00f, 2.39f, 0.000869f}},
    {1604, 32, 64, 4, 0, {2.82f, 0.849f, 0.236f, 0.54f, 1.64f, 0.000880f}, {2.70f, 0.710f, 0.223f, 0.38f, 1.77f, 0.000865f}},
    {1702, 64, 16, 2, 0, {3.12f, 0.191f, 0.128f, 0.07f, 2.47f, 0.000369f}, {3.26f, 0.001f, 0.118f, 0.09f, 2.40f, 0.000336f}},
    {2001, 128, 128, 1, 0, {3.55f, 0.511f, 0.599f, 1.31f, 1.53f, 0.000330f}, {3.34f, 0.475f, 0.460f, 1.37f, 1.18f, 0.000422f}},
    {2005, 128, 128, 1, 0, {5.33f, 0.753f, 0.625f, 0.68f, 1.26f, 0.000308f}, {5.18f, 0.455f, 0.423f, 0.79f, 0.92f, 0.000375f}},
    {2010, 128, 64, 1, 0, {3.69f, 0.487f, 0.282f, 0.99f, 1.83f, 0.000404f}, {3.49f, 0.329f, 0.239f, 0.98f, 1.83f, 0.000424f}},
    {2011, 128, 64, 1, 0, {3.93f, 0.406f, 0.319f, 0.72f, 2.08f, 0.000370f}, {3.55f, 0.278f, 0.269f, 1.09f, 1.93f, 0.000406f}},
    {2012, 64, 32, 1, 0, {2.70f, 0.241f, 0.135f, 0.18f, 2.38f, 0.000638f}, {2.93f, 0.172f, 0.116f, 0.29f, 2.57f, 0.000507f}},
    {2013, 64, 64, 1, 0, {3.21f, 0.342f, 0.225f, 0.47f, 2.32f, 0.000468f}, {3.38f, 0.233f, 0.179f, 0.45f, 2.39f, 0.000464f}},
    {2015, 128, 32, 1, 0, {2.81f, 0.297f, 0.192f, 0.51f, 2.40f, 0.000509f}, {3.07f, 0.206f, 0.188f, 0.70f, 2.38f, 0.000430f}},
    {3001, 256, 256, 1, 1, {2.76f, 1.210f, 0.000f, 6.51f, 0.00f, 0.000283f}, {4.26f, 0.974f, 0.000f, 4.70f, 0.00f, 0.000334f}},
    {3002, 192, 128, 1, 1, {2.12f, 0.602f, 0.000f, 4.30f, 0.59f, 0.000353f}, {2.47f, 0.466f, 0.000f, 4.37f, 0.30f, 0.000414f}},
    {3003, 256, 128, 1, 1, {2.32f, 0.742f, 0.000f, 4.24f, 0.80f, 0.000326f}, {3.05f, 0.536f, 0.000f, 4.46f, 0.33f, 0.000401f}},
    {3004, 192, 256, 1, 1, {2.85f, 0.945f, 0.000f, 5.97f, 0.00f, 0.000294f}, {2.93f, 0.685f, 0.000f, 6.03f, 0.00f, 0.000337f}},
    {3006, 128, 128, 1, 1, {4.05f, 0.498f, 0.000f, 0.74f, 1.84f, 0.000365f}, {1.43f, 0.368f, 0.000f, 3.89f, 1.40f, 0.000440f}},
    {3007, 128, 128, 1, 2, {0.00f, 0.938f, 0.000f, 4.29f, 1.30f, 0.000492f}, {0.00f, 0.598f, 0.000f, 4.72f, 1.06f, 0.000555f}},
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
