// Which build of the MXFP4 products a shape runs on, and into how many parts its K is split.
//
// A model of the time of a launch, in microseconds, for every build:
//     steps = ceil(k / 128) / splits,  w = workgroups / (256 CUs), at least 1
//     streaming builds   a + max(steps / waves * lat, w * (e + steps * thr))     latency of one workgroup, or the CUs' throughput
//     wide builds        a + ceil(w / workgroups a CU holds) * (e + steps * lat)   whole rounds
//     both               at least bytes / 6.3 TB/s + 2.4;  2.4 more where the scales are copied first;  with a K split
//                        s0 + KB of partial sums * s1 more
// The constants are fitted to 49035 measured launches on 1100 random shapes (1..2048 rows, 128..65536 x 256..32768, cold weights, every
// build and split there is room for; nearly all of them in profiles/mxfp4_choice_samples.csv): the choice costs 3.3 % (to 16 rows) and
// 4.6 % over the best of them in the geometric mean, as much on shapes left out of the fit.  They interpolate and describe no kernel:
// some came out at 0.
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
    {1301, 32, 32, 1, 0, {2.68f, 0.242f, 0.141f, 0.10f, 2.28f, 0.000544f}, {2.76f, 0.190f, 0.127f, 0.04f, 2.40f, 0.000485f}},
    {1304, 32, 32, 4, 0, {2.81f, 0.068f, 0.143f, 0.06f, 1.96f, 0.000934f}, {2.96f, 0.222f, 0.127f, 0.03f, 2.30f, 0.000617f}},
    {1404, 16, 32, 4, 0, {2.77f, 0.383f, 0.121f, 0.06f, 2.24f, 0.000949f}, {2.88f, 0.300f, 0.104f, 0.00f, 2.40f, 0.000781f}},
    {1604, 32, 64, 4, 0, {2.80f, 0.000f, 0.236f, 0.52f, 1.75f, 0.000899f}, {2.88f, 0.620f, 0.210f, 0.33f, 1.87f, 0.000775f}},
    {1702, 64, 16, 2, 0, {3.19f, 0.001f, 0.128f, 0.09f, 2.33f, 0.000371f}, {3.25f, 0.215f, 0.119f, 0.07f, 2.39f, 0.000374f}},
    {2001, 128, 128, 1, 0, {3.62f, 0.598f, 0.595f, 1.21f, 1.38f, 0.000360f}, {2.45f, 0.112f, 0.448f, 2.13f, 1.21f, 0.000451f}},
    {2005, 128, 128, 1, 0, {5.27f, 0.721f, 0.623f, 0.66f, 1.17f, 0.000329f}, {4.26f, 0.439f, 0.419f, 1.38f, 0.95f, 0.000397f}},
    {2010, 128, 64, 1, 0, {3.53f, 0.487f, 0.288f, 0.98f, 1.75f, 0.000434f}, {3.27f, 0.329f, 0.244f, 1.03f, 1.79f, 0.000455f}},
    {2011, 128, 64, 1, 0, {4.02f, 0.393f, 0.316f, 0.62f, 1.84f, 0.000424f}, {3.33f, 0.154f, 0.263f, 1.22f, 1.82f, 0.000452f}},
    {2012, 64, 32, 1, 0, {2.77f, 0.239f, 0.136f, 0.18f, 2.23f, 0.000654f}, {2.89f, 0.172f, 0.112f, 0.26f, 2.49f, 0.000604f}},
    {2013, 64, 64, 1, 0, {3.25f, 0.333f, 0.223f, 0.44f, 2.21f, 0.000483f}, {3.38f, 0.223f, 0.186f, 0.38f, 2.35f, 0.000467f}},
    {2015, 128, 32, 1, 0, {2.86f, 0.299f, 0.196f, 0.50f, 2.32f, 0.000525f}, {3.05f, 0.206f, 0.185f, 0.64f, 2.34f, 0.000476f}},
    {3001, 256, 256, 1, 1, {3.53f, 1.192f, 0.000f, 5.54f, 0.00f, 0.000302f}, {2.90f, 0.893f, 0.000f, 5.94f, 0.00f, 0.000334f}},
    {3002, 192, 128, 1, 1, {1.99f, 0.598f, 0.000f, 4.30f, 0.58f, 0.000393f}, {1.71f, 0.416f, 0.000f, 4.91f, 0.35f, 0.000463f}},
    {3003, 256, 128, 1, 1, {2.40f, 0.713f, 0.000f, 4.20f, 0.64f, 0.000369f}, {1.60f, 0.483f, 0.000f, 5.68f, 0.41f, 0.000426f}},
    {3004, 192, 256, 1, 1, {3.03f, 0.923f, 0.000f, 5.57f, 0.00f, 0.000313f}, {2.80f, 0.620f, 0.000f, 5.98f, 0.00f, 0.000351f}},
    {3006, 128, 128, 1, 1, {4.03f, 0.497f, 0.000f, 0.84f, 1.67f, 0.000406f}, {1.10f, 0.332f, 0.000f, 3.99f, 1.46f, 0.000475f}},
    {3007, 128, 128, 1, 2, {0.00f, 0.930f, 0.000f, 4.31f, 1.21f, 0.000524f}, {0.00f, 0.554f, 0.000f, 4.71f, 1.10f, 0.000580f}},
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
            // Builds most of whose waves have no columns were not fitted.  While a CU has two workgroups such waves cost nothing (14 x 170 x 1280
            // 3.2 us on eight, 3.7 on one); beyond, they take others' places (557 x 10536 x 32 15.8 on four, 8.5 without).
            if (quads / splits < c.waves / 2 && (splits > 1 || grid > 2 * cu_count)) break;
            if (splits > 1 && (grid > (c.wide ? 520 : 1100) * (cu_count / 256.f) || frags * splits > 262144.f)) break;
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
