// Products of bf16 activations with 4-bit integer weights:  D[m,n] = bf16( sum_g s[n,g] * sum_{k in g} A[m,k] * (q[n,k] - z[n,g]) ).
//
// What bounds it is the stream of weights, half a byte a value and the groups' scales.  The matrix instruction takes bf16, so the
// codes are widened on the way: 1 + q / 16 by a rotation and a mask a pair (sg_int4.h), and the product of a group is set right behind it,
//     sum A * (q - z) = 16 * ( sum A * (1 + q / 16)  -  (1 + z / 16) * sum A ),
// the activations' own sum by the same instruction on a matrix of ones, once for all tiles of a wave.  Seven vector operations a
// dword of eight codes: a third of the clocks at the rate at which the memory delivers.
// The correction cancels: both of its terms are up to 16 * sum|A| / |sum A (q - z)| times the result, about 50 at
// groups of 128 of noise, so that 2^-24 of fp32 becomes 2^-18 of a group's sum, against 2^-9 of the output's rounding.
//
// A wave takes NF 16-row weight tiles and all rows of an activation tile, and walks a part of K in steps of 128 columns.  Weights go from
// memory to registers as they lie, two steps in flight.  Activations come by 4 rows x 256 bytes a load, whole lines, and go through
// LDS: NW waves with weight tiles of their own share them (and a barrier a step), KW such groups share K by steps and meet in LDS,
// partial sums added in their order: the result does not depend on which wave is first.
#pragma once

#include "sg_int4.h"

namespace sg {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f32x4 mfma_bf16_16x16x32(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// eight codes of a dword as 1 + q / 16
__device__ __forceinline__ u32x4 int4_widen(uint32_t d) {
    u32x4 v;
#pragma unroll
    for (int p = 0; p < 4; p++) {
        const uint32_t at = p ? __builtin_amdgcn_alignbit(d, d, 4 * p) : d;
        v[p] = (at & 0x00780078u) | 0x3f803f80u;
    }
    return v;
}
// four scales of two dwords, four zeros of one
template <bool F16>
__device__ __forceinline__ f32x4 int4_scales(uint32_t lo, uint32_t hi) {
    if (F16) {
        const f16x2_t a = __builtin_bit_cast(f16x2_t, lo), b = __builtin_bit_cast(f16x2_t, hi);
        return f32x4{(float)a.x, (float)a.y, (float)b.x, (float)b.y};
    }
    return f32x4{bf16_lo(lo), bf16_hi(lo), bf16_lo(hi), bf16_hi(hi)};
}
__device__ __forceinline__ f32x4 int4_zeros(uint32_t z) {      // 1 + z / 16
    f32x4 v;
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = fmaf((float)((z >> (8 * i)) & 0xffu), 0.0625f, 1.0f);
    return v;
}

// N dwords by as few loads as their alignment (N dwords, at most four) allows
template <int N>
__device__ __forceinline__ void int4_take(uint32_t (&v)[N], const uint8_t* p) {
    if constexpr (N == 1) v[0] = *reinterpret_cast<const uint32_t*>(p);
    else if constexpr (N == 2) {
        const u32x2 t = *reinterpret_cast<const u32x2*>(p);
        v[0] = t.x, v[1] = t.y;
    } else {
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            const u32x4 t = *reinterpret_cast<const u32x4*>(p + 16 * i);
#pragma unroll
            for (int j = 0; j < 4; j++) v[4 * i + j] = t[j];
        }
    }
}

// four consecutive n of row m_idx, at n_idx = a multiple of 4
__device__ __forceinline__ void int4_store4(const Int4Args& a, int m_idx, int n_idx, f32x4 v) {
    uint16_t* const d = a.D + (size_t)m_idx * a.n + n_idx;
    const uint32_t lo = pack_bf16x2(v[0], v[1]), hi = pack_bf16x2(v[2], v[3]);
    if (n_idx + 4 <= a.n) {
        // one store at whatever multiple of two bytes an odd n leaves it
        using u32x2_at2 = u32x2 __attribute__((aligned(2)));
        *reinterpret_cast<u32x2_at2*>(d) = u32x2{lo, hi};
    } else {
        d[0] = (uint16_t)lo;
        if (n_idx + 1 < a.n) d[1] = (uint16_t)(lo >> 16);
        if (n_idx + 2 < a.n) d[2] = (uint16_t)hi;
    }
}

// FLAGS: SG_INT4_ZEROS, SG_INT4_F16_SCALES.  The tile has 4 * XU activation rows.
// LDS: [KW][NW > 1 ? 2 : 1][XU KB] activations, then in its place [KW][NW][NF * MF][64 lanes] f32x4.
template <int GPS, int FLAGS, int NF, int XU, int NW>
__global__ void __launch_bounds__(512) int4_gemm_kernel(const Int4Args a) {
    constexpr bool ZEROS = FLAGS & SG_INT4_ZEROS, F16 = FLAGS & SG_INT4_F16_SCALES;
    constexpr int MF = XU < 4 ? 1 : XU / 4, LOADS = XU / NW, ROWS = 4 * XU < 16 ? 4 * XU : 16, BUFFERS = NW > 1 ? 2 : 1;
    static_assert(XU % NW == 0);
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const int lane = lane_id(), r = lane & 15, g = lane >> 4;
    const int wave = wave_id(), waves = (int)(blockDim.x >> 6), KW = waves / NW, kg = wave / NW, nw = wave % NW;
    const int at = xcd_order((int)blockIdx.x, (int)gridDim.x);
    const int tn = at / a.m_groups, tm = at - tn * a.m_groups;       // neighbours share the weights
    const int first_tile = (tn * NW + nw) * NF;

    // ---- operands of lane (r, g): tiles beyond the last and rows beyond m take the last one again, and are not stored ----
    const uint8_t* wp[NF];
    const uint8_t* sp[NF];
    const uint8_t* zp[NF];
#pragma unroll
    for (int i = 0; i < NF; i++) {
        const size_t tile = (size_t)(first_tile + i < a.tiles ? first_tile + i : a.tiles - 1) * a.steps;
        wp[i] = a.P + tile * 1024 + lane * 16;
        sp[i] = a.PS + (tile * 4 + g) * GPS * 8;
        zp[i] = ZEROS ? a.PZ + (tile * 4 + g) * GPS * 4 : nullptr;
    }
    // Activations: load u of the tile has rows 4 u .. 4 u + 3, lane l piece l % 16 (8 columns) of row l / 16; in LDS the pieces of row i stand
    // permuted by i, so that the 16 lanes (r, g) of a fragment's read hit 16 bank groups.
    const uint8_t* xp[LOADS];
    uint32_t xw[LOADS], xr[4];
    const int piece = lane & 15, pieces = a.k / 8;       // k is a multiple of 32
#pragma unroll
    for (int u = 0; u < LOADS; u++) {
        const int in = 4 * (nw * LOADS + u) + g, row = tm * 4 * XU + in;
        xp[u] = reinterpret_cast<const uint8_t*>(a.A + (size_t)(row < a.m ? row : a.m - 1) * a.k);
        xw[u] = (uint32_t)(in * 256 + (piece ^ (in & 15)) * 16);
    }
    const int xrow = r % ROWS;
#pragma unroll
    for (int t = 0; t < 4; t++) xr[t] = (uint32_t)(xrow * 256 + ((4 * t + g) ^ xrow) * 16);
    uint8_t* const xbuf = lds + kg * (BUFFERS * XU * 1024);

    u32x4 w[2][NF], x[2][LOADS];
    uint32_t s[2][NF][2 * GPS], z[2][NF][GPS];
    f32x4 acc[NF][MF];
#pragma unroll
    for (int i = 0; i < NF; i++)
#pragma unroll
        for (int j = 0; j < MF; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    // `step` is inside the matrix.  A piece of a row beyond its end takes the last piece: its weights' scales are zero.
    auto load = [&](auto dc, int step) __attribute__((always_inline)) {
        constexpr int d = decltype(dc)::value;
        const int p = 16 * step + piece;
#pragma unroll
        for (int u = 0; u < LOADS; u++) x[d][u] = *reinterpret_cast<const u32x4*>(xp[u] + (size_t)(p < pieces ? p : pieces - 1) * 16);
#pragma unroll
        for (int i = 0; i < NF; i++) {
            w[d][i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(wp[i] + (size_t)step * 1024));
            int4_take(s[d][i], sp[i] + (size_t)step * (GPS * 32));
            if (ZEROS) int4_take(z[d][i], zp[i] + (size_t)step * (GPS * 16));
        }
    };
    // LDS operations of a wave are carried out in order: with NW = 1 the next step's pieces may be written behind this step's reads.
    auto share_x = [&](auto dc) __attribute__((always_inline)) {
        constexpr int d = decltype(dc)::value;
#pragma unroll
        for (int u = 0; u < LOADS; u++) *reinterpret_cast<u32x4*>(xbuf + (NW > 1 ? d * XU * 1024 : 0) + xw[u]) = x[d][u];
        if (NW > 1) asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    };
    auto multiply = [&](auto dc) __attribute__((always_inline)) {
        constexpr int d = decltype(dc)::value;
        constexpr int PER = 4 / GPS;          // instructions a group
        const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
        const u32x4 ones = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
        const uint8_t* const from = xbuf + (NW > 1 ? d * XU * 1024 : 0);
#pragma unroll
        for (int q = 0; q < GPS; q++) {
            f32x4 sum[MF], part[NF][MF];
#pragma unroll
            for (int t = 0; t < PER; t++) {
                u32x4 y[MF];
#pragma unroll
                for (int j = 0; j < MF; j++) {
                    y[j] = *reinterpret_cast<const u32x4*>(from + j * 4096 + xr[q * PER + t]);
                    sum[j] = mfma_bf16_16x16x32(ones, y[j], t ? sum[j] : zero);
                }
#pragma unroll
                for (int i = 0; i < NF; i++) {
                    const u32x4 v = int4_widen(w[d][i][q * PER + t]);
#pragma unroll
                    for (int j = 0; j < MF; j++) part[i][j] = mfma_bf16_16x16x32(v, y[j], t ? part[i][j] : zero);
                }
            }
#pragma unroll
            for (int i = 0; i < NF; i++) {
                const f32x4 scale = int4_scales<F16>(s[d][i][2 * q], s[d][i][2 * q + 1]);
                const f32x4 zb = ZEROS ? int4_zeros(z[d][i][q]) : f32x4{1.5f, 1.5f, 1.5f, 1.5f};
#pragma unroll
                for (int j = 0; j < MF; j++)
#pragma unroll
                    for (int c = 0; c < 4; c++) acc[i][j][c] = fmaf(scale[c], fmaf(-zb[c], sum[j][c], part[i][j][c]), acc[i][j][c]);
            }
        }
        __builtin_amdgcn_sched_barrier(0);    // steps are not mixed: their temporaries would not fit
    };
    using D0 = std::integral_constant<int, 0>;
    using D1 = std::integral_constant<int, 1>;

    // Steps kg, kg + KW, ...: `left` of them; a group that has one fewer than another goes through the other's barriers.
    int step = kg, left = kg < a.steps ? (a.steps - 1 - kg) / KW + 1 : 0;
    int rounds = NW > 1 ? (a.steps - 1) / KW + 1 : left;
    if (left > 0) load(D0{}, step);
    if (left > 1) load(D1{}, step + KW);
    for (; left >= 4; left -= 2, rounds -= 2, step += 2 * KW) {
        share_x(D0{});
        multiply(D0{});
        load(D0{}, step + 2 * KW);
        share_x(D1{});
        multiply(D1{});
        load(D1{}, step + 3 * KW);
    }
    // at most three are left, the first two of them loaded
    if (rounds > 0) share_x(D0{});
    if (left > 0) multiply(D0{});
    if (left > 2) load(D0{}, step + 2 * KW);
    if (rounds > 1) share_x(D1{});
    if (left > 1) multiply(D1{});
    if (rounds > 2) share_x(D0{});
    if (left > 2) multiply(D0{});
    if (rounds > 3) share_x(D1{});

    // ---- the groups' sums, in their order ----
    auto finish = [&](f32x4 v, int i, int j) __attribute__((always_inline)) {
        const int n_idx = (first_tile + i) * 16 + 4 * g, m_idx = tm * 4 * XU + 16 * j + r;
        if (r < ROWS && m_idx < a.m && n_idx < a.n) int4_store4(a, m_idx, n_idx, v * 16.0f);
    };
    if (KW == 1) {
#pragma unroll
        for (int i = 0; i < NF; i++)
#pragma unroll
            for (int j = 0; j < MF; j++) finish(acc[i][j], i, j);
        return;
    }
    __syncthreads();          // the activations' place is taken over
    f32x4* const part = reinterpret_cast<f32x4*>(lds);
#pragma unroll
    for (int i = 0; i < NF; i++)
#pragma unroll
        for (int j = 0; j < MF; j++) part[((kg * NW + nw) * NF * MF + i * MF + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    for (int f = kg; f < NF * MF; f += KW) {
        f32x4 v = part[(nw * NF * MF + f) * 64 + lane];
        for (int u = 1; u < KW; u++) v += part[((u * NW + nw) * NF * MF + f) * 64 + lane];
        finish(v, f / MF, f % MF);
    }
}

}  // namespace sg
