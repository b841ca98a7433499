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
// A wave takes NF 16-row weight tiles and MF 16-row activation tiles and walks a part of K in steps of 128 columns; operands go
// from memory to registers as they lie, DEPTH steps in flight.  The waves of a workgroup share K by steps and meet in LDS,
// partial sums added in wave order: the result does not depend on which wave is first.
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

// FLAGS: SG_INT4_ZEROS, SG_INT4_F16_SCALES
template <int GPS, int FLAGS, int NF, int MF, int DEPTH>
__global__ void __launch_bounds__(512) int4_gemm_kernel(const Int4Args a) {
    constexpr bool ZEROS = FLAGS & SG_INT4_ZEROS, F16 = FLAGS & SG_INT4_F16_SCALES;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];     // [waves][NF * MF][64 lanes] f32x4
    const int lane = lane_id(), r = lane & 15, g = lane >> 4;
    const int wave = wave_id(), waves = (int)(blockDim.x >> 6);
    const int at = xcd_order((int)blockIdx.x, (int)gridDim.x);
    const int tn = at / a.m_groups, tm = at - tn * a.m_groups;       // neighbours share the weights

    // ---- operands of lane (r, g): tiles beyond the last and rows beyond m take the last one again, and are not stored ----
    const uint8_t* wp[NF];
    const uint8_t* sp[NF];
    const uint8_t* zp[NF];
#pragma unroll
    for (int i = 0; i < NF; i++) {
        const size_t tile = (size_t)(tn * NF + i < a.tiles ? tn * NF + i : a.tiles - 1) * a.steps;
        wp[i] = a.P + tile * 1024 + lane * 16;
        sp[i] = a.PS + (tile * 4 + g) * GPS * 8;
        zp[i] = ZEROS ? a.PZ + (tile * 4 + g) * GPS * 4 : nullptr;
    }
    const uint8_t* xp[MF];
#pragma unroll
    for (int j = 0; j < MF; j++) {
        const int row = (tm * MF + j) * 16 + r < a.m ? (tm * MF + j) * 16 + r : a.m - 1;
        xp[j] = reinterpret_cast<const uint8_t*>(a.A + (size_t)row * a.k);
    }
    const int pieces = a.k / 8;       // of 8 columns; k is a multiple of 32

    u32x4 w[DEPTH][NF], x[DEPTH][MF][4];
    uint32_t s[DEPTH][NF][2 * GPS], z[DEPTH][NF][GPS];
    f32x4 acc[NF][MF];
#pragma unroll
    for (int i = 0; i < NF; i++)
#pragma unroll
        for (int j = 0; j < MF; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    // `step` is inside the matrix.  A piece of a row beyond its end takes the last piece: its weights' scales are zero.
    auto load = [&](auto dc, int step) __attribute__((always_inline)) {
        constexpr int d = decltype(dc)::value;
#pragma unroll
        for (int i = 0; i < NF; i++) {
            w[d][i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(wp[i] + (size_t)step * 1024));
            int4_take(s[d][i], sp[i] + (size_t)step * (GPS * 32));
            if (ZEROS) int4_take(z[d][i], zp[i] + (size_t)step * (GPS * 16));
        }
#pragma unroll
        for (int j = 0; j < MF; j++)
#pragma unroll
            for (int t = 0; t < 4; t++) {
                const int p = 16 * step + 4 * t + g;
                x[d][j][t] = *reinterpret_cast<const u32x4*>(xp[j] + (size_t)(p < pieces ? p : pieces - 1) * 16);
            }
    };
    auto multiply = [&](auto dc) __attribute__((always_inline)) {
        constexpr int d = decltype(dc)::value;
        constexpr int PER = 4 / GPS;          // instructions a group
        const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
        const u32x4 ones = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
#pragma unroll
        for (int q = 0; q < GPS; q++) {
            f32x4 sum[MF], part[NF][MF];
#pragma unroll
            for (int t = 0; t < PER; t++) {
#pragma unroll
                for (int j = 0; j < MF; j++) sum[j] = mfma_bf16_16x16x32(ones, x[d][j][q * PER + t], t ? sum[j] : zero);
#pragma unroll
                for (int i = 0; i < NF; i++) {
                    const u32x4 v = int4_widen(w[d][i][q * PER + t]);
#pragma unroll
                    for (int j = 0; j < MF; j++) part[i][j] = mfma_bf16_16x16x32(v, x[d][j][q * PER + t], t ? part[i][j] : zero);
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
    using D1 = std::integral_constant<int, 1 % DEPTH>;
    static_assert(DEPTH <= 2);

    // Steps wave, wave + waves, ...: `left` of them.
    int step = wave, left = wave < a.steps ? (a.steps - 1 - wave) / waves + 1 : 0;
    if (left > 0) load(D0{}, step);
    if (DEPTH > 1 && left > 1) load(D1{}, step + waves);
    for (; left >= 2 * DEPTH; left -= DEPTH, step += DEPTH * waves) {
        multiply(D0{});
        load(D0{}, step + DEPTH * waves);
        if (DEPTH > 1) {
            multiply(D1{});
            load(D1{}, step + (DEPTH + 1) * waves);
        }
    }
    // fewer than 2 * DEPTH are left, the first DEPTH of them loaded
    if (left > 0) {
        multiply(D0{});
        if (left > DEPTH) load(D0{}, step + DEPTH * waves);
        if (DEPTH > 1 && left > 1) multiply(D1{});
        if (left > DEPTH) multiply(D0{});
    }

    // ---- the waves' sums, in wave order ----
    auto finish = [&](f32x4 v, int i, int j) __attribute__((always_inline)) {
        const int n_idx = (tn * NF + i) * 16 + 4 * g, m_idx = (tm * MF + j) * 16 + r;
        if (m_idx < a.m && n_idx < a.n) int4_store4(a, m_idx, n_idx, v * 16.0f);
    };
    if (waves == 1) {
#pragma unroll
        for (int i = 0; i < NF; i++)
#pragma unroll
            for (int j = 0; j < MF; j++) finish(acc[i][j], i, j);
        return;
    }
    f32x4* const part = reinterpret_cast<f32x4*>(lds);
#pragma unroll
    for (int i = 0; i < NF; i++)
#pragma unroll
        for (int j = 0; j < MF; j++) part[(wave * NF * MF + i * MF + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    for (int f = wave; f < NF * MF; f += waves) {
        f32x4 v = part[f * 64 + lane];
        for (int u = 1; u < waves; u++) v += part[(u * NF * MF + f) * 64 + lane];
        finish(v, f / MF, f % MF);
    }
}

}  // namespace sg
