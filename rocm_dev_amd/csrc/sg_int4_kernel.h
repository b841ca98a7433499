// Products of bf16 activations with 4-bit integer weights:  D[m,n] = bf16( sum_g s[n,g] * sum_{k in g} A[m,k] * (q[n,k] - z[n,g]) ).
//
// What bounds it is the stream of weights, half a byte a value and the groups' scales.  The matrix instruction takes bf16, so the
// codes are widened on the way: u (1 + q / 16) by a rotation and a mask a pair (sg_int4.h), u = 2^-13, and the product of a group is set
// right behind it,
//     sum A * (q - z) = 16 / u * ( sum A * u (1 + q / 16)  -  (1 + z / 16) * sum A * u ),
// the activations' own sum by the same instruction on a matrix of u, once for all tiles of a wave - or, where waves share the activations,
// by those that bring them.  Up to 16 rows what is left beside that stream is the way of everything into a CU, 64 bytes a clock: the
// activations, read again for every tile or two, are four times a tile's codes.  Beyond, vector units and matrix units are busy in turn:
// the two fp32 multiply-adds an output and group and the widening, then the products (64 rows of 57344 x 8192 in groups of 64, 98 to 104 us: of a
// SIMD's time vector instructions take 60 %, 251 a wave and step, products 30 %, and LDS is read for 29 % of a CU's).
// u keeps the sums of finite activations finite: 128 columns below 2^128 times 1 + 255 / 16 are below 2^140, and fp32 ends at 2^128.  What it costs
// lies at the other end: products of activations below 2^-113 reach into fp32's subnormals, steps of 2^-149, 2^-132 * |s| of a result.
// The correction cancels: both of its terms are up to 16 * sum|A| / |sum A (q - z)| times the result, about 50 at
// groups of 128 of noise, so that 2^-24 of fp32 becomes 2^-18 of a group's sum, against 2^-9 of the output's rounding.
//
// A wave takes NF 16-row weight tiles and all rows of an activation tile, and walks a part of K in steps of 128 columns.  Weights go from
// memory to registers as they lie, DW steps in flight, two where a wave has few.  Activations come by 4 rows x 256 bytes a load, whole lines, and go through
// LDS: NW waves with weight tiles of their own share them (and a barrier a step), KW such groups share K by steps and meet in LDS,
// partial sums added in their order: the result does not depend on which wave is first.
#pragma once

#include <type_traits>

#include "sg_int4.h"

namespace sg {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_vec __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f32x4 mfma_bf16_16x16x32(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

constexpr uint32_t kInt4Units = 0x39003900u;      // u = 2^-13 in two bf16
constexpr float kInt4OutOfUnits = 131072.0f;      // 16 / u
// eight codes of a dword as u (1 + q / 16); `units` in a vector register, so that mask and units are one instruction
// (it takes one constant from elsewhere)
__device__ __forceinline__ u32x4 int4_widen(uint32_t d, uint32_t units) {
    return u32x4{(d & 0x00780078u) | units, (d >> 4 & 0x00780078u) | units, (d >> 8 & 0x00780078u) | units,
                 (__builtin_amdgcn_alignbit(d, d, 12) & 0x00780078u) | units};
}
// u times the sum of eight bf16
__device__ __forceinline__ float int4_sum8(u32x4 v, uint32_t units) {
    const bf16x2_vec unit = __builtin_bit_cast(bf16x2_vec, units);
    float sum = 0.0f;
#pragma unroll
    for (int c = 0; c < 4; c++) {
        const uint32_t two = v[c];          // (a bit cast of v[c] itself takes element 0)
        sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_vec, two), unit, sum, false);
    }
    return sum;
}
// four scales of two dwords
template <bool F16>
__device__ __forceinline__ f32x4 int4_scales(uint32_t lo, uint32_t hi) {
    if (F16) {
        const f16x2_t a = __builtin_bit_cast(f16x2_t, lo), b = __builtin_bit_cast(f16x2_t, hi);
        return f32x4{(float)a.x, (float)a.y, (float)b.x, (float)b.y};
    }
    return f32x4{bf16_lo(lo), bf16_hi(lo), bf16_lo(hi), bf16_hi(hi)};
}
// 1 + z / 16 in fp16, exactly, two a register as the multiply-add takes them: bytes under 1024's exponent, 1024 + z, times 1 / 16, less 63
__device__ __forceinline__ f16x2_t int4_zeros(uint32_t z, uint32_t bytes) {
    const f16x2_t v = __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(0x64646464u, z, bytes));
    return __builtin_elementwise_fma(v, f16x2_t{(_Float16)0.0625f, (_Float16)0.0625f}, f16x2_t{(_Float16)-63.0f, (_Float16)-63.0f});
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

// a step's activations in LDS, and where waves share them, the sums of their groups
__host__ __device__ constexpr int int4_buffer(int gps, int xu, int nw) { return xu * 1024 + (nw > 1 ? (gps * xu * 16 + 1023) / 1024 * 1024 : 0); }

// the sum over 4 * N neighbouring lanes, in all of them
template <int N>
__device__ __forceinline__ float int4_over_lanes(float v) {
    auto from = [&](float w, auto ctrl) {
        return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(w), decltype(ctrl)::value, 0xf, 0xf, true));
    };
    v += from(v, std::integral_constant<int, 0xb1>{});                  // the lane beside it, then the pair beside it
    v += from(v, std::integral_constant<int, 0x4e>{});
    if (N > 1) v += from(v, std::integral_constant<int, 0x141>{});      // mirrored in 8 and in 16 lanes: the other half
    if (N > 2) v += from(v, std::integral_constant<int, 0x140>{});
    return v;
}

// FLAGS: SG_INT4_ZEROS, SG_INT4_F16_SCALES.  The tile has 4 * XU activation rows.
// LDS: [KW][2][XU KB activations, NW > 1: [4 * XU][GPS] sums of groups], [KW][NW][NF][256 bytes of scales and zeros], then in its place [KW][NW][NF * MF][64 lanes] f32x4.
template <int GPS, int FLAGS, int NF, int XU, int NW, int DW, int DX, int MAXW, int MINB>
__global__ void __launch_bounds__(64 * MAXW, MINB) int4_gemm_kernel(const Int4Args a) {
    constexpr bool ZEROS = FLAGS & SG_INT4_ZEROS, F16 = FLAGS & SG_INT4_F16_SCALES;
    constexpr int MF = XU < 4 ? 1 : XU / 4, LOADS = XU / NW, ROWS = 4 * XU < 16 ? 4 * XU : 16, PER = 4 / GPS;     // PER: instructions a group
    constexpr bool SHARED = NW > 1;
    constexpr int BUFFER = int4_buffer(GPS, XU, NW);
    static_assert(XU % NW == 0 && (DX == 2 || DX == 4) && (DW == 2 || DW == 4));
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const int lane = lane_id(), r = lane & 15, g = lane >> 4;
    const int wave = wave_id(), waves = (int)(blockDim.x >> 6), KW = waves / NW, kg = wave / NW, nw = wave % NW;
    const int at = xcd_order((int)blockIdx.x, (int)gridDim.x);
    const int rest = at / a.m_groups, tm = at - rest * a.m_groups;       // neighbours share the weights, then the activations
    const int split = a.splits > 1 ? rest / a.n_groups : 0, tn = a.splits > 1 ? rest - split * a.n_groups : rest;
    const int begin = a.splits > 1 ? (int)((long long)a.steps * split / a.splits) : 0;
    const int steps = a.splits > 1 ? (int)((long long)a.steps * (split + 1) / a.splits) : a.steps;      // the end of this part of K
    const int first_tile = (tn * NW + nw) * NF;

    // ---- operands: tiles beyond the last and rows beyond m take the last one again, and are not stored ----
    // Scales and zeros: a dword a lane, 8 * GPS of scales and behind them 4 * GPS of zeros, by way of LDS to the lanes that use them.  (Each lane
    // loading what it uses itself loads everything 16 times: 4 KB a tile and step in groups of 32, by a path of 64 bytes a clock.)
    const bool of_zeros = ZEROS && lane >= 8 * GPS && lane < 12 * GPS;
    const uint32_t s_step = of_zeros ? GPS * 16 : GPS * 32, s_lane = (of_zeros ? lane - 8 * GPS : lane < 8 * GPS ? lane : 0) * 4;
    const uint8_t *wb[NF], *sb[NF];
#pragma unroll
    for (int i = 0; i < NF; i++) {
        const size_t tile = (size_t)(first_tile + i < a.tiles ? first_tile + i : a.tiles - 1) * a.steps;
        wb[i] = a.P + tile * 1024;
        sb[i] = (of_zeros ? a.PZ : a.PS) + (tile * s_step + s_lane);
    }
    // Activations: load u of the tile has rows 4 u .. 4 u + 3, lane l piece l % 16 (8 columns) of row l / 16; in LDS the pieces of row i stand
    // permuted by i, so that the 16 lanes (r, g) of a fragment's read hit 16 bank groups.
    const uint8_t* const xb = reinterpret_cast<const uint8_t*>(a.A + (size_t)tm * 4 * XU * a.k);
    uint32_t xo[LOADS], xw[LOADS], xr[4];
    const int piece = lane & 15, pieces = a.k / 8, rows_left = a.m - tm * 4 * XU;       // k is a multiple of 32
#pragma unroll
    for (int u = 0; u < LOADS; u++) {
        const int row = 4 * (nw * LOADS + u) + g;
        xo[u] = (uint32_t)(row < rows_left ? row : rows_left - 1) * (uint32_t)(2 * a.k);
        xw[u] = (uint32_t)(row * 256 + (piece ^ (row & 15)) * 16);
    }
    const int xrow = r % ROWS;
#pragma unroll
    for (int t = 0; t < 4; t++) xr[t] = (uint32_t)(xrow * 256 + ((4 * t + g) ^ xrow) * 16);
    uint8_t *const xbuf = lds + kg * 2 * BUFFER, *const sbuf = lds + KW * 2 * BUFFER + wave * (NF * 256);

    uint32_t units = kInt4Units;
    asm volatile("" : "+v"(units));
    u32x4 w[DW][NF], x[DX][LOADS];
    uint32_t s[DW][NF];
    f32x4 acc[NF][MF];
#pragma unroll
    for (int i = 0; i < NF; i++)
#pragma unroll
        for (int j = 0; j < MF; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    // A step beyond this part of K loads one piece for all lanes, which is not multiplied: a load that may not be issued would make every wait one
    // for all loads.  A piece of a row beyond its end is the last piece again: its weights' scales are zero.  (32-bit offsets: k is below 2^24.)
    auto load_x = [&](auto dc, int step) __attribute__((always_inline)) {
        constexpr int d = decltype(dc)::value % DX;
        const uint32_t live = step < steps ? ~0u : 0u;
        const int p = 16 * step + piece;
        const uint32_t po = (uint32_t)(p < pieces ? p : pieces - 1) * 16;
#pragma unroll
        for (int u = 0; u < LOADS; u++) x[d][u] = *reinterpret_cast<const u32x4*>(xb + ((xo[u] + po) & live));
    };
    auto load_w = [&](auto dc, int step) __attribute__((always_inline)) {
        constexpr int d = decltype(dc)::value % DW;
        const uint32_t live = step < steps ? ~0u : 0u, from = (uint32_t)step;
        const uint32_t wo = (from * 1024 + lane * 16) & live, so = (from * s_step) & live;
#pragma unroll
        for (int i = 0; i < NF; i++) {
            w[d][i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(wb[i] + wo));
            s[d][i] = *reinterpret_cast<const uint32_t*>(sb[i] + so);
        }
    };
    // A step's activations are brought to LDS a step before they are read, in two places in turn.
    auto share_x = [&](auto dc) __attribute__((always_inline)) {
        constexpr int d = decltype(dc)::value;
        uint8_t* const to = xbuf + d % 2 * BUFFER;
#pragma unroll
        for (int u = 0; u < LOADS; u++) *reinterpret_cast<u32x4*>(to + xw[u]) = x[d % DX][u];
        if constexpr (SHARED) {
            // the sums of the groups: 4 * PER neighbouring lanes have a group's pieces
#pragma unroll
            for (int u = 0; u < LOADS; u++) {
                const float sum = int4_over_lanes<PER>(int4_sum8(x[d % DX][u], units));
                if (piece % (4 * PER) == 0)
                    reinterpret_cast<float*>(to + XU * 1024)[piece / (4 * PER) * (4 * XU) + 4 * (nw * LOADS + u) + g] = sum;
            }
        }
    };
    // behind a step: all waves have read its activations, and have brought the next one's
    auto meet = [&]() __attribute__((always_inline)) {
        if (SHARED) asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    };
    auto multiply = [&](auto dc) __attribute__((always_inline)) {
        constexpr int d = decltype(dc)::value % DW;
        const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
        const uint8_t* const from = xbuf + decltype(dc)::value % 2 * BUFFER;
        // A unit is a group of a tile; a unit's scales are applied behind the next one's products, whose results take their time.
        constexpr int Y = MF < 4 ? 2 : 1;      // groups' activations at a time
        u32x4 y[Y][PER][MF];
        float sum[2][MF];
        f32x4 part[2][MF];
        uint32_t scales[NF][2 * GPS], zeros[NF][GPS];
#pragma unroll
        for (int i = 0; i < NF; i++) *reinterpret_cast<uint32_t*>(sbuf + i * 256 + lane * 4) = s[d][i];
        auto products = [&](int unit) __attribute__((always_inline)) {
            const int q = unit / NF, i = unit % NF, h = q % 2, u = unit % 2, hy = q % Y;
            if (q == 0) {
                int4_take(scales[i], sbuf + i * 256 + g * (GPS * 8));
                if (ZEROS) int4_take(zeros[i], sbuf + i * 256 + GPS * 32 + g * (GPS * 4));
            }
            if (i == 0) {
#pragma unroll
                for (int j = 0; j < MF; j++) {
#pragma unroll
                    for (int t = 0; t < PER; t++) y[hy][t][j] = *reinterpret_cast<const u32x4*>(from + j * 4096 + xr[q * PER + t]);
                    if constexpr (SHARED) {
                        sum[h][j] = reinterpret_cast<const float*>(from + XU * 1024)[q * (4 * XU) + 16 * j + r];
                    } else {
                        f32x4 of_all = zero;
#pragma unroll
                        for (int t = 0; t < PER; t++) of_all = mfma_bf16_16x16x32(u32x4{units, units, units, units}, y[hy][t][j], of_all);
                        sum[h][j] = of_all[0];
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < PER; t++) {
                const u32x4 v = int4_widen(w[d][i][q * PER + t], units);
#pragma unroll
                for (int j = 0; j < MF; j++) part[u][j] = mfma_bf16_16x16x32(v, y[hy][t][j], t ? part[u][j] : zero);
            }
        };
        auto apply = [&](int unit) __attribute__((always_inline)) {
            const int q = unit / NF, i = unit % NF, h = q % 2, u = unit % 2;
            const f32x4 scale = int4_scales<F16>(scales[i][2 * q], scales[i][2 * q + 1]);
            f16x2_t zb[2];
            if (ZEROS) zb[0] = int4_zeros(zeros[i][q], 0x04010400u), zb[1] = int4_zeros(zeros[i][q], 0x04030402u);
#pragma unroll
            for (int j = 0; j < MF; j++)
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const float by = ZEROS ? (float)(c % 2 ? zb[c / 2].y : zb[c / 2].x) : 1.5f;
                    acc[i][j][c] = fmaf(scale[c], fmaf(-by, sum[h][j], part[u][j][c]), acc[i][j][c]);
                }
        };
#pragma unroll
        for (int unit = 0; unit <= GPS * NF; unit++) {
            if (unit < GPS * NF) products(unit);
            if (unit > 0) apply(unit - 1);
        }
        __builtin_amdgcn_sched_barrier(0);    // steps are not mixed: their temporaries would not fit
    };
    // Steps kg, kg + KW, ...  A group with one fewer than another goes through the other's barriers.
    const int end = SHARED ? begin + (steps - begin - 1) / KW * KW + KW : steps;
    int step = begin + kg, left = step < end ? (end - 1 - step) / KW + 1 : 0;
    auto turn = [&](auto dc) __attribute__((always_inline)) {
        using Next = std::integral_constant<int, (decltype(dc)::value + 1) % 4>;
        share_x(Next{});                                     // (behind the last step what a step beyond the matrix loads)
        load_x(Next{}, step + (DX + 1) * KW);
        if (!SHARED || step < steps) multiply(dc);
        load_w(dc, step + DW * KW);
        step += KW;
        left--;
        meet();
    };
    using D0 = std::integral_constant<int, 0>;
    using D1 = std::integral_constant<int, 1>;
    using D2 = std::integral_constant<int, 2>;
    using D3 = std::integral_constant<int, 3>;
    if (left > 0) {
        load_x(D0{}, step);
        load_w(D0{}, step);
        load_x(D1{}, step + KW);
        load_w(D1{}, step + KW);
        if (DX > 2) load_x(D2{}, step + 2 * KW);
        if (DW > 2) load_w(D2{}, step + 2 * KW);
        if (DX > 2) load_x(D3{}, step + 3 * KW);
        if (DW > 2) load_w(D3{}, step + 3 * KW);
        share_x(D0{});
        load_x(D0{}, step + DX * KW);
        meet();
        // As many turns as there are places by turn, and what is left behind them: a loop with an exit in its midst has its head waiting for all
        // loads in flight.
        constexpr int TURNS = DW > DX ? DW : DX;
        while (left >= TURNS) {
            turn(D0{});
            turn(D1{});
            if constexpr (TURNS > 2) {
                turn(D2{});
                turn(D3{});
            }
        }
        if (left > 0) turn(D0{});
        if constexpr (TURNS > 2) {
            if (left > 0) turn(D1{});
            if (left > 0) turn(D2{});
        }
    }

    // ---- the groups' sums, in their order ----
    auto finish = [&](f32x4 v, int i, int j) __attribute__((always_inline)) {
        if (a.splits > 1) {        // into the workspace, whole fragments
            const int tile = first_tile + i, m_frag = tm * MF + j, m_frags = (a.m - 1) / 16 + 1;
            if (tile < a.tiles && m_frag < m_frags) reinterpret_cast<f32x4*>(a.ws)[(((size_t)split * m_frags + m_frag) * a.tiles + tile) * 64 + lane] = v;
            return;
        }
        const int n_idx = (first_tile + i) * 16 + 4 * g, m_idx = tm * 4 * XU + 16 * j + r;
        if (r < ROWS && m_idx < a.m && n_idx < a.n) int4_store4(a, m_idx, n_idx, v * kInt4OutOfUnits);
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
