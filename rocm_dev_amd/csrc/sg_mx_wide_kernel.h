// Products with MXFP4 weights on wide tiles (a prefill chunk):  D[m,n] = bf16(scale * row[m] * sum_k A[m,k] * B[n,k]).
//
// Bound by the matrix cores - 8 PFLOP/s of MXFP4 products, 4.2 of E4M3 x MXFP4 on random operands in registers - and next to
// them by the LDS.  Four waves, one a SIMD, in a 2 x 2 grid own RGW x MH fragments of 16 x 16 each.  A stage is 128 bytes of
// every activation row: 128 columns of E4M3 (one step of the matrix instruction) or 256 of MXFP4 (two).  Weights,
// activations and the block scales of both reach LDS by direct loads: the weights by contiguous KBs of the packed buffer
// (sg_mx.h), read back as they lie; the activations row by row, piece p of row x at p ^ ((x / 2) % 8).
//
// As in the E4M3 kernel of this shape (sg_wide_kernel.h) nothing is read in front of its use and no burst of memory
// instructions stands between two products: a stage's activation fragments are in registers, two sets; the weight
// fragments stream through a ring, AHEAD groups (of MH fragments) early; the barrier between two stages stands AHEAD groups
// before the end of a stage, and LDS reads and refills are dealt out to the products they are issued in front of.
//
// Block scales come by groups of four steps (512 columns) into two LDS slots, asked for a group ahead.  Direct loads take 16
// bytes at a 16-byte address, so the scales of MXFP4 activations have to lie on rows of whole groups: where k is no
// multiple of 512 (or their address none of 16) a small launch copies them so first.
//
// 1024 x 57344 x 8192: E4M3 activations 360 us = 2.7 PFLOP/s, 63 % of the instruction's rate and level with the E4M3 kernel of this shape;
// MXFP4 268 us on 192 x 256 tiles = 3.6 PFLOP/s, 44 % of its rate: a stage of 1536 clocks of products takes 3500, a quarter of them
// in waits and at barriers, a fifth before an instruction may issue (profiles/mxfp4_gemm_counters.md).  Tried there, against 272 to 285
// at the time, and not kept: stages of 64 bytes a row on rings of four and five slots (300 us on 256 x 256, the others 8 to 17 % behind),
// lines asked for three stages ahead (286 to 314), weights straight to registers on eight waves (366), two workgroups a CU (325).
#pragma once

#include <utility>

#include "sg_mx_tile_kernel.h"
#include "sg_wide_kernel.h"

namespace sg {

// dma_1kb_if (sg_wide_kernel.h) with an address a lane: 64 x 16 bytes, lane by lane, to LDS from lds_base on
__device__ __forceinline__ void dma_1kb_v_if(const void* gptr, unsigned lds_base, int on) {
    lds_base = __builtin_amdgcn_readfirstlane(lds_base);
    asm volatile("s_mov_b32 m0, %1\n\ts_cmp_gt_i32 %2, 0\n\ts_cbranch_scc0 .Lmx%=\n\tglobal_load_lds_dwordx4 %0, off\n.Lmx%=:"
                 ::"v"(gptr), "s"(lds_base), "s"(on) : "memory", "m0", "scc");
}

// f(0), ..., f(N - 1) with constant arguments: `#pragma unroll` gives up on the largest tile's stage
template <class F, int... I>
__device__ __forceinline__ void mx_each(F&& f, std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>{}), ...); }
template <int N, class F>
__device__ __forceinline__ void mx_each(F&& f) { mx_each(f, std::make_integer_sequence<int, N>{}); }

template <bool FP4, int RGW, int MH, int DW, int DX>
__global__ void __launch_bounds__(256) mx_wide_kernel(const MxArgs a) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t ring[];   // [DW][W_BYTES] | [DX][X_BYTES] | [2][4 KB] | [2][BM * 16]
    constexpr int S = FP4 ? 2 : 1, U = 4 / S;               // steps of a stage, stages of a group of four steps
    constexpr int BN = 32 * RGW, BM = 32 * MH;
    constexpr int W_BYTES = 2 * RGW * S * 1024, X_BYTES = BM * 128;
    constexpr int WI = 2 * RGW * S / 4, XI = MH;            // 1 KB direct loads of a wave and stage
    static_assert(2 * RGW * S % 4 == 0 && MH % 4 == 0 && RGW <= 8 && MH <= 8, "tile");
    static_assert(DX >= 2 && DX <= DW && DW - 2 <= DX && DX <= U + 1, "rings; a group's scales arrive with the activations behind them");
    constexpr int WR = RGW == 8 ? 4 : RGW, AHEAD = WR > 4 ? 4 : WR - 1, LATE = RGW - AHEAD;
    static_assert(AHEAD < WR && 2 * RGW % WR == 0, "the loop's two stages leave both register rings in phase");
    constexpr int SW_AT = DW * W_BYTES + DX * X_BYTES, SX_AT = SW_AT + 2 * 4096;

    const int lane = lane_id(), wave = wave_id(), wn = wave & 1, wm = wave >> 1;
    const MxPlace place = mx_place(a);
    const int tn = place.tn, tm = place.tm;
    const int m0 = tm * BM, tile0 = tn * 2 * RGW;
    const int all = (a.steps + S - 1) / S, first = place.q0 * U;
    const int stages = (place.q1 * U < all ? place.q1 * U : all) - first;     // this workgroup's, counted from `first`
    const int quads = place.q1 - place.q0;
    const int pieces = FP4 ? a.k / 32 : a.k / 16;           // of an activation row

    // ---- direct loads ----
    // Activations: instruction i covers rows 8 * (4 i + wave) .. + 7; a lane's piece is the same for every i.
    const int d_row = lane >> 3, d_piece = (lane & 7) ^ ((4 * wave + (d_row >> 1)) & 7);
    unsigned xoff[XI];                                      // 32 bits: the launcher refuses rows beyond 8 MB
#pragma unroll
    for (int i = 0; i < XI; i++) {
        const int row = 8 * (4 * i + wave) + d_row;
        xoff[i] = (unsigned)(row < a.m - m0 ? row : a.m - 1 - m0) * (unsigned)(pieces * 16) + d_piece * 16;
    }
    // Beyond the end of a row (the last stage) its last piece: the weights there are zero.
    const int past = 8 * (all - 1) + d_piece - (pieces - 1);
    const unsigned back = past > 0 ? past * 16 : 0;
    const uint8_t* const x_src = a.A + (size_t)m0 * ((size_t)pieces * 16);
    const unsigned lds0 = lds_addr(ring);
    auto issue_x = [&](int i, int s, int slot, int on) __attribute__((always_inline)) {
        const unsigned off = xoff[i] - (first + s == all - 1 ? back : 0u);
        dma_1kb_if<false>(x_src + (size_t)(first + s) * 128, off, lds0 + DW * W_BYTES + (unsigned)slot * X_BYTES + (4 * i + wave) * 1024, on);
    };
    // Weights: 1 KB a (tile, step); instruction i of a wave: the (4 i + wave)-th of the stage, tile by tile
    const unsigned lane16 = lane * 16;
    auto issue_w = [&](int i, int s, int slot, int on) __attribute__((always_inline)) {
        const int e = 4 * i + wave, t = tile0 + e / S < a.tiles ? tile0 + e / S : a.tiles - 1;
        dma_1kb_if<true>(a.P + ((size_t)t * a.pitch + (S * (first + s) + e % S)) * kMxStepBytes, lane16,
                         lds0 + (unsigned)slot * W_BYTES + e * 1024, on);
    };
    // Scales of a group: four tiles an instruction (beyond 2 * RGW tiles a copy that nobody reads), 64 activation rows an
    // instruction (a tile of 128 rows: fetched twice, the same bytes to the same place)
    const int s_tile = tile0 + 4 * wave + (lane >> 4) < a.tiles ? tile0 + 4 * wave + (lane >> 4) : a.tiles - 1;
    const size_t sw_off = (size_t)s_tile * a.quads * kMxQuadBytes + (lane & 15) * 16;
    const int s_row = (64 * wave + lane) % BM;
    const size_t sx_off = FP4 ? (size_t)(m0 + s_row < a.m ? m0 + s_row : a.m - 1) * ((size_t)a.quads * 16) : 0;
    auto issue_scales = [&](int q, int on) __attribute__((always_inline)) {
        dma_1kb_v_if(a.PS + sw_off + (size_t)(place.q0 + q) * kMxQuadBytes, lds0 + SW_AT + (q & 1) * 4096 + wave * 1024, on);
        if (FP4) dma_1kb_v_if(a.SX + sx_off + (size_t)(place.q0 + q) * 16, lds0 + SX_AT + (q & 1) * (BM * 16) + (64 * wave % BM) * 16, on);
    };

    // ---- LDS reads: lane (r, g) ----
    const int r = lane & 15, g = lane >> 4;
    const int rd = r * 128 + ((g ^ ((r >> 1) & 7)) << 4);
    const uint8_t* const w_lds = ring + wn * RGW * S * 1024 + lane * 16;
    const uint8_t* const x_lds = ring + DW * W_BYTES + wm * MH * 2048;
    const uint8_t* const sw_lds = ring + SW_AT + wn * RGW * 256 + lane * 4;
    const uint8_t* const sx_lds = ring + SX_AT + (wm * MH * 16 + r) * 16;
    const unsigned pick = (unsigned)g | (unsigned)(4 + g) << 8;         // of a row's 8 scales of a stage: one a step

    const int one = mx_scale_one();
    f32x4 acc[RGW][MH];
#pragma unroll
    for (int i = 0; i < RGW; i++)
#pragma unroll
        for (int j = 0; j < MH; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    i32x4 w[WR][S];
    int ws[WR];
    i32x8 x8[2][FP4 ? 1 : MH];
    i32x4 x4[2][FP4 ? MH : 1][2];
    u32x2 xraw[FP4 ? MH : 1];
    int xs[FP4 ? MH : 1];

    // part p of weight fragment i of the stage whose operands lie at wb, its scales at sb: codes, then the scales
    auto read_w = [&](int slot, int p, int i, const uint8_t* wb, const uint8_t* sb) __attribute__((always_inline)) {
        if (p < S) w[slot][p] = *reinterpret_cast<const i32x4*>(wb + (i * S + p) * 1024);
        else ws[slot] = FP4 ? *reinterpret_cast<const uint16_t*>(sb + i * 256) : *(sb + i * 256);
    };
    auto read_x = [&](int set, int p, int j, const uint8_t* xb, const uint8_t* sb) __attribute__((always_inline)) {
        if (p == 2) {
            if constexpr (FP4) xraw[j] = *reinterpret_cast<const u32x2*>(sb + j * 256);
            return;
        }
        const i32x4 v = *reinterpret_cast<const i32x4*>(xb + j * 2048 + (p ? rd ^ 64 : rd));
        if constexpr (FP4) {
            x4[set][j][p] = v;
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) x8[set][j][p * 4 + e] = v[e];
        }
    };
    constexpr int WP = S + 1, XP = FP4 ? 3 : 2;             // reads of a fragment
    auto w_scales = [&](int s) { return sw_lds + ((s / U) & 1) * 4096 + (s % U) * S; };
    auto x_scales = [&](int s) { return sx_lds + ((s / U) & 1) * (BM * 16) + (s % U) * 8; };

    // Refill group j: scales (where stage j ends a group of steps) and activations of stage j + DX behind the barrier of stage j,
    // weights of stage j + DW in front of the barrier of stage j + 1.  In front of the barrier of stage s, behind the
    // last instruction of X(s + 1) and of W(s + 1), the queue holds at least this many younger ones:
    constexpr int PER = WI + XI;
    constexpr int IN_FLIGHT = (WI + (DX - 2) * PER) < (DW - 2) * PER ? (WI + (DX - 2) * PER) : (DW - 2) * PER;
    static_assert(IN_FLIGHT <= 63, "vmcnt");

    issue_scales(0, 1);
    issue_scales(1, quads - 1);
#pragma unroll
    for (int j = -DW; j < 0; j++) {
        if (j + DX >= 0) {
#pragma unroll
            for (int i = 0; i < XI; i++) issue_x(i, j + DX, j + DX, stages - (j + DX));
        }
        if (j < -1) {
#pragma unroll
            for (int i = 0; i < WI; i++) issue_w(i, j + DW, j + DW, stages - (j + DW));
        }
    }
    wait_vmcnt_if<IN_FLIGHT>(stages - DW + 1);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < AHEAD; i++)
#pragma unroll
        for (int p = 0; p < WP; p++) read_w(i, p, i, w_lds, w_scales(0));
#pragma unroll
    for (int j = 0; j < MH; j++)
#pragma unroll
        for (int p = 0; p < XP; p++) read_x(0, p, j, x_lds, x_scales(0));

    int slot_w = 0, slot_x = 0;
    // stage s, of parity u: products of x?[u] and of the weight ring from index u * RGW on
    auto stage = [&](int s, auto uc) __attribute__((always_inline)) {
        constexpr int u = decltype(uc)::value;
        const int next_w = slot_w + 1 == DW ? 0 : slot_w + 1, next_x = slot_x + 1 == DX ? 0 : slot_x + 1;
        const int prev_w = slot_w == 0 ? DW - 1 : slot_w - 1;
        const uint8_t* const wcur = w_lds + slot_w * W_BYTES;
        const uint8_t* const wnext = w_lds + next_w * W_BYTES;
        const uint8_t* const xnext = x_lds + next_x * X_BYTES;
        const uint8_t* const swcur = w_scales(s);
        const uint8_t* const swnext = w_scales(s + 1);
        const uint8_t* const sxnext = x_scales(s + 1);
        const int fill_w = stages - (s - 1 + DW), fill_x = stages - (s + DX);   // positive: there is such a stage
        const int fill_s = s % U == U - 1 ? quads - (s / U + 2) : 0;
        if constexpr (FP4) {
#pragma unroll
            for (int j = 0; j < MH; j++) xs[j] = (int)__builtin_amdgcn_perm(xraw[j].y, xraw[j].x, pick);
        }
        mx_each<RGW>([&](auto ic) __attribute__((always_inline)) {
            constexpr int i = decltype(ic)::value;
            if (i == LATE) {
                // this wave's reads of stage s have arrived, its loads of stage s + 1 have landed; behind the barrier that
                // holds for all waves
                wait_vmcnt_if<IN_FLIGHT>(fill_w);
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
                __builtin_amdgcn_sched_barrier(0);
                issue_scales(s / U + 2, fill_s);
            }
            constexpr int ring_at = (u * RGW + i) % WR;
            mx_each<MH * S>([&](auto ec) __attribute__((always_inline)) {
                constexpr int e = decltype(ec)::value;
                // weight fragment i + AHEAD, of this stage or the next, in the first slots of the group
                if (e < WP) {
                    const bool here = i + AHEAD < RGW;
                    read_w((u * RGW + i + AHEAD) % WR, e, here ? i + AHEAD : i + AHEAD - RGW, here ? wcur : wnext, here ? swcur : swnext);
                }
                constexpr int FREE = MH * S - WP;            // the other slots of a group
                if (e >= WP && i >= LATE) {
                    constexpr int Q = AHEAD * FREE, OPS = XP * MH + XI;
                    const int q = (i - LATE) * FREE + e - WP;
#pragma unroll
                    for (int op = wide_first_op(q, Q, OPS); op < wide_first_op(q + 1, Q, OPS); op++) {
                        const int read = op < 2 * XI ? op / 2 : op - XI;
                        if (op < 2 * XI && op % 2 == 0) issue_x(op / 2, s + DX, slot_x, fill_x);
                        else read_x((u + 1) & 1, read % XP, read / XP, xnext, sxnext);
                    }
                }
                if (e >= WP && i < LATE) {
                    constexpr int Q = LATE * FREE;
                    const int q = i * FREE + e - WP;
#pragma unroll
                    for (int op = wide_first_op(q, Q, WI); op < wide_first_op(q + 1, Q, WI); op++) issue_w(op, s - 1 + DW, prev_w, fill_w);
                }
                __builtin_amdgcn_sched_barrier(0);
                const int j = e % MH;
                if constexpr (FP4) {
                    if constexpr (e < MH) mfma_mx_acc<i == 0 && e == 0, 0, 0>(acc[i][j], w[ring_at][0], x4[u][j][0], ws[ring_at], xs[j]);
                    else mfma_mx_acc<false, 1, 1>(acc[i][j], w[ring_at][S - 1], x4[u][j][1], ws[ring_at], xs[j]);
                } else {
                    mfma_mx_acc<i == 0 && e == 0, 0>(acc[i][j], w[ring_at][0], x8[u][j], ws[ring_at], one);
                }
                __builtin_amdgcn_sched_barrier(0);
            });
        });
        mx_drain(acc);
        slot_w = next_w;
        slot_x = next_x;
    };
    int s = 0;
    for (; s + 1 < stages; s += 2) {
        stage(s, std::integral_constant<int, 0>{});
        stage(s + 1, std::integral_constant<int, 1>{});
    }
    if (s < stages) stage(s, std::integral_constant<int, 0>{});
    __syncthreads();

    if (a.splits > 1) {
#pragma unroll
        for (int j = 0; j < MH; j++)
#pragma unroll
            for (int i = 0; i < RGW; i++) {
                keep_in_accumulator(acc[i][j]);
                mx_put(a, place.split, tile0 + wn * RGW + i, (tm * 2 + wm) * MH + j, lane, acc[i][j], 1.0f);
            }
        return;
    }
    // ---- epilogue: the wave turns its tile around in LDS and stores runs of 32 * RGW bytes a row ----
    const float scale = a.scale ? a.scale[0] : 1.0f;
    constexpr int PITCH = 32 * RGW + 16, ROWS = 16 * MH;
    uint8_t* const mine = ring + (size_t)wave * (ROWS * PITCH);
    const int m_wave = m0 + wm * ROWS, n_wave = (tile0 + wn * RGW) * 16;
#pragma unroll
    for (int j = 0; j < MH; j++) {
        const int m_idx = m_wave + j * 16 + r;
        const float row = a.row_scale && m_idx < a.m ? a.row_scale[m_idx] : 1.0f;
#pragma unroll
        for (int i = 0; i < RGW; i++) {
            keep_in_accumulator(acc[i][j]);
            f32x4 v = acc[i][j] * scale;
            v *= row;
            *reinterpret_cast<u32x2*>(mine + (j * 16 + r) * PITCH + i * 32 + 8 * g) = u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
        }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    constexpr int PIECES = 2 * RGW;                         // 16-byte pieces of a row
    using u32x4_at2 = u32x4 __attribute__((aligned(2)));    // n may be odd
#pragma unroll 4
    for (int p = lane; p < ROWS * PIECES; p += 64) {
        const int row = p / PIECES, c = p - row * PIECES;
        const int m_idx = m_wave + row, n_idx = n_wave + 8 * c;
        if (m_idx >= a.m || n_idx >= a.n) continue;
        uint16_t* const to = a.D + (size_t)m_idx * a.n + n_idx;
        const u32x4 v = *reinterpret_cast<const u32x4*>(mine + row * PITCH + 16 * c);
        if (n_idx + 8 <= a.n) {
            *reinterpret_cast<u32x4_at2*>(to) = v;
        } else {
#pragma unroll
            for (int e = 0; e < 7; e++)
                if (n_idx + e < a.n) to[e] = (uint16_t)(v[e / 2] >> (16 * (e & 1)));
        }
    }
}

constexpr size_t mx_wide_lds(bool fp4, int rgw, int mh, int dw, int dx) {
    const size_t rings = (size_t)dw * 2 * rgw * (fp4 ? 2 : 1) * 1024 + (size_t)dx * 32 * mh * 128 + 2 * 4096 + (fp4 ? 2 * 32 * mh * 16 : 0);
    const size_t turn = (size_t)4 * 16 * mh * (32 * rgw + 16);
    return rings > turn ? rings : turn;
}

}  // namespace sg
