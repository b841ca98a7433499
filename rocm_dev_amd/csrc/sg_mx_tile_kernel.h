// Products with MXFP4 weights on tiles of many activation rows:  D[m,n] = bf16(scale * row[m] * sum_k A[m,k] * B[n,k]).
//
// A workgroup of WN x WM waves owns 16 * NF * WN weight rows by 16 * MF * WM activation rows, a wave NF x MF fragments of
// 16 x 16.  A stage is 128 bytes of every activation row: 128 columns of E4M3 (one step of the matrix instruction) or 256 of
// MXFP4 (two).  The activations of a stage, which all waves along n read, go through LDS, two buffers, one barrier a stage (and
// through registers, so that the compiler's own waits order everything); the weights, which only the WM waves along m share, go
// straight to registers by contiguous KBs of the packed buffer (sg_mx.h): through LDS they would be a quarter (E4M3) to a half
// (MXFP4) of its traffic.
//
// LDS: row x 128 bytes, the 16-byte piece p of row x at p ^ ((x / 2) % 8), so that the 16 rows of a fragment's read meet all
// banks; lane (r, g) reads pieces g and g + 4 - of E4M3 the 32 columns the instruction wants of it, of MXFP4 block g of
// each of the stage's two steps.  MXFP4's block scales lie beside, 8 bytes a row in the order a lane reads them: 2 bytes, one a step.
//
// What bounds it is how much a CU has in flight: a weight stage asked for one stage ahead leaves a workgroup waiting for most of an
// HBM round trip, so small tiles hold four stages of weights in registers (E4M3 activations on 64 x 32: 100 x 10944 x 3712 16.9 -> 14.0 us,
// 32 x 28672 x 4096 20.6 -> 15.6); 128 x 128 tiles have no registers for that and run several workgroups a CU.
#pragma once

#include "sg_mx_kernel.h"

namespace sg {

// The matrix instruction as text, accumulators in the accumulation registers: the builtin, which has no form that adds in place
// for mixed formats, gives every accumulator of the tile two to four homes.  Scale bytes T of ws and XT of xs.
//
// The compiler knows none of its waits.  An operand that a vector instruction wrote has to be two states old: IDLE puts two idle
// states in front of a stage's first product, and nothing else writes one so late - with them in front of every product a
// launch of the wide kernel is 3 to 8 % longer (1024 x 10240 x 8192, MXFP4, 58.7 us, 53.8 without).  A result takes up to 19: mx_drain
// ends every stage with as many, and inside a stage an accumulator is touched by these instructions only.
// tests/test_mx_codegen.py checks both in the assembly.
template <bool IDLE, int T, int XT>
__device__ __forceinline__ void mfma_mx_acc(f32x4& c, const i32x4& w, const i32x4& x, int ws, int xs) {
    if constexpr (IDLE)
        asm volatile("s_nop 1\n\tv_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[%5,%6,0] op_sel_hi:[%7,%8,0] cbsz:4 blgp:4"
                     : "+a"(c) : "v"(w), "v"(x), "v"(ws), "v"(xs), "n"(T & 1), "n"(XT & 1), "n"(T >> 1), "n"(XT >> 1));
    else
        asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[%5,%6,0] op_sel_hi:[%7,%8,0] cbsz:4 blgp:4"
                     : "+a"(c) : "v"(w), "v"(x), "v"(ws), "v"(xs), "n"(T & 1), "n"(XT & 1), "n"(T >> 1), "n"(XT >> 1));
}
template <bool IDLE, int T>
__device__ __forceinline__ void mfma_mx_acc(f32x4& c, const i32x4& w, const i32x8& x, int ws, int xs) {
    if constexpr (IDLE)
        asm volatile("s_nop 1\n\tv_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[%5,0,0] op_sel_hi:[%6,0,0] cbsz:4"
                     : "+a"(c) : "v"(w), "v"(x), "v"(ws), "v"(xs), "n"(T & 1), "n"(T >> 1));
    else
        asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[%5,0,0] op_sel_hi:[%6,0,0] cbsz:4"
                     : "+a"(c) : "v"(w), "v"(x), "v"(ws), "v"(xs), "n"(T & 1), "n"(T >> 1));
}
// scale 1 of E4M3 activations, in a register that the compiler cannot write anew in front of a product
__device__ __forceinline__ int mx_scale_one() {
    int one = 127;
    asm volatile("" : "+v"(one));
    return one;
}
template <int NF, int MF>
__device__ __forceinline__ void mx_drain(f32x4 (&acc)[NF][MF]) {
    asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
    // what follows uses the values of these, so a copy that the compiler makes stands behind the idle states
#pragma unroll
    for (int i = 0; i < NF; i++)
#pragma unroll
        for (int j = 0; j < MF; j++) asm volatile("" : "+a"(acc[i][j]));
}

// WR: ring of weight stages in registers, asked for WR - 1 stages ahead; XR: of activation stages on their way to LDS, XR ahead.
template <bool FP4, int NF, int MF, int WN, int WM, int WR, int XR>
__global__ void __launch_bounds__(64 * WN * WM) mx_tile_kernel(const MxArgs a) {
    static_assert((WR == 2 && XR == 1) || (WR == 4 && XR == 2), "the loops' unrolled stages leave both rings and the LDS buffers in phase");
    constexpr int THREADS = 64 * WN * WM, BM = 16 * MF * WM;
    constexpr int S = FP4 ? 2 : 1;                       // steps of a stage
    constexpr int U = 4 / S;                             // stages of a group of four steps
    constexpr int PIECES = BM * 8 / THREADS;             // 16-byte pieces of a stage that a thread brings
    static_assert(BM * 8 % THREADS == 0 && (!FP4 || THREADS >= BM), "tile");
    constexpr int BUF = BM * 128 + (FP4 ? BM * 8 : 0);
    __shared__ __attribute__((aligned(128))) uint8_t lds[2 * BUF];

    const int tid = threadIdx.x, lane = lane_id(), r = lane & 15, g = lane >> 4;
    const int wave = wave_id(), wn = wave % WN, wm = wave / WN;
    const MxPlace place = mx_place(a);
    const int tn = place.tn, tm = place.tm;
    const int m0 = tm * BM, tile0 = (tn * WN + wn) * NF;
    const int k_blocks = a.k / kMxBlock;
    const int pieces = FP4 ? k_blocks : 2 * k_blocks;    // of an activation row
    const int first = place.q0 * U, stages = (place.q1 * U < (a.steps + S - 1) / S ? place.q1 * U : (a.steps + S - 1) / S);   // [first, stages)

    // ---- activations: memory -> registers -> LDS ----
    const uint8_t* xp[PIECES];
    int xlds[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; i++) {
        const int row = (i * THREADS + tid) >> 3, p = tid & 7;
        xp[i] = a.A + (size_t)(m0 + row < a.m ? m0 + row : a.m - 1) * ((size_t)pieces * 16);
        xlds[i] = row * 128 + ((p ^ ((row >> 1) & 7)) << 4);
    }
    const uint8_t* sp = FP4 && tid < BM ? a.SA + (size_t)(m0 + tid < a.m ? m0 + tid : a.m - 1) * k_blocks : nullptr;
    i32x4 xr[XR][PIECES];
    u32x2 sr[XR];
    auto load_x = [&](int s, auto qc) __attribute__((always_inline)) {
        constexpr int q = decltype(qc)::value;
#pragma unroll
        for (int i = 0; i < PIECES; i++) {
            const int p = 8 * s + (tid & 7);
            xr[q][i] = *reinterpret_cast<const i32x4*>(xp[i] + (size_t)(p < pieces ? p : pieces - 1) * 16);
        }
        if (FP4 && tid < BM) {
            if (8 * s + 8 <= k_blocks) {
                __builtin_memcpy(&sr[q], sp + 8 * s, 8);
            } else {
                sr[q] = u32x2{0, 0};
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int b = 8 * s + e < k_blocks ? 8 * s + e : k_blocks - 1;
                    sr[q][e / 4] |= (uint32_t)sp[b] << (8 * (e % 4));
                }
            }
        }
    };
    auto store_x = [&](int s, uint8_t* buf, auto qc) __attribute__((always_inline)) {
        constexpr int q = decltype(qc)::value;
        // a piece beyond the row's end is zero: whatever weights it meets, under the scale of the row's own last block
        const bool beyond = 8 * s + (tid & 7) >= pieces;
#pragma unroll
        for (int i = 0; i < PIECES; i++) *reinterpret_cast<i32x4*>(buf + xlds[i]) = beyond ? i32x4{0, 0, 0, 0} : xr[q][i];
        if (FP4 && tid < BM) {
            const uint32_t lo = sr[q].x, hi = sr[q].y;           // blocks 0-3 and 4-7 -> 0 4 1 5, 2 6 3 7
            *reinterpret_cast<u32x2*>(buf + BM * 128 + tid * 8) =
                u32x2{__builtin_amdgcn_perm(hi, lo, 0x05010400u), __builtin_amdgcn_perm(hi, lo, 0x07030602u)};
        }
    };

    // ---- weights ----
    const uint8_t* wp[NF];
    const uint8_t* wsp[NF];
#pragma unroll
    for (int i = 0; i < NF; i++) {
        const int tile = tile0 + i < a.tiles ? tile0 + i : a.tiles - 1;
        wp[i] = a.P + (size_t)tile * a.pitch * kMxStepBytes + lane * 16;
        wsp[i] = a.PS + (size_t)tile * a.quads * kMxQuadBytes + lane * 4;
    }
    i32x4 w[WR][S][NF];
    int ws[NF], ws_next[NF];
    auto load_w = [&](int s, auto bc) __attribute__((always_inline)) {
        constexpr int b = decltype(bc)::value;
#pragma unroll
        for (int t = 0; t < S; t++) {
            const int step = S * s + t < a.steps ? S * s + t : a.steps - 1;
#pragma unroll
            for (int i = 0; i < NF; i++) w[b][t][i] = *reinterpret_cast<const i32x4*>(wp[i] + (size_t)step * kMxStepBytes);
        }
    };
    auto load_ws = [&](int q) __attribute__((always_inline)) {
        const int qq = q < a.quads ? q : a.quads - 1;
#pragma unroll
        for (int i = 0; i < NF; i++) ws_next[i] = *reinterpret_cast<const int*>(wsp[i] + (size_t)qq * kMxQuadBytes);
    };

    const int one = mx_scale_one();
    f32x4 acc[NF][MF];
#pragma unroll
    for (int i = 0; i < NF; i++)
#pragma unroll
        for (int j = 0; j < MF; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    const int rd = r * 128 + ((g ^ ((r >> 1) & 7)) << 4);
    auto multiply = [&](const uint8_t* buf, auto bc) __attribute__((always_inline)) {
        constexpr int b = decltype(bc)::value;             // of the weight ring
#pragma unroll
        for (int j = 0; j < MF; j++) {
            const uint8_t* x = buf + (wm * MF + j) * 2048 + rd;
            const i32x4 lo = *reinterpret_cast<const i32x4*>(x);
            const i32x4 hi = *reinterpret_cast<const i32x4*>(buf + (wm * MF + j) * 2048 + (rd ^ 64));
            if constexpr (FP4) {
                const int xs = *reinterpret_cast<const uint16_t*>(buf + BM * 128 + ((wm * MF + j) * 16 + r) * 8 + g * 2);
#pragma unroll
                for (int i = 0; i < NF; i++) {
                    if (i == 0 && j == 0) mfma_mx_acc<true, 0, 0>(acc[i][j], w[b][0][i], lo, ws[i], xs);
                    else mfma_mx_acc<false, 0, 0>(acc[i][j], w[b][0][i], lo, ws[i], xs);
                }
#pragma unroll
                for (int i = 0; i < NF; i++) mfma_mx_acc<false, 1, 1>(acc[i][j], w[b][S - 1][i], hi, ws[i], xs);
            } else {
                const i32x8 x8 = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
                for (int i = 0; i < NF; i++) {
                    if (i == 0 && j == 0) mfma_mx_acc<true, 0>(acc[i][j], w[b][0][i], x8, ws[i], one);
                    else mfma_mx_acc<false, 0>(acc[i][j], w[b][0][i], x8, ws[i], one);
                }
            }
        }
        mx_drain(acc);
    };

    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    const auto in = [&](int s) __attribute__((always_inline)) { return s < stages ? s : stages - 1; };
    load_x(first, I0{});
    load_ws(place.q0);
    load_w(first, I0{});
    store_x(first, lds, I0{});
    load_x(in(first + 1), std::integral_constant<int, 1 % XR>{});
    if constexpr (XR == 2) load_x(in(first + 2), I0{});
    if constexpr (WR == 4) {
        load_w(in(first + 1), I1{});
        load_w(in(first + 2), std::integral_constant<int, 2 % WR>{});
    }
    __syncthreads();

    // Stage s, the c-th of the unrolled ones: the next stage's activations from registers to the other buffer, loads (LAST: where
    // there is such a stage) into what that frees, then the products.  The other buffer was last read in front of the barrier.
    auto stage = [&](int s, auto cc, auto lc) __attribute__((always_inline)) {
        constexpr int c = decltype(cc)::value, x = (c + 1) % XR;
        constexpr bool LAST = decltype(lc)::value;
        store_x(s + 1, lds + (c & 1 ? 0 : BUF), std::integral_constant<int, x>{});
        if (!LAST || s + 1 + XR < stages) load_x(s + 1 + XR, std::integral_constant<int, x>{});
        if (!LAST || s + WR - 1 < stages) load_w(s + WR - 1, std::integral_constant<int, (c + WR - 1) % WR>{});
        if (s % U == 0) {
#pragma unroll
            for (int i = 0; i < NF; i++) ws[i] = ws_next[i];
            load_ws(s / U + 1);
        }
        multiply(lds + (c & 1 ? BUF : 0), std::integral_constant<int, c % WR>{});
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NF; i++) ws[i] = (int)((unsigned)ws[i] >> (8 * S));      // the next stage's scales to the low bytes
    };
    constexpr std::false_type MORE{};
    constexpr std::true_type LAST{};
    constexpr int REACH = WR - 1 > 1 + XR ? WR - 1 : 1 + XR;      // the farthest stage that a stage's loads are of
    int s = first;                                       // a multiple of U: even
    for (; s + 3 + REACH < stages; s += 4) {             // every load is of a stage there is
        stage(s, I0{}, MORE);
        stage(s + 1, I1{}, MORE);
        stage(s + 2, std::integral_constant<int, 2>{}, MORE);
        stage(s + 3, std::integral_constant<int, 3>{}, MORE);
    }
    for (; s < stages; s += 4) {
        stage(s, I0{}, LAST);
        if (s + 1 < stages) stage(s + 1, I1{}, LAST);
        if (s + 2 < stages) stage(s + 2, std::integral_constant<int, 2>{}, LAST);
        if (s + 3 < stages) stage(s + 3, std::integral_constant<int, 3>{}, LAST);
    }

    const float scale = a.scale ? a.scale[0] : 1.0f;
#pragma unroll
    for (int j = 0; j < MF; j++)
#pragma unroll
        for (int i = 0; i < NF; i++) mx_put(a, place.split, tile0 + i, (tm * WM + wm) * MF + j, lane, acc[i][j], scale);
}

}  // namespace sg
