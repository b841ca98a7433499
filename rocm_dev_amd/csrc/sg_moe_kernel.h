// The experts of a mixture-of-experts layer for a few tokens: E4M3 weights with a scale a row, bf16 activations.
//
// What bounds it is the stream of the reached experts' weights, a byte a value, read once.  The codes are widened on the way to bf16
// (v_cvt_scalef32_pk_bf16_fp8, two a lane and instruction, exact) and multiplied by v_mfma_f32_16x16x32_bf16: activations keep
// their 16 bits, and the products lose nothing that fp32 sums hold.  An expert's tokens are the columns of the product, 16 at a
// time: MB blocks of 16.
//
// Lane (r, g) of a wave takes row r of a 16-row tile and, of a step of 128 columns, columns 16 g .. + 15 and 64 + 16 g .. + 15: 16 contiguous bytes
// each, two instructions each; the activations' lanes take the same columns, 32 contiguous bytes each.
#pragma once

#include "sg_moe.h"

namespace sg {

typedef __bf16 moe_bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 moe_bf16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4 moe_mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(moe_bf16x8, a), __builtin_bit_cast(moe_bf16x8, b), c, 0, 0, 0);
}
// eight E4M3 codes as bf16
__device__ __forceinline__ u32x4 moe_widen(uint32_t lo, uint32_t hi) {
    u32x4 v;
    v[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false));
    v[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true));
    v[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false));
    v[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true));
    return v;
}

// A step of 128 columns of RT row tiles and MB activation blocks.
template <int RT, int MB>
struct MoeStep {
    u32x4 w[RT][2], x[MB][2][2];

    // wp, xp: the lane's rows (16-byte aligned); pieces: 16-column pieces a row; a piece beyond the row's end is the last one again.
    __device__ __forceinline__ void load(const uint8_t* const (&wp)[RT], const uint8_t* const (&xp)[MB], int blocks, int step, int pieces) {
        const int g = lane_id() >> 4;
        int p[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            p[h] = 8 * step + 4 * h + g;
            p[h] = p[h] < pieces ? p[h] : pieces - 1;
        }
#pragma unroll
        for (int i = 0; i < RT; i++)
#pragma unroll
            for (int h = 0; h < 2; h++) w[i][h] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(wp[i] + (size_t)p[h] * 16));
#pragma unroll
        for (int j = 0; j < MB; j++)
            if (j < blocks || MB == 1)
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int u = 0; u < 2; u++) x[j][h][u] = *reinterpret_cast<const u32x4*>(xp[j] + (size_t)p[h] * 32 + 16 * u);
    }
    __device__ __forceinline__ void multiply(f32x4 (&acc)[RT][MB], int blocks, int step, int pieces) {
        const int g = lane_id() >> 4;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const bool inside = 8 * step + 4 * h + g < pieces;
#pragma unroll
            for (int u = 0; u < 2; u++) {
                u32x4 v[RT];
#pragma unroll
                for (int i = 0; i < RT; i++) {
                    v[i] = moe_widen(w[i][h][2 * u], w[i][h][2 * u + 1]);
                    // beyond the row's end: zeros on both sides, so that no infinity or NaN of the last piece counts twice
                    if (!inside) v[i] = u32x4{0, 0, 0, 0};
                }
#pragma unroll
                for (int j = 0; j < MB; j++)
                    if (j < blocks || MB == 1) {
                        const u32x4 y = inside ? x[j][h][u] : u32x4{0, 0, 0, 0};
#pragma unroll
                        for (int i = 0; i < RT; i++) acc[i][j] = moe_mfma(v[i], y, acc[i][j]);
                    }
            }
        }
        __builtin_amdgcn_sched_barrier(0);       // steps are not mixed: their temporaries would not fit
    }
};

// A product's result may be read 12 wait states behind it, counted across branches here: the ties keep products in front of the
// idle states and uses behind them.
template <int RT, int MB>
__device__ __forceinline__ void moe_settle(f32x4 (&acc)[RT][MB]) {
#pragma unroll
    for (int i = 0; i < RT; i++)
#pragma unroll
        for (int j = 0; j < MB; j++) asm volatile("" : "+v"(acc[i][j]));
    asm volatile("s_nop 11" ::: "memory");
#pragma unroll
    for (int i = 0; i < RT; i++)
#pragma unroll
        for (int j = 0; j < MB; j++) asm volatile("" : "+v"(acc[i][j]));
}

// Steps begin, begin + stride, ... below `end` of one product, two in flight.
template <int RT, int MB>
__device__ __forceinline__ void moe_product(f32x4 (&acc)[RT][MB], const uint8_t* const (&wp)[RT], const uint8_t* const (&xp)[MB], int blocks,
                                            int begin, int stride, int end, int pieces) {
    MoeStep<RT, MB> s0, s1;
    int step = begin;
    if (step < end) s0.load(wp, xp, blocks, step, pieces);
    if (step + stride < end) s1.load(wp, xp, blocks, step + stride, pieces);
    for (; step + 3 * stride < end; step += 2 * stride) {
        s0.multiply(acc, blocks, step, pieces);
        s0.load(wp, xp, blocks, step + 2 * stride, pieces);
        s1.multiply(acc, blocks, step + stride, pieces);
        s1.load(wp, xp, blocks, step + 3 * stride, pieces);
    }
    if (step >= end) return;
    s0.multiply(acc, blocks, step, pieces);
    if (step + 2 * stride < end) s0.load(wp, xp, blocks, step + 2 * stride, pieces);
    if (step + stride < end) s1.multiply(acc, blocks, step + stride, pieces);
    if (step + 2 * stride < end) s0.multiply(acc, blocks, step + 2 * stride, pieces);
}

// v / (1 + exp(-v)), by the exponential that does not overflow
__device__ __forceinline__ float moe_silu(float v) {
    const float t = expf(-fabsf(v));
    return v * ((v < 0.0f ? t : 1.0f) / (1.0f + t));
}

// The plan in LDS
__device__ __forceinline__ void moe_take_plan(const MoeArgs& a, int32_t* plan, int dwords) {
    for (int i = (int)threadIdx.x * 4; i < dwords; i += (int)blockDim.x * 4)
        *reinterpret_cast<i32x4*>(plan + i) = *reinterpret_cast<const i32x4*>(a.plan + i);
    __syncthreads();
}

// h = bf16( silu(S1 * (gate x)) * (S1 * (up x)) ): a workgroup's waves share hidden of 16 gate rows and their 16 up rows.
// LDS: plan, then [waves][2 * MB][64 lanes] f32x4.
template <int MB>
__global__ void __launch_bounds__(512) moe_gate_up_kernel(const MoeArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    int32_t* const plan = reinterpret_cast<int32_t*>(lds);
    const MoePlanLayout l = moe_plan_layout(a.m, a.experts, a.top_k);
    f32x4* const part = reinterpret_cast<f32x4*>(lds + (size_t)l.dwords * 4);
    const int lane = lane_id(), r = lane & 15, g = lane >> 4, wave = wave_id(), waves = (int)(blockDim.x >> 6);
    moe_take_plan(a, plan, l.dwords);
    const int tiles = a.inner / 16, items = plan[0] * tiles;
    const int pieces = a.hidden / 16, steps = (a.hidden + 127) / 128;
    for (int item = (int)blockIdx.x; item < items; item += (int)gridDim.x) {
        const int which = item / tiles, tile = item - which * tiles;
        const int packed = plan[l.experts_at + which], e = packed & 0xffff, count = packed >> 16;
        const int32_t* const rows = plan + l.rows_at + plan[l.first_at + which];
        const int blocks = (count + 15) / 16;
        const size_t row = (size_t)e * 2 * a.inner + tile * 16;
        const uint8_t* const wp[2] = {a.W1 + (row + r) * a.hidden, a.W1 + (row + a.inner + r) * a.hidden};
        const uint8_t* xp[MB];
#pragma unroll
        for (int j = 0; j < MB; j++) xp[j] = a.X + (size_t)(rows[16 * j + r < count ? 16 * j + r : count - 1] / a.top_k) * a.hidden * 2;
        f32x4 acc[2][MB];
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int j = 0; j < MB; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        moe_product<2, MB>(acc, wp, xp, blocks, wave, waves, steps, pieces);
        moe_settle(acc);
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int j = 0; j < MB; j++) part[(wave * 2 * MB + i * MB + j) * 64 + lane] = acc[i][j];
        __syncthreads();
        for (int j = wave; j < blocks; j += waves) {
            f32x4 gate = part[j * 64 + lane], up = part[(MB + j) * 64 + lane];
            for (int w = 1; w < waves; w++) {
                gate += part[(w * 2 * MB + j) * 64 + lane];
                up += part[(w * 2 * MB + MB + j) * 64 + lane];
            }
            if (16 * j + r < count) {
                float h[4];
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const float s = a.S1 ? a.S1[row + 4 * g + c] : 1.0f, t = a.S1 ? a.S1[row + a.inner + 4 * g + c] : 1.0f;
                    const float v = gate[c] * s;
                    h[c] = moe_silu(v) * (up[c] * t);
                }
                const u32x2 o = {pack_bf16x2(h[0], h[1]), pack_bf16x2(h[2], h[3])};
                *reinterpret_cast<u32x2*>(a.H + ((size_t)rows[16 * j + r] * a.inner + tile * 16 + 4 * g) * 2) = o;
            }
        }
        __syncthreads();
    }
}

// D = bf16( sum over experts of weight * S2 * (W2 h) ): a workgroup has 16 rows of hidden for all tokens, its waves share the reached
// experts' steps.  A wave adds an expert's product, scaled, to sums of its own - [tokens][16 rows] in LDS, where no other wave and no
// second lane writes -, the waves' sums are added in wave order: no atomics, one order.
// LDS: plan, S2 of the tile [experts reached][16], then [waves][m][16] floats.
template <int MB>
__global__ void __launch_bounds__(512) moe_down_kernel(const MoeArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    int32_t* const plan = reinterpret_cast<int32_t*>(lds);
    const MoePlanLayout l = moe_plan_layout(a.m, a.experts, a.top_k);
    float* const total = reinterpret_cast<float*>(lds + (size_t)l.dwords * 4);
    const int lane = lane_id(), r = lane & 15, g = lane >> 4, wave = wave_id(), waves = (int)(blockDim.x >> 6);
    const int tile = xcd_order((int)blockIdx.x, (int)gridDim.x);
    for (int i = (int)threadIdx.x; i < waves * a.m * 16; i += (int)blockDim.x) total[i] = 0.0f;
    moe_take_plan(a, plan, l.dwords);
    const int reached = plan[0], pieces = a.inner / 16, steps = (a.inner + 127) / 128;
    float* const own = total + wave * a.m * 16;
    // this wave's share of all experts' steps
    const long long all = (long long)reached * steps;
    const long long begin = all * wave / waves, end = all * (wave + 1) / waves;
    int which = (int)(begin / steps), from = (int)(begin - (long long)which * steps);
    for (long long at = begin; at < end; which++, from = 0) {
        const int to = end - at < steps - from ? from + (int)(end - at) : steps;
        const int packed = plan[l.experts_at + which], e = packed & 0xffff, count = packed >> 16, first = plan[l.first_at + which];
        const int blocks = (count + 15) / 16;
        const uint8_t* const wp[1] = {a.W2 + ((size_t)e * a.hidden + tile * 16 + r) * a.inner};
        const uint8_t* xp[MB];
        f32x4 acc[1][MB];
#pragma unroll
        for (int j = 0; j < MB; j++) {
            xp[j] = a.H + (size_t)plan[l.rows_at + first + (16 * j + r < count ? 16 * j + r : count - 1)] * a.inner * 2;
            acc[0][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        moe_product<1, MB>(acc, wp, xp, blocks, from, 1, to, pieces);
        moe_settle(acc);
        f32x4 scale = {1.f, 1.f, 1.f, 1.f};
        if (a.S2)
#pragma unroll
            for (int c = 0; c < 4; c++) scale[c] = a.S2[(size_t)e * a.hidden + tile * 16 + 4 * g + c];
#pragma unroll
        for (int j = 0; j < MB; j++)
            if (16 * j + r < count) {
                const int entry = first + 16 * j + r, token = plan[l.rows_at + entry] / a.top_k;
                const float weight = __uint_as_float((uint32_t)plan[l.weights_at + entry]);
                f32x4* const sum = reinterpret_cast<f32x4*>(own + token * 16 + 4 * g);
                *sum += acc[0][j] * scale * weight;
            }
        at += to - from;
    }
    __syncthreads();
    for (int i = (int)threadIdx.x; i < a.m * 4; i += (int)blockDim.x) {
        const int token = i >> 2, c = i & 3;
        f32x4 v = *reinterpret_cast<const f32x4*>(total + token * 16 + 4 * c);
        for (int w = 1; w < waves; w++) v += *reinterpret_cast<const f32x4*>(total + (w * a.m + token) * 16 + 4 * c);
        const u32x2 o = {pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
        *reinterpret_cast<u32x2*>(a.D + (size_t)token * a.hidden + tile * 16 + 4 * c) = o;
    }
}

}  // namespace sg
