// The experts of a mixture-of-experts layer for a few tokens: E4M3 weights with a scale a row, bf16 activations.
//
// What bounds it is the stream of the reached experts' weights, a byte a value, read once.  The codes are widened on the way to bf16
// (v_cvt_scalef32_pk_bf16_fp8, two a lane and instruction, exact) and multiplied by v_mfma_f32_16x16x32_bf16: activations keep
// their 16 bits, and the products lose nothing that fp32 sums hold.  An expert's tokens are the columns of the product: MB blocks
// of 16.
//
// Lane (r, g) of a wave takes row r of a 16-row tile and, of a step of 128 columns, columns 16 g .. + 15 and 64 + 16 g .. + 15: 16 contiguous bytes
// each, two instructions each; the activations' lanes take the same columns, 32 contiguous bytes each.
#pragma once

#include "sg_moe_route_kernel.h"

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

    // wb: the tiles' first rows, xb: the activations, both the wave's; wo, xo: the lane's rows, bytes from there.  pieces: 16-column pieces
    // a row; a piece beyond the row's end is the last one again.  live: all ones, or 0 where there is nothing to load: the loads of all
    // lanes go to the first bytes then, since a load that may not be issued would make every wait one for all loads.
    __device__ __forceinline__ void load(const uint8_t* const (&wb)[RT], uint32_t wo, const uint8_t* xb, const uint32_t (&xo)[MB], int blocks,
                                         int step, int pieces, uint32_t live = ~0u) {
        const int g = lane_id() >> 4;
        uint32_t p[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int piece = 8 * step + 4 * h + g;
            p[h] = (uint32_t)(piece < pieces ? piece : pieces - 1) * 16;
        }
#pragma unroll
        for (int i = 0; i < RT; i++)
#pragma unroll
            for (int h = 0; h < 2; h++) w[i][h] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(wb[i] + ((wo + p[h]) & live)));
#pragma unroll
        for (int j = 0; j < MB; j++)
            if (j < blocks || MB == 1)
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int u = 0; u < 2; u++) x[j][h][u] = *reinterpret_cast<const u32x4*>(xb + ((xo[j] + 2 * p[h] + 16 * u) & live));
    }
    // Beyond the row's end the activations are zeros.  (The weights there are the row's last ones again: a NaN among them is in the row's
    // sum already, and there is no infinity in E4M3.)
    __device__ __forceinline__ void multiply(f32x4 (&acc)[RT][MB], int blocks, int step, int pieces) const {
        const int g = lane_id() >> 4;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const bool inside = 8 * step + 4 * h + g < pieces;
#pragma unroll
            for (int u = 0; u < 2; u++) {
                u32x4 v[RT];
#pragma unroll
                for (int i = 0; i < RT; i++) v[i] = moe_widen(w[i][h][2 * u], w[i][h][2 * u + 1]);
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

// v / (1 + exp(-v)), by the exponential that does not overflow
__device__ __forceinline__ float moe_silu(float v) {
    const float t = expf(-fabsf(v));
    return v * ((v < 0.0f ? t : 1.0f) / (1.0f + t));
}

// h = bf16( silu(S1 * (gate x)) * (S1 * (up x)) ).  An item is 16 gate rows and their 16 up rows of a part of the plan; `share` of a
// workgroup's four waves share its columns, step by step in turn, and meet in LDS.  A wave has two steps of 4 KB of weights in flight,
// from one item into the next.
// LDS: plan, then the room that it is made in, then in its place [4 waves][2 * MB][64 lanes] f32x4.
template <int MB, bool CHOOSE>
__global__ void __launch_bounds__(256, MB == 1 ? 4 : 3) moe_gate_up_kernel(const MoeArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    int32_t* const plan = reinterpret_cast<int32_t*>(lds);
    const MoePlanLayout l = moe_plan_layout(a.m, a.experts, a.top_k);
    f32x4* const part = reinterpret_cast<f32x4*>(lds + (size_t)l.dwords * 4);
    const int lane = lane_id(), r = lane & 15, g = lane >> 4, wave = wave_id();
    {
        const MoePlanRoom room = moe_room(lds + (size_t)l.dwords * 4, a.m * a.top_k);
        moe_make_plan<MB, CHOOSE>(a, l, room, plan);
        if (blockIdx.x == 0) {       // for the second launch, and the caller
            for (int i = (int)threadIdx.x; i < l.dwords; i += 256) a.plan[i] = plan[i];
            if (CHOOSE)
                for (int i = (int)threadIdx.x; i < a.m * a.top_k; i += 256) a.ids[i] = room.ids[i], a.weights[i] = room.weights[i];
        }
        __syncthreads();
    }
    const int tiles = a.inner / 16, items = __builtin_amdgcn_readfirstlane(plan[0]) * tiles;
    const int pieces = a.hidden / 16, steps = (a.hidden + 127) / 128, share = a.share;
    const int sharer = wave % share, stride = (int)gridDim.x * (4 / share);
    const int mine = ((steps - 1) / share + 2) / 2 * 2;        // steps of a wave and item, beyond the last: the last one again, times zeros

    struct Item {
        const uint8_t* wb[2];
        uint32_t xo[MB], live;
        int row, first, tile, count, blocks;      // row of W1's rows of all experts: below 2^31
    };
    auto find = [&](int item) __attribute__((always_inline)) {
        Item t;
        t.live = item < items ? ~0u : 0u;
        const int at = item < items ? item : 0, which = at / tiles;
        t.tile = at - which * tiles;
        const int packed = __builtin_amdgcn_readfirstlane(plan[l.parts_at + which]);
        const int e = packed & 0xffff;
        t.count = packed >> 16;
        t.blocks = (t.count + 15) / 16;
        t.first = l.rows_at + __builtin_amdgcn_readfirstlane(plan[l.first_at + which]);
        t.row = e * 2 * a.inner + t.tile * 16;
        t.wb[0] = a.W1 + (size_t)t.row * a.hidden;
        t.wb[1] = t.wb[0] + (size_t)a.inner * a.hidden;
#pragma unroll
        for (int j = 0; j < MB; j++)
            t.xo[j] = (uint32_t)plan[t.first + (16 * j + r < t.count ? 16 * j + r : t.count - 1)] / (uint32_t)a.top_k * (uint32_t)(a.hidden * 2);
        return t;
    };
    MoeStep<2, MB> s0, s1;
    f32x4 acc[2][MB];
    const uint32_t wo = (uint32_t)(r * a.hidden);
    auto load = [&](MoeStep<2, MB>& s, const Item& t, int i) __attribute__((always_inline)) {
        const int step = sharer + i * share;
        s.load(t.wb, wo, a.X, t.xo, t.blocks, step < steps ? step : steps - 1, pieces, t.live);
    };
    auto multiply = [&](const MoeStep<2, MB>& s, const Item& t, int i) __attribute__((always_inline)) {
        s.multiply(acc, t.blocks, sharer + i * share, pieces);
    };

    if (items == 0) return;
    int item = (int)blockIdx.x * (4 / share) + wave / share;
    Item now = find(item);
    load(s0, now, 0);
    load(s1, now, 1);
    for (int round = (int)blockIdx.x * (4 / share); round < items; round += stride, item += stride) {
        const Item next = find(item + stride);
        f32x4 scale[2] = {{1.f, 1.f, 1.f, 1.f}, {1.f, 1.f, 1.f, 1.f}};      // loaded here, in front of the next item's steps
        if (a.S1) {
            using f32x4_at4 = f32x4 __attribute__((aligned(4)));
            scale[0] = *reinterpret_cast<const f32x4_at4*>(a.S1 + now.row + 4 * g);
            scale[1] = *reinterpret_cast<const f32x4_at4*>(a.S1 + now.row + a.inner + 4 * g);
        }
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int j = 0; j < MB; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        int i = 0;
        for (; i + 2 < mine; i += 2) {
            multiply(s0, now, i);
            load(s0, now, i + 2);
            multiply(s1, now, i + 1);
            load(s1, now, i + 3);
        }
        multiply(s0, now, i);
        load(s0, next, 0);
        multiply(s1, now, i + 1);
        load(s1, next, 1);
        moe_settle(acc);
        auto finish = [&](f32x4 gate, f32x4 up, int j) __attribute__((always_inline)) {
            if (!now.live || 16 * j + r >= now.count) return;
            gate *= scale[0];
            up *= scale[1];
            const u32x2 o = {pack_bf16x2(moe_silu(gate[0]) * up[0], moe_silu(gate[1]) * up[1]),
                             pack_bf16x2(moe_silu(gate[2]) * up[2], moe_silu(gate[3]) * up[3])};
            *reinterpret_cast<u32x2*>(a.H + ((size_t)plan[now.first + 16 * j + r] * a.inner + now.tile * 16 + 4 * g) * 2) = o;
        };
        if (share == 1) {
#pragma unroll
            for (int j = 0; j < MB; j++) finish(acc[0][j], acc[1][j], j);
        } else {
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int j = 0; j < MB; j++) part[(wave * 2 * MB + i * MB + j) * 64 + lane] = acc[i][j];
            __syncthreads();
            const f32x4* const p = part + (wave - sharer) * 2 * MB * 64 + lane;
            for (int j = sharer; j < now.blocks; j += share) {
                f32x4 gate = p[j * 64], up = p[(MB + j) * 64];
#pragma unroll 1
                for (int w = 1; w < share; w++) {
                    gate += p[(w * 2 * MB + j) * 64];
                    up += p[(w * 2 * MB + MB + j) * 64];
                }
                finish(gate, up, j);
            }
            __syncthreads();
        }
        now = next;
    }
}

// D = bf16( sum over experts of weight * S2 * (W2 h) ): a workgroup has 16 rows of hidden for all tokens, its waves share the steps of all
// parts, in one range each, DEPTH steps of 2 KB of weights in flight.  A wave adds a part's product, scaled, to sums of its own - [tokens][16 rows]
// in LDS, where no other wave and no second lane writes -, the waves' sums are added in wave order: no atomics, one order.
// LDS: plan, S2 of the tile [parts][16], then [waves][m][16] floats.
template <int MB, int DEPTH, int WAVES>
__global__ void __launch_bounds__(64 * WAVES, MB == 1 ? 4 : WAVES / 4) moe_down_kernel(const MoeArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    int32_t* const plan = reinterpret_cast<int32_t*>(lds);
    const MoePlanLayout l = moe_plan_layout(a.m, a.experts, a.top_k);
    float* const scales = reinterpret_cast<float*>(lds + (size_t)l.dwords * 4);
    float* const total = scales + l.most * 16;
    const int tid = (int)threadIdx.x, lane = lane_id(), r = lane & 15, g = lane >> 4, wave = wave_id();
    const int tile = xcd_order((int)blockIdx.x, (int)gridDim.x);
    for (int i = tid * 4; i < l.dwords; i += 64 * WAVES * 4) *reinterpret_cast<i32x4*>(plan + i) = *reinterpret_cast<const i32x4*>(a.plan + i);
    float* const own = total + wave * a.m * 16;
    for (int i = lane; i < a.m * 16; i += 64) own[i] = 0.0f;
    __syncthreads();
    const int parts = __builtin_amdgcn_readfirstlane(plan[0]), pieces = a.inner / 16, steps = (a.inner + 127) / 128;
    auto scale_of = [&](int i) {      // row i % 16 of part i / 16
        return a.S2 ? a.S2[(size_t)(plan[l.parts_at + (i >> 4)] & 0xffff) * a.hidden + tile * 16 + (i & 15)] : 1.0f;
    };
    const float first_scale = tid < parts * 16 ? scale_of(tid) : 1.0f;

    const long long all = (long long)parts * steps;
    const long long begin = all * wave / WAVES;
    const int steps_here = (int)(all * (wave + 1) / WAVES - begin);
    // ---- where to load next ----
    const uint8_t* wb[1] = {};
    uint32_t xo[MB] = {};
    const uint32_t wo = (uint32_t)(r * a.inner);
    int which = (int)(begin / steps), step = (int)(begin - (long long)which * steps), blocks = 0;
    auto find = [&]() __attribute__((always_inline)) {
        const int packed = __builtin_amdgcn_readfirstlane(plan[l.parts_at + which]), e = packed & 0xffff, count = packed >> 16;
        const int32_t* const rows = plan + l.rows_at + __builtin_amdgcn_readfirstlane(plan[l.first_at + which]);
        blocks = (count + 15) / 16;
        wb[0] = a.W2 + ((size_t)e * a.hidden + tile * 16) * a.inner;
#pragma unroll
        for (int j = 0; j < MB; j++) xo[j] = (uint32_t)rows[16 * j + r < count ? 16 * j + r : count - 1] * (uint32_t)(a.inner * 2);
    };
    MoeStep<1, MB> s[DEPTH];
    auto load = [&](MoeStep<1, MB>& to) __attribute__((always_inline)) {
        to.load(wb, wo, a.H, xo, blocks, step, pieces);
        if (++step == steps) {
            step = 0;
            if (++which < parts) find();
        }
    };
    // ---- where to multiply ----
    int part = which, at = step, part_count = 0, part_first = 0;
    f32x4 acc[1][MB];
    auto open = [&]() __attribute__((always_inline)) {
        part_count = __builtin_amdgcn_readfirstlane(plan[l.parts_at + part]) >> 16;
        part_first = __builtin_amdgcn_readfirstlane(plan[l.first_at + part]);
#pragma unroll
        for (int j = 0; j < MB; j++) acc[0][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    };
    auto close = [&]() __attribute__((always_inline)) {
        moe_settle(acc);
        const f32x4 scale = *reinterpret_cast<const f32x4*>(scales + part * 16 + 4 * g);
#pragma unroll
        for (int j = 0; j < MB; j++)
            if (16 * j + r < part_count) {
                const int entry = part_first + 16 * j + r, token = plan[l.rows_at + entry] / a.top_k;
                const float weight = __uint_as_float((uint32_t)plan[l.weights_at + entry]);
                f32x4* const sum = reinterpret_cast<f32x4*>(own + token * 16 + 4 * g);
                *sum += acc[0][j] * scale * weight;
            }
    };
    auto multiply = [&](MoeStep<1, MB>& from) __attribute__((always_inline)) {
        from.multiply(acc, (part_count + 15) / 16, at, pieces);
        if (++at == steps) {
            close();
            at = 0;
            if (++part < parts) open();
        }
    };
    if (steps_here > 0) {
        find();
        open();
#pragma unroll
        for (int d = 0; d < DEPTH; d++)
            if (d < steps_here) load(s[d]);
    }
    if (tid < parts * 16) scales[tid] = first_scale;
    for (int i = tid + 64 * WAVES; i < parts * 16; i += 64 * WAVES) scales[i] = scale_of(i);
    __syncthreads();
    if (steps_here > 0) {
        int left = steps_here;
        for (; left >= 2 * DEPTH; left -= DEPTH)
#pragma unroll
            for (int d = 0; d < DEPTH; d++) {
                multiply(s[d]);
                load(s[d]);
            }
#pragma unroll
        for (int d = 0; d < DEPTH; d++) {
            if (d < left) multiply(s[d]);
            if (d + DEPTH < left) load(s[d]);
        }
#pragma unroll
        for (int d = 0; d < DEPTH; d++)
            if (d + DEPTH < left) multiply(s[d]);
        if (at != 0) close();
    }
    __syncthreads();
    for (int i = tid; i < a.m * 4; i += 64 * WAVES) {
        const int token = i >> 2, c = i & 3;
        f32x4 v = *reinterpret_cast<const f32x4*>(total + token * 16 + 4 * c);
        for (int w = 1; w < WAVES; w++) v += *reinterpret_cast<const f32x4*>(total + (w * a.m + token) * 16 + 4 * c);
        const u32x2 o = {pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
        *reinterpret_cast<u32x2*>(a.D + (size_t)token * a.hidden + tile * 16 + 4 * c) = o;
    }
}

}  // namespace sg
