// The experts of a mixture-of-experts layer for a few tokens: E4M3 weights with a scale a row, bf16 activations.
//
// What bounds it is the stream of the reached experts' weights, a byte a value, read once.  The codes are widened on the way to bf16
// (v_cvt_scalef32_pk_bf16_fp8, two a lane and instruction, exact) and multiplied by v_mfma_f32_16x16x32_bf16: activations keep
// their 16 bits, and the products lose nothing that fp32 sums hold.  An expert's tokens are the columns of the product: MB blocks
// of 16.
//
// Operands reach LDS by direct loads, 1 KB an instruction: 8 rows x 128 bytes of weights, 4 rows x 256 bytes of activations, so that every
// line is asked for once and whole.  (Lane (r, g) loading 16 bytes of row r straight into its operand register asks for every line in
// pieces: 1.29 GB of gate and up 277 us, 4.7 TB/s, however much is in flight.)  Every wave has a ring of its own, DEPTH stages of
// 128 columns, filled and emptied by itself in order, with no barrier.  The hardware puts lane l's 16 bytes at slot + 16 l; which piece of
// its row a lane fetches is free, and the pieces of row i stand permuted by i so that the 16 lanes (r, g) of a fragment's read hit
// 16 bank groups.
#pragma once

#include "sg_lds_kernel.h"
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

// a pointer that is the same in all lanes, in scalar registers
__device__ __forceinline__ const uint8_t* moe_uniform(const uint8_t* p) {
    const uint64_t v = reinterpret_cast<uintptr_t>(p);
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
    return reinterpret_cast<const uint8_t*>((uint64_t)hi << 32 | lo);
}

// Stages of 128 columns of RT 16-row tiles of weights and of 4 * XU rows of activations.
// Columns: lane (r, g) takes the 16-byte pieces g and 4 + g of its weight row, codes 64 h + 16 g + 8 t .. + 7 for instruction (h, t), and
// of its activations' row the same columns, piece 8 h + 2 g + t.
//
// LINES: rows that do not start on a 128-byte line (their pitch, a multiple of 16 bytes, is no multiple of 128).  128 bytes from anywhere lie on
// two lines, and the next stage would ask for the second one again; so a stage's weights are the lines of each row, stage s its line s, and
// a row that starts `shift` pieces into its first line has the columns of step s in stages s and s + 1: the shift is applied where
// fragments are read, and a run of n steps takes n + 1 stages.  16 rows are a multiple of 256 bytes: a lane's shift is the same everywhere.
template <int RT, int XU, bool LINES>
struct MoeStages {
    static constexpr int kRows = 4 * XU, kBlocks = XU < 4 ? 1 : XU / 4;      // activation rows, blocks of 16 columns of the product
    static constexpr int kLoads = 2 * RT + XU, kBytes = kLoads * 1024;
    int pieces;                       // 16-column pieces a row
    uint32_t wo[2];                   // the lane's rows of a tile's loads, bytes from the first row
    int wp[2], xp[XU];                // ... and its pieces of stage 0
    int wr[2], xr[4];                 // where its fragments lie in a slot: pieces g and 4 + g; pieces (h, t) at 2 h + t
    bool behind[2];                   // LINES: the piece is in the next stage

    // weights: any tile's first row
    __device__ __forceinline__ void init(const uint8_t* weights, int columns) {
        const int l = lane_id(), r = l & 15, g = l >> 4;
        auto shift = [&](int row) { return LINES ? (int)((uint32_t)(reinterpret_cast<uintptr_t>(weights) + (uint32_t)(row * columns)) & 127u) >> 4 : 0; };
        pieces = columns / 16;
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int row = 8 * u + (l >> 3);
            wo[u] = (uint32_t)(row * columns);
            wp[u] = ((l & 7) ^ (row >> 1)) - shift(row);
        }
#pragma unroll
        for (int u = 0; u < XU; u++) xp[u] = (l & 15) ^ ((4 * u + (l >> 4)) & 15);
        const int at = r % (kRows < 16 ? kRows : 16);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int place = 4 * h + g + shift(r);
            behind[h] = place >= 8;
            wr[h] = r * 128 + ((place & 7) ^ (r >> 1)) * 16;
#pragma unroll
            for (int t = 0; t < 2; t++) xr[2 * h + t] = at * 256 + ((8 * h + 2 * g + t) ^ at) * 16;
        }
    }
    // wb: the tiles' first rows; xb, xo: the activations and the lane's rows there, bytes.  A piece beyond a row's ends is its first or last one.
    __device__ __forceinline__ void issue(unsigned slot, const uint8_t* const (&wb)[RT], const uint8_t* xb, const uint32_t (&xo)[XU], int step) const {
        uint32_t p[2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            int piece = 8 * step + wp[u];
            if (LINES) piece = piece > 0 ? piece : 0;
            p[u] = wo[u] + (uint32_t)(piece < pieces ? piece : pieces - 1) * 16;
        }
#pragma unroll
        for (int i = 0; i < RT; i++)
#pragma unroll
            for (int u = 0; u < 2; u++) dma_1kb_stream_at(moe_uniform(wb[i]), p[u], slot + (2 * i + u) * 1024);
#pragma unroll
        for (int u = 0; u < XU; u++) {
            const int piece = 16 * step + xp[u];
            dma_1kb_at(xb, xo[u] + (uint32_t)(piece < 2 * pieces ? piece : 2 * pieces - 1) * 16, slot + (2 * RT + u) * 1024);
        }
    }
    // next: the slot of the stage behind (LINES).  Beyond the row's end the activations count as zeros.  (The weights there are the row's
    // first or last ones again: a NaN among them is in the row's sum already, and there is no infinity in E4M3.)
    __device__ __forceinline__ void multiply(const uint8_t* slot, const uint8_t* next, f32x4 (&acc)[RT][kBlocks], int blocks, int step) const {
        const int g = lane_id() >> 4;
        u32x4 w[RT][2], x[kBlocks][4];
#pragma unroll
        for (int i = 0; i < RT; i++)
#pragma unroll
            for (int h = 0; h < 2; h++) w[i][h] = *reinterpret_cast<const u32x4*>((LINES && behind[h] ? next : slot) + 2048 * i + wr[h]);
#pragma unroll
        for (int j = 0; j < kBlocks; j++)
#pragma unroll
            for (int t = 0; t < 4; t++) x[j][t] = *reinterpret_cast<const u32x4*>(slot + 2048 * RT + 4096 * j + xr[t]);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const bool inside = 8 * step + 4 * h + g < pieces;
#pragma unroll
            for (int t = 0; t < 2; t++) {
                u32x4 v[RT];
#pragma unroll
                for (int i = 0; i < RT; i++) v[i] = moe_widen(w[i][h][2 * t], w[i][h][2 * t + 1]);
#pragma unroll
                for (int j = 0; j < kBlocks; j++)
                    if (j < blocks || kBlocks == 1) {
                        const u32x4 y = inside ? x[j][2 * h + t] : u32x4{0, 0, 0, 0};
#pragma unroll
                        for (int i = 0; i < RT; i++) acc[i][j] = moe_mfma(v[i], y, acc[i][j]);
                    }
            }
        }
    }
};

// Of `flying` stages, DEPTH at most, the oldest - LINES: and the one behind it - has landed when at most the younger ones' loads are
// outstanding.  `here` steps are left of its item, this one counted: with stages of the next item in flight, whose `scales` were asked for in
// front of them, there is a load more: without it the last step of an item would wait for a load issued just before.
template <int DEPTH, int LOADS, bool LINES>
__device__ __forceinline__ void moe_wait(int flying, int here, bool scales) {
    static_assert(DEPTH >= (LINES ? 3 : 2));
    const bool more = scales && flying > here + LINES;
    if (flying != DEPTH) wait_vmcnt_upto((flying - 1 - LINES) * LOADS + more);
    else if (more) wait_vmcnt<(DEPTH - 1 - LINES) * LOADS + 1>();
    else wait_vmcnt<(DEPTH - 1 - LINES) * LOADS>();
}
// All fragments are read: the slot may be filled again.
__device__ __forceinline__ void moe_slot_read() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

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

// Row scales reach LDS as a product's operands do, by a load in front of its first stage: a vector load to registers would be waited for behind
// every stage in flight, scalar loads 0.8 us at the head of an item.
// A wave's ring has DEPTH stages in flight, each of an item of its own at the least, and one found that has none: DEPTH + 2 slots.
// first, second: 16 floats each, by lanes 0 to 15 and 16 to 31 (second: or NULL)
__device__ __forceinline__ void moe_issue_scales(const float* first, const float* second, unsigned slot) {
    const int lane = lane_id();
    const float* const from = (lane < 16 ? first : second) + (lane & 15);
    slot = __builtin_amdgcn_readfirstlane(slot);
    if (lane < (second ? 32 : 16)) asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(from), "s"(slot) : "memory", "m0");
}

// h = bf16( silu(S1 * (gate x)) * (S1 * (up x)) ): rounded to bf16, since the second product's instruction takes nothing wider at its rate.  It
// shows as one more rounding of an output's size, 2.3e-3 in the norm against 1.65e-3.  Two bf16 parts would undo that but double the activations of the down
// projections, which cost as much of the way into a CU as the weights: by the next wider builds 112.9 -> 126.1 us for 32 tokens on 128 experts and
// 29.7 -> 44.2 for 61 on 40 off their lines (8 tokens or one: the same within 1 %, but then a token's result would hang on how many come with it).
// An item is 16 gate rows and their 16 up rows of a part of the plan; `share` of a
// workgroup's four waves share its columns, a range each, and meet in LDS.  A wave's ring runs from one item into the next.
// LDS: plan, the waves' scales, [4 waves][2 * blocks][64 lanes] f32x4 where waves share, then the rings, and before them in their place
// the room for the plan.
template <int XU, int DEPTH, bool LINES, bool CHOOSE>
__global__ void __launch_bounds__(256) moe_gate_up_kernel(const MoeArgs a) {
    using Stages = MoeStages<2, XU, LINES>;
    constexpr int BLOCKS = Stages::kBlocks;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    int32_t* const plan = reinterpret_cast<int32_t*>(lds);
    const MoePlanLayout l = moe_plan_layout(a.m, a.experts, a.top_k, Stages::kRows);
    const int share_log = a.share_log, share = 1 << share_log;
    constexpr int SCALES = DEPTH + 2;
    const int lane = lane_id(), r = lane & 15, g = lane >> 4, wave = wave_id();
    float* const scales = reinterpret_cast<float*>(lds + (size_t)l.weights_at * 4) + wave * SCALES * 32;
    f32x4* const part = reinterpret_cast<f32x4*>(lds + (size_t)l.weights_at * 4 + 4 * SCALES * 128);
    uint8_t* const rings = lds + (size_t)l.weights_at * 4 + 4 * SCALES * 128 + (share > 1 ? 4 * 2 * BLOCKS * 1024 : 0);
    const int tiles = a.inner / 16, steps = (a.hidden + 127) / 128, sharer = wave & (share - 1), stride = (int)gridDim.x * 4 >> share_log;
    const int first = ((int)blockIdx.x * 4 + wave) >> share_log;
    const int from = steps * sharer >> share_log, of_item = (steps * (sharer + 1) >> share_log) - from;       // (there are more steps than sharers)
    const int first_part = (int)fast_div((unsigned)first, (unsigned)tiles, a.inv_tiles);
    Stages stages;
    stages.init(a.W1, a.hidden);
    if (CHOOSE && a.m == 1) {
        if (wave == 0) moe_plan_token(a, l, blockIdx.x == 0, plan);
        __syncthreads();
    } else {
        const MoePlanRoom room = moe_room(rings, a.m * a.top_k);
        moe_make_plan<Stages::kRows, CHOOSE>(a, l, room, plan);
        if (CHOOSE && blockIdx.x == 0)
            for (int i = (int)threadIdx.x; i < a.m * a.top_k; i += 256) a.ids[i] = room.ids[i], a.weights[i] = room.weights[i];
        __syncthreads();
    }
    if (blockIdx.x == 0)             // for the second launch
        for (int i = (int)threadIdx.x; i < l.weights_at; i += 256) a.plan[i] = plan[i];
    const int items = __builtin_amdgcn_readfirstlane(plan[0]) * tiles;
    uint8_t* const ring = rings + wave * (DEPTH * Stages::kBytes);
    const unsigned ring_at = lds_addr(ring);

    // A tile's steps begin a step behind the one before where rows are multiples of 512 bytes apart: waves that walk them in step meet in a
    // few memory channels then (hidden 4096: 229 -> 207 us).  Elsewhere waves in step share lines of the activations (2064: 60, with it 65 us).
    const bool rotate = !LINES && a.hidden % 512 == 0;
    auto begin_of = [&](int tile) { return rotate ? from + (int)((uint64_t)((uint32_t)tile * a.turn) * (uint32_t)of_item >> 32) : from; };
    auto after = [&](int step) { return LINES || step + 1 < from + of_item ? step + 1 : from; };
    // ---- what to load next ----
    const uint8_t* wb[2] = {};
    uint32_t xo[XU] = {};
    struct Item {
        int part, tile;
    };
    auto advance = [&](Item& i) __attribute__((always_inline)) {
        i.part += a.stride_parts;
        i.tile += a.stride_tiles;
        if (i.tile >= tiles) i.tile -= tiles, i.part++;
    };
    Item next = {first_part, first - first_part * tiles};
    int next_item = first, next_step = 0, next_left = 0, next_slot = 0, next_scales = 0, flying = 0;
    auto find = [&]() __attribute__((always_inline)) {
        next_step = begin_of(next.tile);
        next_left = of_item + LINES;
        const int packed = __builtin_amdgcn_readfirstlane(plan[l.parts_at + next.part]), e = packed & 0xffff, count = packed >> 16;
        const int32_t* const rows = plan + l.rows_at + __builtin_amdgcn_readfirstlane(plan[l.first_at + next.part]);
        wb[0] = a.W1 + ((size_t)e * 2 * a.inner + next.tile * 16) * a.hidden;
        wb[1] = wb[0] + (size_t)a.inner * a.hidden;
#pragma unroll
        for (int u = 0; u < XU; u++) {
            const int row = 4 * u + g;
            xo[u] = (uint32_t)(rows[row < count ? row : count - 1] >> 16) * (uint32_t)(a.hidden * 2);
        }
        if (a.S1) {
            const float* const s = a.S1 + (e * 2 * a.inner + next.tile * 16);      // below 2^31
            moe_issue_scales(s, s + a.inner, lds_addr(scales + next_scales * 32));
            next_scales = next_scales + 1 == SCALES ? 0 : next_scales + 1;
        }
    };
    auto issue = [&]() __attribute__((always_inline)) {
        stages.issue(ring_at + next_slot * Stages::kBytes, wb, a.X, xo, next_step);
        next_slot = next_slot + 1 == DEPTH ? 0 : next_slot + 1;
        flying++;
        next_step = after(next_step);
        if (--next_left == 0) {
            advance(next);
            next_item += stride;
            if (next_item < items) find();
        }
    };
    if (first < items) {
        find();
        for (int d = 0; d < DEPTH && next_item < items; d++) issue();
    }
    int slot = 0, item = first, scales_at = 0;
    Item now = {first_part, first - first_part * tiles};
    for (int round = (int)blockIdx.x * 4 >> share_log; round < items; round += stride, item += stride, advance(now)) {
        f32x4 acc[2][BLOCKS];
        int count = 0, blocks = 0, entry = 0;
        if (item < items) {
            const int packed = __builtin_amdgcn_readfirstlane(plan[l.parts_at + now.part]);
            count = packed >> 16;
            blocks = (count + 15) / 16;
            entry = l.rows_at + __builtin_amdgcn_readfirstlane(plan[l.first_at + now.part]);
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int j = 0; j < BLOCKS; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
            int step = begin_of(now.tile);
            for (int left = of_item; left > 0; left--, step = after(step)) {
                moe_wait<DEPTH, Stages::kLoads, LINES>(flying, left, a.S1 != nullptr);
                const int next = slot + 1 == DEPTH ? 0 : slot + 1;
                stages.multiply(ring + slot * Stages::kBytes, ring + next * Stages::kBytes, acc, blocks, step);
                slot = next;
                moe_slot_read();
                flying--;
                if (next_item < items) issue();
                __builtin_amdgcn_sched_barrier(0);
            }
            if (LINES) {                 // the stage behind the last step is read
                slot = slot + 1 == DEPTH ? 0 : slot + 1;
                flying--;
                if (next_item < items) issue();
                __builtin_amdgcn_sched_barrier(0);
            }
            moe_settle(acc);
        }
        auto finish = [&](f32x4 gate, f32x4 up, int j) __attribute__((always_inline)) {
            if (a.S1) {
                gate *= *reinterpret_cast<const f32x4*>(scales + scales_at * 32 + 4 * g);
                up *= *reinterpret_cast<const f32x4*>(scales + scales_at * 32 + 16 + 4 * g);
            }
            const u32x2 o = {pack_bf16x2(moe_silu(gate[0]) * up[0], moe_silu(gate[1]) * up[1]),
                             pack_bf16x2(moe_silu(gate[2]) * up[2], moe_silu(gate[3]) * up[3])};
            if (16 * j + r < count) *reinterpret_cast<u32x2*>(a.H + ((size_t)(plan[entry + 16 * j + r] & 0xffff) * a.inner + now.tile * 16 + 4 * g) * 2) = o;
        };
        if (share == 1) {
#pragma unroll
            for (int j = 0; j < BLOCKS; j++)
                if (j < blocks) finish(acc[0][j], acc[1][j], j);
        } else {
            if (item < items)
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int j = 0; j < BLOCKS; j++) part[(wave * 2 * BLOCKS + i * BLOCKS + j) * 64 + lane] = acc[i][j];
            __syncthreads();
            const f32x4* const p = part + (wave - sharer) * 2 * BLOCKS * 64 + lane;
            for (int j = sharer; j < blocks; j += share) {
                f32x4 gate = p[j * 64], up = p[(BLOCKS + j) * 64];
#pragma unroll 1
                for (int w = 1; w < share; w++) {
                    gate += p[(w * 2 * BLOCKS + j) * 64];
                    up += p[(w * 2 * BLOCKS + BLOCKS + j) * 64];
                }
                finish(gate, up, j);
            }
            __syncthreads();
        }
        scales_at = scales_at + 1 == SCALES ? 0 : scales_at + 1;
    }
}

// D = bf16( sum over experts of weight * S2 * (W2 h) ): a workgroup has 16 rows of hidden for all tokens, its waves share the stages of all
// parts, in one range each.  A wave adds a part's product, scaled, to sums of its own - [tokens][16 rows] in LDS, where no other wave and
// no second lane writes -, the waves' sums are added in wave order: no atomics, one order.
// With fewer tiles than CUs, `splits` workgroups share a tile's steps, and moe_sum_kernel adds their sums up, in their order.
// LDS: plan, the waves' scales, sums [waves][m][16], the rings.
template <int XU, int DEPTH, bool LINES, int WAVES>
__global__ void __launch_bounds__(64 * WAVES) moe_down_kernel(const MoeArgs a) {
    using Stages = MoeStages<1, XU, LINES>;
    constexpr int BLOCKS = Stages::kBlocks;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    int32_t* const plan = reinterpret_cast<int32_t*>(lds);
    const MoePlanLayout l = moe_plan_layout(a.m, a.experts, a.top_k, Stages::kRows);
    constexpr int SCALES = DEPTH + 2;
    float* const sums = reinterpret_cast<float*>(lds + (size_t)l.dwords * 4) + WAVES * SCALES * 16;
    const int tid = (int)threadIdx.x, lane = lane_id(), r = lane & 15, g = lane >> 4, wave = wave_id();
    uint8_t* const ring = reinterpret_cast<uint8_t*>(sums + WAVES * a.m * 16) + wave * (DEPTH * Stages::kBytes);
    const unsigned ring_at = lds_addr(ring);
    float* const scales = reinterpret_cast<float*>(lds + (size_t)l.dwords * 4) + wave * SCALES * 16;
    const int at_grid = xcd_order((int)blockIdx.x, (int)gridDim.x);
    const int tile = a.splits > 1 ? at_grid / a.splits : at_grid, split = a.splits > 1 ? at_grid - tile * a.splits : 0;
    for (int i = tid * 4; i < l.dwords; i += 64 * WAVES * 4) *reinterpret_cast<i32x4*>(plan + i) = *reinterpret_cast<const i32x4*>(a.plan + i);
    float* const own = sums + wave * a.m * 16;
    for (int i = lane; i < a.m * 16; i += 64) own[i] = 0.0f;
    __syncthreads();
    const int parts = __builtin_amdgcn_readfirstlane(plan[0]), steps = (a.inner + 127) / 128;
    const uint32_t all = (uint32_t)(parts * steps);          // up to 768 parts of 8192 steps, and 64 sharers
    const uint32_t sharer = (uint32_t)(split * WAVES + wave), sharers = (uint32_t)(a.splits * WAVES);
    const int begin = (int)fast_div(all * sharer, sharers, a.inv_sharers), mine = (int)fast_div(all * (sharer + 1), sharers, a.inv_sharers) - begin;
    Stages stages;
    stages.init(a.W2, a.inner);
    // ---- what to load next ----
    const uint8_t* wb[1] = {};
    uint32_t xo[XU] = {};
    int next_part = (int)fast_div((unsigned)begin, (unsigned)steps, a.inv_steps), next_step = begin - next_part * steps, next_slot = 0, next_scales = 0, flying = 0;
    int part = next_part, step = next_step;                  // what to multiply next
    int next_left = mine, next_of_part = 0;                  // steps of parts to come, and stages of this one (LINES: one more than steps)
    auto find = [&]() __attribute__((always_inline)) {
        const int packed = __builtin_amdgcn_readfirstlane(plan[l.parts_at + next_part]), e = packed & 0xffff, count = packed >> 16;
        const int32_t* const rows = plan + l.rows_at + __builtin_amdgcn_readfirstlane(plan[l.first_at + next_part]);
        wb[0] = a.W2 + ((size_t)e * a.hidden + tile * 16) * a.inner;
#pragma unroll
        for (int u = 0; u < XU; u++) {
            const int row = 4 * u + g;
            xo[u] = (uint32_t)(rows[row < count ? row : count - 1] & 0xffff) * (uint32_t)(a.inner * 2);
        }
        const int here = steps - next_step < next_left ? steps - next_step : next_left;
        next_left -= here;
        next_of_part = here + LINES;
        if (a.S2) {
            moe_issue_scales(a.S2 + ((size_t)e * a.hidden + tile * 16), nullptr, lds_addr(scales + next_scales * 16));
            next_scales = next_scales + 1 == SCALES ? 0 : next_scales + 1;
        }
    };
    auto issue = [&]() __attribute__((always_inline)) {
        stages.issue(ring_at + next_slot * Stages::kBytes, wb, a.H, xo, next_step);
        next_slot = next_slot + 1 == DEPTH ? 0 : next_slot + 1;
        flying++;
        next_step++;
        if (--next_of_part == 0) {
            next_step = 0;
            next_part++;
            if (next_left > 0) find();
        }
    };
    if (mine > 0) {
        find();
        for (int d = 0; d < DEPTH && next_of_part > 0; d++) issue();
    }
    int scales_at = 0;
    for (int slot = 0, left = mine; left > 0; part++, step = 0) {
        const int count = __builtin_amdgcn_readfirstlane(plan[l.parts_at + part]) >> 16, blocks = (count + 15) / 16;
        const int first = __builtin_amdgcn_readfirstlane(plan[l.first_at + part]);
        f32x4 acc[1][BLOCKS];
#pragma unroll
        for (int j = 0; j < BLOCKS; j++) acc[0][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (; step < steps && left > 0; step++, left--) {
            moe_wait<DEPTH, Stages::kLoads, LINES>(flying, steps - step < left ? steps - step : left, a.S2 != nullptr);
            const int next = slot + 1 == DEPTH ? 0 : slot + 1;
            stages.multiply(ring + slot * Stages::kBytes, ring + next * Stages::kBytes, acc, blocks, step);
            slot = next;
            moe_slot_read();
            flying--;
            if (next_of_part > 0) issue();
            __builtin_amdgcn_sched_barrier(0);
        }
        if (LINES) {                     // the stage behind the last step is read
            slot = slot + 1 == DEPTH ? 0 : slot + 1;
            flying--;
            if (next_of_part > 0) issue();
            __builtin_amdgcn_sched_barrier(0);
        }
        moe_settle(acc);
        f32x4 scale = {1.0f, 1.0f, 1.0f, 1.0f};
        if (a.S2) scale = *reinterpret_cast<const f32x4*>(scales + scales_at * 16 + 4 * g);
        scales_at = scales_at + 1 == SCALES ? 0 : scales_at + 1;
#pragma unroll
        for (int j = 0; j < BLOCKS; j++)
            if (16 * j + r < count) {
                const int entry = first + 16 * j + r, token = plan[l.rows_at + entry] >> 16;
                const float weight = __uint_as_float((uint32_t)plan[l.weights_at + entry]);
                f32x4* const sum = reinterpret_cast<f32x4*>(own + token * 16 + 4 * g);
                *sum += acc[0][j] * scale * weight;
            }
    }
    __syncthreads();
    for (int i = tid; i < a.m * 4; i += 64 * WAVES) {
        const int token = i >> 2, c = i & 3;
        f32x4 v = *reinterpret_cast<const f32x4*>(sums + token * 16 + 4 * c);
        for (int w = 1; w < WAVES; w++) v += *reinterpret_cast<const f32x4*>(sums + (w * a.m + token) * 16 + 4 * c);
        const size_t at = (size_t)token * a.hidden + tile * 16 + 4 * c;
        if (a.splits > 1) {
            *reinterpret_cast<f32x4*>(a.sums + (size_t)split * a.m * a.hidden + at) = v;
        } else {
            const u32x2 o = {pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
            *reinterpret_cast<u32x2*>(a.D + at) = o;
        }
    }
}

// Four columns a thread.
__global__ __launch_bounds__(256) void moe_sum_kernel(const MoeArgs a) {
    const size_t n = (size_t)a.m * a.hidden, at = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (at >= n) return;
    f32x4 v = *reinterpret_cast<const f32x4*>(a.sums + at);
    for (int s = 1; s < a.splits; s++) v += *reinterpret_cast<const f32x4*>(a.sums + s * n + at);
    const u32x2 o = {pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
    *reinterpret_cast<u32x2*>(a.D + at) = o;
}

}  // namespace sg
