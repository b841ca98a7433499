// The router of a mixture-of-experts layer: logits, choice of experts, and the plan that the experts' launches work by.
#pragma once

#include "sg_moe.h"

namespace sg {

// a + b over lanes that differ in bit `o` of their number: half of the values each, N / 2 of them kept
template <int N>
__device__ __forceinline__ void halve(double (&v)[N], int o) {
    const bool upper = lane_id() & o;
#pragma unroll
    for (int i = 0; i < N / 2; i++) {
        const double keep = upper ? v[i + N / 2] : v[i], give = upper ? v[i] : v[i + N / 2];
        v[i] = keep + __shfl_xor(give, o);
    }
}

// logits[t][e] = sum_k X[t][k] * R[e][k].  A workgroup of four waves an expert and up to TOKENS (1, 8) tokens: it reads the expert's row once.
// Which experts are chosen is decided by these sums, so they are held in 64 bits - a product of bf16 is exact there, whatever its size - and
// rounded to fp32 once: an order of summation could only show where a sum lies within 2^-53 of its terms' size of a border between two
// fp32 values.
template <int TOKENS>
__global__ void __launch_bounds__(256) moe_logits_kernel(const MoeArgs a) {
    __shared__ double of_wave[4][TOKENS];
    const int lane = lane_id(), wave = wave_id(), e = (int)blockIdx.x, t0 = (int)blockIdx.y * TOKENS;
    const int pieces = a.hidden / 8;
    const u32x4* const r = reinterpret_cast<const u32x4*>(a.R) + (size_t)e * pieces;
    double sum[TOKENS];
    const u32x4* x[TOKENS];
#pragma unroll
    for (int t = 0; t < TOKENS; t++) {
        sum[t] = 0.0;
        x[t] = reinterpret_cast<const u32x4*>(a.X) + (size_t)(t0 + t < a.m ? t0 + t : a.m - 1) * pieces;
    }
    for (int p = (int)threadIdx.x; p < pieces; p += 512) {      // two pieces in flight
        const int second = p + 256 < pieces ? p + 256 : p;
        u32x4 w[2] = {r[p], r[second]}, v[2][TOKENS];
#pragma unroll
        for (int t = 0; t < TOKENS; t++) v[0][t] = x[t][p];
#pragma unroll
        for (int t = 0; t < TOKENS; t++) v[1][t] = x[t][second];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            if (h && second == p) break;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const double lo = bf16_lo(w[h][j]), hi = bf16_hi(w[h][j]);
#pragma unroll
                for (int t = 0; t < TOKENS; t++) {
                    sum[t] = fma(lo, (double)bf16_lo(v[h][t][j]), sum[t]);
                    sum[t] = fma(hi, (double)bf16_hi(v[h][t][j]), sum[t]);
                }
            }
        }
    }
    // over the lanes: each step halves the values that a lane has of its own
    int mine = 0;
    if constexpr (TOKENS == 8) {
        double four[4], two[2];
        halve<8>(sum, 32);
#pragma unroll
        for (int i = 0; i < 4; i++) four[i] = sum[i];
        halve<4>(four, 16);
#pragma unroll
        for (int i = 0; i < 2; i++) two[i] = four[i];
        halve<2>(two, 8);
        sum[0] = two[0];
        mine = lane >> 3;
    }
#pragma unroll
    for (int o = TOKENS == 8 ? 4 : 32; o > 0; o >>= 1) sum[0] += __shfl_xor(sum[0], o);
    if (lane % (64 / TOKENS) == 0) of_wave[wave][mine] = sum[0];
    __syncthreads();
    if ((int)threadIdx.x < TOKENS && t0 + (int)threadIdx.x < a.m) {
        const int t = (int)threadIdx.x;
        a.logits[(size_t)(t0 + t) * a.experts + e] = (float)(of_wave[0][t] + of_wave[1][t] + of_wave[2][t] + of_wave[3][t]);
    }
}

// Order of floats as unsigned integers: NaNs first of all (0), which is last in a choice of the largest.
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t u = __float_as_uint(v + 0.0f);        // -0 is 0
    if ((u & 0x7fffffffu) > 0x7f800000u) return 0;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// the largest value of a wave's lanes, in all of them
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
    auto step = [&](uint32_t o) { v = o > v ? o : v; };
    step(__builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false));      // lanes 1, 2, 4, 8 before, in rows of 16
    step(__builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false));
    step(__builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false));
    step(__builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false));
    step(__builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false));      // a row's last lane to the next row
    step(__builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false));      // lane 31 to the upper half
    return __builtin_amdgcn_readlane(v, 63);
}

// One wave: the top_k experts of a token and their weights, by top_k rounds of a maximum over the lanes' own logits.
// PER: experts a lane, lane l has l, l + 64, ...  Lane c returns the c-th choice and, asked for it, its weight.
template <int PER>
__device__ __forceinline__ int moe_choose(const MoeArgs& a, int t, bool weighed, float& weight) {
    const int lane = lane_id();
    float v[PER];
    uint32_t key[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int e = lane + 64 * i;
        v[i] = a.logits[(size_t)t * a.experts + (e < a.experts ? e : a.experts - 1)];
        key[i] = e < a.experts ? ordered(v[i]) : 0;
    }
    uint32_t taken = 0;                                  // bit i: v[i] is chosen, or beyond the last expert
#pragma unroll
    for (int i = 0; i < PER; i++) taken |= lane + 64 * i < a.experts ? 0u : 1u << i;
    float mine = 0.0f, first = 0.0f;                     // lane c keeps the c-th choice
    int id = 0;
    for (int c = 0; c < a.top_k; c++) {
        uint32_t best = 0;
#pragma unroll
        for (int i = 0; i < PER; i++) best = taken >> i & 1u ? best : (key[i] > best ? key[i] : best);
        best = wave_max_u32(best);
        // the lowest expert with that key
        int e = -1;
        float at = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const bool here = !(taken >> i & 1u) && key[i] == best;
            const unsigned long long lanes = __ballot(here);
            if (e < 0 && lanes) {
                const int l = __ffsll(lanes) - 1;
                e = l + 64 * i;
                at = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v[i]), l));
                if (lane == l) taken |= 1u << i;
            }
        }
        if (c == 0) first = at;
        if (lane == c) mine = at, id = e;
    }
    if (!weighed) return id;
    const float p = expf(mine - first);
    float all = 0.0f;
    if (a.renormalize) {
        all = lane < a.top_k ? p : 0.0f;
    } else {
#pragma unroll
        for (int i = 0; i < PER; i++) all += lane + 64 * i < a.experts ? expf(v[i] - first) : 0.0f;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) all += __shfl_xor(all, o);
    weight = p / all;
    return id;
}

__device__ __forceinline__ int moe_choose_any(const MoeArgs& a, int t, bool weighed, float& weight) {
    if (a.experts <= 64) return moe_choose<1>(a, t, weighed, weight);
    if (a.experts <= 128) return moe_choose<2>(a, t, weighed, weight);
    if (a.experts <= 256) return moe_choose<4>(a, t, weighed, weight);
    return moe_choose<8>(a, t, weighed, weight);
}
__device__ __forceinline__ void moe_choose_into(const MoeArgs& a, int t, int32_t* ids, float* weights) {
    float weight = 0.0f;
    const int id = moe_choose_any(a, t, true, weight);
    if (lane_id() < a.top_k) {
        ids[lane_id()] = id;
        weights[lane_id()] = weight;
    }
}

// A wave a token.
__global__ void __launch_bounds__(64) moe_choose_kernel(const MoeArgs a) {
    const size_t at = (size_t)blockIdx.x * a.top_k;
    moe_choose_into(a, (int)blockIdx.x, a.ids + at, a.weights + at);
}

// The plan of one token, by one wave: its choices in the order of their experts.  What the products wait for is this: the weights
// are left to the workgroup that hands the plan on.
__device__ __forceinline__ void moe_plan_token(const MoeArgs& a, const MoePlanLayout& l, bool hands_on, int32_t* plan) {
    float weight = 0.0f;
    const int lane = lane_id(), id = moe_choose_any(a, 0, hands_on, weight);
    int at = 0;
    for (int c = 0; c < a.top_k; c++) at += __builtin_amdgcn_readlane(id, c) < id;
    if (lane >= a.top_k) return;
    plan[0] = a.top_k;
    plan[l.parts_at + at] = id | 1 << 16;
    plan[l.first_at + at] = at;
    plan[l.rows_at + at] = lane;
    if (hands_on) {
        a.plan[l.weights_at + at] = (int32_t)__float_as_uint(weight);
        a.ids[lane] = id;
        a.weights[lane] = weight;
    }
}

// LDS that a workgroup makes the plan in.
struct MoePlanRoom {
    int32_t* ids;                    // [pairs]
    float* weights;                  // [pairs]
    uint32_t* tokens;                // [512][2]: which tokens name the expert
    int32_t* place;                  // [512]: its first entry
    int32_t* sums;                   // [4][2]
};
constexpr int moe_plan_room(int pairs) { return pairs * 8 + kMoeExperts * 12 + 32; }
__device__ __forceinline__ MoePlanRoom moe_room(uint8_t* at, int pairs) {
    MoePlanRoom r;
    r.tokens = reinterpret_cast<uint32_t*>(at);
    r.place = reinterpret_cast<int32_t*>(r.tokens + 2 * kMoeExperts);
    r.sums = r.place + kMoeExperts;
    r.ids = r.sums + 8;
    r.weights = reinterpret_cast<float*>(r.ids + pairs);
    return r;
}

// Who goes where, by a workgroup of 256 threads: the choices (made here, or the caller's) into the room, the plan into `plan`, both LDS, but
// for the weights: the workgroup that hands the plan on writes them to its place.
template <int COLS, bool CHOOSE>
__device__ __forceinline__ void moe_make_plan(const MoeArgs& a, const MoePlanLayout& l, const MoePlanRoom& room, int32_t* plan) {
    const int tid = (int)threadIdx.x, pairs = a.m * a.top_k;
    if (CHOOSE) {
        for (int t = wave_id(); t < a.m; t += 4) moe_choose_into(a, t, room.ids + t * a.top_k, room.weights + t * a.top_k);
    } else {
        for (int i = tid; i < pairs; i += 256) {
            room.ids[i] = a.ids[i];
            room.weights[i] = a.weights[i];
        }
    }
    for (int i = tid; i < 2 * kMoeExperts; i += 256) room.tokens[i] = 0;
    __syncthreads();
    for (int i = tid; i < pairs; i += 256) {
        const int e = room.ids[i], t = i / a.top_k;
        if (e >= 0 && e < a.experts) atomicOr(&room.tokens[2 * e + (t >> 5)], 1u << (t & 31));
    }
    __syncthreads();
    // a thread two experts: how many parts and entries there are up to and with them
    static_assert(kMoeExperts == 512);
    int count[2], parts = 0, entries = 0;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        count[i] = __popc(room.tokens[4 * tid + 2 * i]) + __popc(room.tokens[4 * tid + 2 * i + 1]);
        parts += (count[i] + COLS - 1) / COLS;
        entries += count[i];
    }
    const int own_parts = parts, own_entries = entries, lane = lane_id(), wave = wave_id();
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int p = __shfl_up(parts, o), n = __shfl_up(entries, o);
        if (lane >= o) parts += p, entries += n;
    }
    if (lane == 63) room.sums[2 * wave] = parts, room.sums[2 * wave + 1] = entries;
    __syncthreads();
    for (int w = 0; w < wave; w++) parts += room.sums[2 * w], entries += room.sums[2 * w + 1];
    if (tid == 255) plan[0] = parts;
    int part = parts - own_parts, first = entries - own_entries;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        room.place[2 * tid + i] = first;
        for (int left = count[i]; left > 0; left -= COLS) {
            const int here = left < COLS ? left : COLS;
            plan[l.parts_at + part] = (2 * tid + i) | here << 16;
            plan[l.first_at + part] = first;
            part++;
            first += here;
        }
    }
    __syncthreads();
    // an entry for each token and expert, written by the choice that names the expert first, with all its choices' weights
    for (int i = tid; i < pairs; i += 256) {
        const int e = room.ids[i], t = i / a.top_k;
        if (e < 0 || e >= a.experts) continue;
        bool earlier = false;
        float weight = 0.0f;
        for (int c = t * a.top_k; c < (t + 1) * a.top_k; c++) {
            if (room.ids[c] != e) continue;
            if (c < i) earlier = true;
            weight += room.weights[c];
        }
        if (earlier) continue;
        const uint32_t lo = room.tokens[2 * e], hi = room.tokens[2 * e + 1];
        const int before = t < 32 ? __popc(lo & ((1u << t) - 1u)) : __popc(lo) + __popc(hi & ((1u << (t - 32)) - 1u));
        const int at = room.place[e] + before;
        plan[l.rows_at + at] = t << 16 | i;
        if (blockIdx.x == 0) a.plan[l.weights_at + at] = (int32_t)__float_as_uint(weight);
    }
    __syncthreads();
}

}  // namespace sg
