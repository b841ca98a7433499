// The router of a mixture-of-experts layer: logits, choice of experts, and the plan that the experts' launches work by.
#pragma once

#include "sg_moe.h"

namespace sg {

// logits[t][e] = sum_k X[t][k] * R[e][k].  A wave an expert and up to TOKENS tokens: it reads the expert's row once.
// Which experts are chosen is decided by these sums, so they are held in 64 bits - products of bf16 are exact in fp32, eight of
// them are added in fp32, those sums in fp64 - and rounded to fp32 once: which expert comes first does not depend on an
// order of summation but where two logits are equal to fp32's last bit.
template <int TOKENS>
__global__ void __launch_bounds__(256) moe_logits_kernel(const MoeArgs a) {
    const int lane = lane_id(), e = (int)blockIdx.x * 4 + wave_id(), t0 = (int)blockIdx.y * TOKENS;
    if (e >= a.experts) return;
    const int pieces = a.hidden / 8;
    const u32x4* const r = reinterpret_cast<const u32x4*>(a.R) + (size_t)e * pieces;
    double sum[TOKENS];
    const u32x4* x[TOKENS];
#pragma unroll
    for (int t = 0; t < TOKENS; t++) {
        sum[t] = 0.0;
        x[t] = reinterpret_cast<const u32x4*>(a.X) + (size_t)(t0 + t < a.m ? t0 + t : a.m - 1) * pieces;
    }
#pragma unroll 4
    for (int p = lane; p < pieces; p += 64) {
        const u32x4 w = r[p];
#pragma unroll
        for (int t = 0; t < TOKENS; t++) {
            const u32x4 v = x[t][p];
            float s = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                s = fmaf(bf16_lo(w[j]), bf16_lo(v[j]), s);
                s = fmaf(bf16_hi(w[j]), bf16_hi(v[j]), s);
            }
            sum[t] += (double)s;
        }
    }
#pragma unroll
    for (int t = 0; t < TOKENS; t++) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) sum[t] += __shfl_xor(sum[t], o);
        if (lane == 0 && t0 + t < a.m) a.logits[(size_t)(t0 + t) * a.experts + e] = (float)sum[t];
    }
}

// Order of floats as unsigned integers: NaNs first of all (0), which is last in a choice of the largest.
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t u = __float_as_uint(v + 0.0f);        // -0 is 0
    if ((u & 0x7fffffffu) > 0x7f800000u) return 0;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One wave: the top_k experts of a token and their weights, by top_k rounds of a maximum over the lanes' own logits.
// PER: experts a lane, lane l has l, l + 64, ...
template <int PER>
__device__ __forceinline__ void moe_choose(const MoeArgs& a, int t) {
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
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const uint32_t other = __shfl_xor(best, o);
            best = other > best ? other : best;
        }
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
                at = __shfl(v[i], l);
                if (lane == l) taken |= 1u << i;
            }
        }
        if (c == 0) first = at;
        if (lane == c) mine = at, id = e;
    }
    float p = expf(mine - first), all = 0.0f;
    if (a.renormalize) {
        all = lane < a.top_k ? p : 0.0f;
    } else {
#pragma unroll
        for (int i = 0; i < PER; i++) all += lane + 64 * i < a.experts ? expf(v[i] - first) : 0.0f;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) all += __shfl_xor(all, o);
    if (lane < a.top_k) {
        a.ids[(size_t)t * a.top_k + lane] = id;
        a.weights[(size_t)t * a.top_k + lane] = p / all;
    }
}

__device__ __forceinline__ void moe_choose_any(const MoeArgs& a, int t) {
    if (a.experts <= 64) moe_choose<1>(a, t);
    else if (a.experts <= 128) moe_choose<2>(a, t);
    else if (a.experts <= 256) moe_choose<4>(a, t);
    else moe_choose<8>(a, t);
}

// Who goes where, from ids and weights, by one workgroup of 512 threads.
__device__ __forceinline__ void moe_make_plan(const MoeArgs& a) {
    __shared__ int32_t ids[kMoeTokens * kMoeTopK];
    __shared__ float weights[kMoeTokens * kMoeTopK];
    __shared__ uint32_t tokens[kMoeExperts][2];          // which tokens name the expert
    __shared__ int32_t place[kMoeExperts];               // its first entry
    __shared__ int32_t sums[8][2];
    const int tid = (int)threadIdx.x, pairs = a.m * a.top_k;
    const MoePlanLayout l = moe_plan_layout(a.m, a.experts, a.top_k);
    for (int i = tid; i < pairs; i += 512) {
        ids[i] = a.ids[i];
        weights[i] = a.weights[i];
    }
    for (int e = tid; e < kMoeExperts; e += 512) tokens[e][0] = tokens[e][1] = 0;
    __syncthreads();
    for (int i = tid; i < pairs; i += 512) {
        const int e = ids[i], t = i / a.top_k;
        if (e >= 0 && e < a.experts) atomicOr(&tokens[e][t >> 5], 1u << (t & 31));
    }
    __syncthreads();
    // a thread an expert: how many experts before it are reached, how many entries they have
    static_assert(kMoeExperts == 512);
    const int count = __popc(tokens[tid][0]) + __popc(tokens[tid][1]);
    const int lane = lane_id(), wave = tid >> 6;
    int reached = count > 0, entries = count;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int r = __shfl_up(reached, o), n = __shfl_up(entries, o);
        if (lane >= o) reached += r, entries += n;
    }
    if (lane == 63) sums[wave][0] = reached, sums[wave][1] = entries;
    __syncthreads();
    for (int w = 0; w < wave; w++) reached += sums[w][0], entries += sums[w][1];
    if (tid == 511) a.plan[0] = reached;
    place[tid] = entries - count;
    if (count) {
        a.plan[l.experts_at + reached - 1] = tid | count << 16;
        a.plan[l.first_at + reached - 1] = entries - count;
    }
    __syncthreads();
    // an entry for each token and expert, written by the choice that names the expert first, with all its choices' weights
    for (int i = tid; i < pairs; i += 512) {
        const int e = ids[i], t = i / a.top_k;
        if (e < 0 || e >= a.experts) continue;
        bool earlier = false;
        float weight = 0.0f;
        for (int c = t * a.top_k; c < (t + 1) * a.top_k; c++) {
            if (ids[c] != e) continue;
            if (c < i) earlier = true;
            weight += weights[c];
        }
        if (earlier) continue;
        const uint32_t lo = tokens[e][0], hi = tokens[e][1];
        const int before = t < 32 ? __popc(lo & ((1u << t) - 1u)) : __popc(lo) + __popc(hi & ((1u << (t - 32)) - 1u));
        const int at = place[e] + before;
        a.plan[l.rows_at + at] = i;
        a.plan[l.weights_at + at] = (int32_t)__float_as_uint(weight);
    }
}

// CHOOSE: ids and weights from the logits first.  PLAN: and the plan.
template <bool CHOOSE, bool PLAN>
__global__ void __launch_bounds__(512) moe_plan_kernel(const MoeArgs a) {
    if (CHOOSE) {
        for (int t = wave_id() + 8 * (int)blockIdx.x; t < a.m; t += 8 * (int)gridDim.x) moe_choose_any(a, t);
        if (PLAN) {
            __threadfence_block();
            __syncthreads();
        }
    }
    if (PLAN) moe_make_plan(a);
}

}  // namespace sg
