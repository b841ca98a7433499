// A mixture-of-experts layer for a few tokens: launches and C entry points (include/sgemm.h).
#include <math.h>

#include "sg_moe_kernel.h"

namespace sg {

static int launched(const char* what) { return report_hip(what, hipGetLastError()) == hipSuccess ? SG_SUCCESS : SG_LAUNCH_FAILED; }

static int launch_logits(const MoeArgs& a, hipStream_t stream) {
    if (a.m == 1) moe_logits_kernel<1><<<dim3((unsigned)a.experts, 1), 256, 0, stream>>>(a);
    else moe_logits_kernel<8><<<dim3((unsigned)a.experts, (unsigned)(a.m + 7) / 8), 256, 0, stream>>>(a);
    return launched("moe_logits launch");
}

static int launch_choose(const MoeArgs& a, hipStream_t stream) {
    moe_choose_kernel<<<(unsigned)a.m, 64, 0, stream>>>(a);
    return launched("moe_choose launch");
}

constexpr size_t kLdsBytes = 160 * 1024;      // a CU's, given out in pieces of 1280
static int lds_workgroups(size_t lds) { return (int)(128 / ((lds + 1279) / 1280)); }

template <int XU, int DEPTH>
static size_t gate_up_lds(const MoeArgs& a) {
    using Stages = MoeStages<2, XU, false>;
    const size_t ring = (size_t)4 * DEPTH * Stages::kBytes, room = moe_plan_room(a.m * a.top_k);
    return (size_t)moe_plan_layout(a.m, a.experts, a.top_k, Stages::kRows).weights_at * 4 + 4 * (DEPTH + 2) * 128 +
           (a.share_log > 0 ? 4 * 2 * Stages::kBlocks * 1024 : 0) + (room > ring ? room : ring);
}
template <int XU, int DEPTH, bool LINES>
static int launch_gate_up(MoeArgs& a, bool choose, long long groups, int cu_count, hipStream_t stream) {
    using Stages = MoeStages<2, XU, LINES>;
    const size_t lds = gate_up_lds<XU, DEPTH>(a);
    const long long at_once = (long long)lds_workgroups(lds) * cu_count;
    const unsigned grid = (unsigned)(groups < at_once ? groups : at_once);
    const long long stride = (long long)grid * 4 >> a.share_log;
    a.stride_parts = (int)(stride / (a.inner / 16));
    a.stride_tiles = (int)(stride % (a.inner / 16));
    a.turn = (uint32_t)(0x100000000ull * (1u << a.share_log) / (unsigned)((a.hidden + 127) / 128) + 1);
    a.inv_tiles = div_reciprocal((unsigned)a.inner / 16);
    auto* kernel = moe_gate_up_kernel<XU, DEPTH, LINES, false>;
    if constexpr (Stages::kRows <= kMoeFused) {      // (wider parts are for more tokens: part_columns)
        if (choose) kernel = moe_gate_up_kernel<XU, DEPTH, LINES, true>;
    } else if (choose) {
        return SG_INVALID_CONFIG;
    }
    static LdsGranted granted[2];
    if (int rc = request_dynamic_lds(reinterpret_cast<const void*>(kernel), lds, granted[choose])) return rc;
    kernel<<<grid, 256, lds, stream>>>(a);
    return launched("moe_gate_up launch");
}

template <int XU, int DEPTH, int WAVES>
static size_t down_lds(const MoeArgs& a) {
    const MoePlanLayout l = moe_plan_layout(a.m, a.experts, a.top_k, 4 * XU);
    return (size_t)l.dwords * 4 + WAVES * (DEPTH + 2) * 64 + (size_t)WAVES * a.m * 64 + (size_t)WAVES * DEPTH * MoeStages<1, XU, false>::kBytes;
}
template <int XU, int DEPTH, bool LINES, int WAVES>
static int launch_down(MoeArgs& a, hipStream_t stream) {
    a.inv_steps = div_reciprocal((unsigned)(a.inner + 127) / 128);
    a.inv_sharers = div_reciprocal((unsigned)(a.splits * WAVES));
    const size_t lds = down_lds<XU, DEPTH, WAVES>(a);
    static LdsGranted granted;
    if (int rc = request_dynamic_lds(reinterpret_cast<const void*>(moe_down_kernel<XU, DEPTH, LINES, WAVES>), lds, granted)) return rc;
    moe_down_kernel<XU, DEPTH, LINES, WAVES><<<(unsigned)(a.hidden / 16 * a.splits), 64 * WAVES, lds, stream>>>(a);
    return launched("moe_down launch");
}

static bool off_lines(const uint8_t* weights, int columns) { return columns % 128 != 0 || (reinterpret_cast<uintptr_t>(weights) & 127u) != 0; }

// Builds of the down projections: four waves, or eight where the rings fit (not with 32 rows of activations a stage), on N stages in flight
// if the LDS holds them.
template <int XU, int N, bool LINES>
struct DownBuilds {
    static constexpr int kFew = LINES ? 3 : 2;
    static constexpr bool kEight = 8 * 2 * MoeStages<1, XU, false>::kBytes < kLdsBytes;
    // LDS of the build on that many waves; more than there is: none
    static size_t lds(const MoeArgs& a, int waves) {
        if (waves == 4) return down_lds<XU, kFew, 4>(a);
        if (!kEight) return kLdsBytes + 1;
        const size_t all = down_lds<XU, N, 8>(a);
        return all <= kLdsBytes ? all : down_lds<XU, kFew, 8>(a);
    }
    static int launch(MoeArgs& a, int waves, hipStream_t stream) {
        if constexpr (kEight)
            if (waves == 8) return down_lds<XU, N, 8>(a) <= kLdsBytes ? launch_down<XU, N, LINES, 8>(a, stream) : launch_down<XU, kFew, LINES, 8>(a, stream);
        return launch_down<XU, kFew, LINES, 4>(a, stream);
    }
};

// How many workgroups share a tile of the down projections, and how many waves they have: eight, one workgroup a CU, or four, two where they
// fit.  Shared sums pay a launch that adds them up.  (2064 rows, 40 experts x 1376, 61 tokens: 129 tiles as they are 39.6 us, three workgroups each
// 30.8 and 4.6 for the sums.  Sums joined by the last workgroup to arrive instead: 95 us, for the fences that write the L2s back.)
template <class Builds>
static int down_splits(const MoeArgs& a, int cu_count, int* waves) {
    const int tiles = a.hidden / 16, most = moe_most_splits(a.hidden);
    const float bytes = a.experts * (1.0f - powf(1.0f - (float)a.top_k / a.experts, (float)a.m)) * a.hidden * (float)a.inner;
    const long long steps = (long long)((a.inner + 127) / 128) * a.top_k;      // of one token: there are more
    float best = 0.0f;
    int splits = 1;
    *waves = 4;
    for (int w = 8; w >= 4; w -= 4) {
        const size_t lds = Builds::lds(a, w);
        if (lds > kLdsBytes) continue;
        const int at_once = w == 4 && lds_workgroups(lds) > 1 ? 2 : 1;
        for (int s = 1; s <= most && (s == 1 || steps >= 2ll * s * w); s++) {
            const int slots = cu_count * at_once, all = tiles * s;
            // of the memory's rate, 6 TB/s: a CU by itself takes in up to 1.4 times its part of it.  Sums are written and read at 4 TB/s.
            const float used = (float)all / (float)((all + slots - 1) / slots * slots), rate = 1.4f * used < 1.0f ? 1.4f * used : 1.0f;
            const float us = bytes / (6.0e6f * rate) + (s > 1 ? 4.0f + (float)s * a.m * a.hidden * 8 / 4e6f : 0.0f);
            if (best == 0.0f || us < 0.97f * best) best = us, splits = s, *waves = w;
        }
    }
    return splits;
}
template <class Builds>
static int launch_down_of(MoeArgs& a, int cu_count, hipStream_t stream) {
    int waves;
    a.splits = down_splits<Builds>(a, cu_count, &waves);
    return Builds::launch(a, waves, stream);
}

// Parts of up to 4 * XU tokens; G and N stages in flight a wave.
template <int XU, int G, int N>
static int launch_parts(MoeArgs& a, bool choose, int cu_count, hipStream_t stream) {
    const int pairs = a.m * a.top_k, most = a.experts < pairs ? a.experts : pairs, steps = (a.hidden + 127) / 128;
    const long long items = (long long)most * (a.inner / 16);
    // Waves that share an item, and stages in flight: what leaves the least to the last round.
    // (32 rows of activations a stage leave no room for a third one)
    constexpr bool kLines = 4 * 3 * MoeStages<2, XU, true>::kBytes + 4 * 2 * MoeStages<2, XU, true>::kBlocks * 1024 < kLdsBytes;
    const bool lines = kLines && off_lines(a.W1, a.hidden) && (a.share_log = 2, gate_up_lds<XU, 3>(a) <= kLdsBytes);
    float best = 0.0f;
    int share_log = 0;
    bool shorter = false;
    for (a.share_log = 0; a.share_log <= 2 && (a.share_log == 0 || steps >= 2 << a.share_log); a.share_log++)
        for (int s = 0; s < (lines ? 1 : 2); s++) {
            const size_t lds = lines ? gate_up_lds<XU, 3>(a) : s ? gate_up_lds<XU, 2>(a) : gate_up_lds<XU, G>(a);
            const long long slots = (long long)lds_workgroups(lds) * cu_count * 4;
            const float rounds = (float)(((items << a.share_log) + slots - 1) / slots) / (1 << a.share_log);
            if (best == 0.0f || rounds < 0.97f * best) best = rounds, share_log = a.share_log, shorter = s;
        }
    a.share_log = share_log;
    const long long groups = ((items << share_log) + 3) / 4;
    int rc;
    if (lines) rc = launch_gate_up<XU, kLines ? 3 : 2, kLines>(a, choose, groups, cu_count, stream);
    else rc = shorter ? launch_gate_up<XU, 2, false>(a, choose, groups, cu_count, stream) : launch_gate_up<XU, G, false>(a, choose, groups, cu_count, stream);
    if (!rc) rc = off_lines(a.W2, a.inner) ? launch_down_of<DownBuilds<XU, N, true>>(a, cu_count, stream) : launch_down_of<DownBuilds<XU, N, false>>(a, cu_count, stream);
    if (rc || a.splits == 1) return rc;
    moe_sum_kernel<<<(unsigned)((a.m * (long long)a.hidden + 1023) / 1024), 256, 0, stream>>>(a);
    return launched("moe_sum launch");
}

// How many columns a part has.  An expert's tokens are as many as independent choices of top_k / experts give; each part reads the expert's
// weights, 6 KB a stage of gate, up and down, beside XU KB of activations, which come out of the caches (0.2 of a KB by how it weighed: 32
// tokens on 128 experts 330 us in parts of 4, 312 in parts of 8).
static int part_columns(const MoeArgs& a) {
    const float p = (float)a.top_k / a.experts;
    float cost[4] = {};
    float chance = 1.0f;                                     // of n tokens
    for (int i = 0; i < a.m; i++) chance *= 1.0f - p;
    if (chance < 1e-30f) return a.m <= 4 ? 1 : a.m <= 8 ? 2 : a.m <= 16 ? 4 : 8;      // (nearly) every token
    for (int n = 1; n <= a.m; n++) {
        chance *= (float)(a.m - n + 1) / n * p / (1.0f - p);
        for (int c = 0; c < 4; c++) cost[c] += chance * (float)((n - 1) / (4 << c) + 1) * (6.0f + 0.2f * (1 << c));
    }
    int best = 0;
    for (int c = 1; c < 4 && 2 << c < a.m; c++)              // (twice the columns of a part that holds all tokens cost more)
        if (cost[c] < cost[best]) best = c;
    return 1 << best;
}

// choose: by the logits, in the gate's launch
static int launch_experts(MoeArgs& a, bool choose, int cu_count, hipStream_t stream) {
    switch (part_columns(a)) {
        case 1: return launch_parts<1, 3, 5>(a, choose, cu_count, stream);
        case 2: return launch_parts<2, 3, 4>(a, choose, cu_count, stream);
        case 4: return launch_parts<4, 2, 3>(a, choose, cu_count, stream);
        default: return launch_parts<8, 2, 2>(a, choose, cu_count, stream);
    }
}

}  // namespace sg

using namespace sg;

namespace {
bool off(const void* p, unsigned bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }

// Sizes, pointers that every entry point has, and the workspace.
int begin(MoeArgs& a, const void* X, const int32_t* ids, const float* weights, int m, int hidden, int inner, int experts, int top_k,
          void* workspace, size_t need, size_t workspace_bytes) {
    if (!X || !ids || !weights || !moe_takes(m, hidden, inner, experts, top_k)) return SG_BAD_ARGUMENT;
    if (off(X, 16) || off(ids, 4) || off(weights, 4)) return SG_BAD_ALIGNMENT;
    if (!workspace || workspace_bytes < need) return SG_WORKSPACE_TOO_SMALL;
    if (off(workspace, 256)) return SG_BAD_ALIGNMENT;
    const MoeLayout l = moe_layout(m, hidden, inner, experts, top_k);
    uint8_t* const w = static_cast<uint8_t*>(workspace);
    a.X = static_cast<const uint8_t*>(X);
    a.ids = const_cast<int32_t*>(ids);
    a.weights = const_cast<float*>(weights);
    a.logits = reinterpret_cast<float*>(w);
    a.plan = reinterpret_cast<int32_t*>(w + l.plan_at);
    a.H = w + l.h_at;
    a.sums = reinterpret_cast<float*>(w + l.sums_at);
    a.m = m;
    a.hidden = hidden;
    a.inner = inner;
    a.experts = experts;
    a.top_k = top_k;
    return SG_SUCCESS;
}
int take_experts(MoeArgs& a, const uint8_t* W1, const float* S1, const uint8_t* W2, const float* S2, void* D) {
    if (!W1 || !W2 || !D) return SG_BAD_ARGUMENT;
    if (off(W1, 16) || off(W2, 16) || off(D, 16) || off(S1, 4) || off(S2, 4)) return SG_BAD_ALIGNMENT;
    a.W1 = W1;
    a.S1 = S1;
    a.W2 = W2;
    a.S2 = S2;
    a.D = static_cast<uint16_t*>(D);
    return SG_SUCCESS;
}
int take_router(MoeArgs& a, const void* R, int renormalize) {
    if (!R) return SG_BAD_ARGUMENT;
    if (off(R, 16)) return SG_BAD_ALIGNMENT;
    a.R = static_cast<const uint8_t*>(R);
    a.renormalize = renormalize;
    return SG_SUCCESS;
}
}  // namespace

// Every entry point below holds its stream's turn from its first launch to its last: they hand each other logits, the plan, h and sums
// through the caller's workspace, and another thread's call on the stream, whose plan may be of other sizes, must not come in between.
extern "C" {

size_t sg_moe_workspace_bytes(int m, int hidden, int inner, int experts, int top_k) {
    return moe_takes(m, hidden, inner, experts, top_k) ? moe_layout(m, hidden, inner, experts, top_k).bytes : 0;
}

int sg_moe_route(const void* X, const void* R, int32_t* ids, float* weights, int m, int hidden, int experts, int top_k, int renormalize,
                 void* workspace, size_t workspace_bytes, void* stream) {
    MoeArgs a{};
    if (int rc = begin(a, X, ids, weights, m, hidden, 16, experts, top_k, workspace, (size_t)m * experts * 4, workspace_bytes)) return rc;
    if (int rc = take_router(a, R, renormalize)) return rc;
    DeviceInfo* dev;
    if (int rc = get_device_info(&dev)) return rc;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    std::lock_guard<std::recursive_mutex> turn(stream_turn(st));
    if (int rc = launch_logits(a, st)) return rc;
    return launch_choose(a, st);
}

int sg_moe_experts(const void* X, const int32_t* ids, const float* weights, const uint8_t* W1, const float* S1, const uint8_t* W2,
                   const float* S2, void* D, int m, int hidden, int inner, int experts, int top_k, void* workspace, size_t workspace_bytes,
                   void* stream) {
    MoeArgs a{};
    if (int rc = begin(a, X, ids, weights, m, hidden, inner, experts, top_k, workspace, sg_moe_workspace_bytes(m, hidden, inner, experts, top_k),
                       workspace_bytes))
        return rc;
    if (int rc = take_experts(a, W1, S1, W2, S2, D)) return rc;
    DeviceInfo* dev;
    if (int rc = get_device_info(&dev)) return rc;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    std::lock_guard<std::recursive_mutex> turn(stream_turn(st));
    return launch_experts(a, false, dev->cu_count, st);
}

int sg_moe_layer(const void* X, const void* R, const uint8_t* W1, const float* S1, const uint8_t* W2, const float* S2, void* D, int32_t* ids,
                 float* weights, int m, int hidden, int inner, int experts, int top_k, int renormalize, void* workspace,
                 size_t workspace_bytes, void* stream) {
    MoeArgs a{};
    if (int rc = begin(a, X, ids, weights, m, hidden, inner, experts, top_k, workspace, sg_moe_workspace_bytes(m, hidden, inner, experts, top_k),
                       workspace_bytes))
        return rc;
    if (int rc = take_router(a, R, renormalize)) return rc;
    if (int rc = take_experts(a, W1, S1, W2, S2, D)) return rc;
    DeviceInfo* dev;
    if (int rc = get_device_info(&dev)) return rc;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    std::lock_guard<std::recursive_mutex> turn(stream_turn(st));
    if (int rc = launch_logits(a, st)) return rc;
    const bool fused = m <= kMoeFused;
    if (!fused)
        if (int rc = launch_choose(a, st)) return rc;
    return launch_experts(a, fused, dev->cu_count, st);
}

}  // extern "C"
