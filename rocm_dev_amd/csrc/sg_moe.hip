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

constexpr size_t kLdsBytes = 160 * 1024;      // a CU's

template <int XU, int DEPTH>
static size_t gate_up_lds(const MoeArgs& a) {
    using Stages = MoeStages<2, XU>;
    const size_t ring = (size_t)4 * DEPTH * Stages::kBytes, room = moe_plan_room(a.m * a.top_k);
    return (size_t)moe_plan_layout(a.m, a.experts, a.top_k).dwords * 4 + (a.share > 1 ? 4 * 2 * Stages::kBlocks * 1024 : 0) + (room > ring ? room : ring);
}
template <int XU, int DEPTH, bool CHOOSE>
static int launch_gate_up(const MoeArgs& a, long long groups, int cu_count, hipStream_t stream) {
    const size_t lds = gate_up_lds<XU, DEPTH>(a);
    const long long at_once = (long long)(kLdsBytes / lds) * cu_count;
    const unsigned grid = (unsigned)(groups < at_once ? groups : at_once);
    static LdsGranted granted;
    if (int rc = request_dynamic_lds(reinterpret_cast<const void*>(moe_gate_up_kernel<XU, DEPTH, CHOOSE>), lds, granted)) return rc;
    moe_gate_up_kernel<XU, DEPTH, CHOOSE><<<grid, 256, lds, stream>>>(a);
    return launched("moe_gate_up launch");
}

template <int XU, int DEPTH, int WAVES>
static size_t down_lds(const MoeArgs& a) {
    const MoePlanLayout l = moe_plan_layout(a.m, a.experts, a.top_k);
    return (size_t)l.dwords * 4 + (size_t)l.most * 64 + (size_t)WAVES * a.m * 64 + (size_t)WAVES * DEPTH * MoeStages<1, XU>::kBytes;
}
template <int XU, int DEPTH, int WAVES>
static int launch_down(const MoeArgs& a, hipStream_t stream) {
    const size_t lds = down_lds<XU, DEPTH, WAVES>(a);
    static LdsGranted granted;
    if (int rc = request_dynamic_lds(reinterpret_cast<const void*>(moe_down_kernel<XU, DEPTH, WAVES>), lds, granted)) return rc;
    moe_down_kernel<XU, DEPTH, WAVES><<<a.hidden / 16, 64 * WAVES, lds, stream>>>(a);
    return launched("moe_down launch");
}

// Parts of up to 4 * XU tokens; G and N stages in flight a wave.
template <int XU, int G, int N>
static int launch_parts(MoeArgs& a, bool choose, int cu_count, hipStream_t stream) {
    const int pairs = a.m * a.top_k, most = a.experts < pairs ? a.experts : pairs, steps = (a.hidden + 127) / 128;
    const long long items = (long long)most * (a.inner / 16);
    a.share = 1;
    while (a.share < 4 && items * a.share < 16ll * cu_count && steps >= 4 * a.share) a.share *= 2;
    const long long groups = (items * a.share + 3) / 4;
    // A few workgroups more than fit at once would take as long again: shorter rings then, if all fit with them.
    const bool shorter = groups > (long long)(kLdsBytes / gate_up_lds<XU, G>(a)) * cu_count && groups <= (long long)(kLdsBytes / gate_up_lds<XU, 2>(a)) * cu_count;
    int rc;
    if (choose) rc = shorter ? launch_gate_up<XU, 2, true>(a, groups, cu_count, stream) : launch_gate_up<XU, G, true>(a, groups, cu_count, stream);
    else rc = shorter ? launch_gate_up<XU, 2, false>(a, groups, cu_count, stream) : launch_gate_up<XU, G, false>(a, groups, cu_count, stream);
    if (rc) return rc;
    if (down_lds<XU, N, 8>(a) <= kLdsBytes) return launch_down<XU, N, 8>(a, stream);
    if (down_lds<XU, 2, 8>(a) <= kLdsBytes) return launch_down<XU, 2, 8>(a, stream);
    return launch_down<XU, 2, 4>(a, stream);
}
// choose: by the logits, in the gate's launch
static int launch_experts(MoeArgs& a, bool choose, int cu_count, hipStream_t stream) {
    // Columns for an expert's tokens: as many as independent choices of m * top_k / experts on average rarely exceed.
    const float mean = (float)a.m * a.top_k / a.experts, want = mean + 3.0f * sqrtf(mean);
    const float columns = want < a.m ? want : a.m;
    if (columns <= 4) return launch_parts<1, 3, 5>(a, choose, cu_count, stream);
    if (columns <= 8) return launch_parts<2, 3, 4>(a, choose, cu_count, stream);
    if (columns <= 16) return launch_parts<4, 2, 3>(a, choose, cu_count, stream);
    return launch_parts<8, 2, 2>(a, choose, cu_count, stream);
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
    const MoeLayout l = moe_layout(m, inner, experts, top_k);
    uint8_t* const w = static_cast<uint8_t*>(workspace);
    a.X = static_cast<const uint8_t*>(X);
    a.ids = const_cast<int32_t*>(ids);
    a.weights = const_cast<float*>(weights);
    a.logits = reinterpret_cast<float*>(w);
    a.plan = reinterpret_cast<int32_t*>(w + l.plan_at);
    a.H = w + l.h_at;
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

extern "C" {

size_t sg_moe_workspace_bytes(int m, int hidden, int inner, int experts, int top_k) {
    return moe_takes(m, hidden, inner, experts, top_k) ? moe_layout(m, inner, experts, top_k).bytes : 0;
}

int sg_moe_route(const void* X, const void* R, int32_t* ids, float* weights, int m, int hidden, int experts, int top_k, int renormalize,
                 void* workspace, size_t workspace_bytes, void* stream) {
    MoeArgs a{};
    if (int rc = begin(a, X, ids, weights, m, hidden, 16, experts, top_k, workspace, (size_t)m * experts * 4, workspace_bytes)) return rc;
    if (int rc = take_router(a, R, renormalize)) return rc;
    DeviceInfo* dev;
    if (int rc = get_device_info(&dev)) return rc;
    const hipStream_t st = static_cast<hipStream_t>(stream);
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
    return launch_experts(a, false, dev->cu_count, static_cast<hipStream_t>(stream));
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
    if (int rc = launch_logits(a, st)) return rc;
    const bool fused = m <= kMoeFused;
    if (!fused)
        if (int rc = launch_choose(a, st)) return rc;
    return launch_experts(a, fused, dev->cu_count, st);
}

}  // extern "C"
