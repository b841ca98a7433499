// A mixture-of-experts layer for a few tokens: launches and C entry points (include/sgemm.h).
#include "sg_moe_kernel.h"
#include "sg_moe_route_kernel.h"

namespace sg {

static int launched(const char* what) { return report_hip(what, hipGetLastError()) == hipSuccess ? SG_SUCCESS : SG_LAUNCH_FAILED; }

static int launch_logits(const MoeArgs& a, hipStream_t stream) {
    const unsigned groups = (unsigned)(a.experts + 3) / 4;
    if (a.m == 1) moe_logits_kernel<1><<<dim3(groups, 1), 256, 0, stream>>>(a);
    else if (a.m <= 4) moe_logits_kernel<4><<<dim3(groups, 1), 256, 0, stream>>>(a);
    else moe_logits_kernel<8><<<dim3(groups, (unsigned)(a.m + 7) / 8), 256, 0, stream>>>(a);
    return launched("moe_logits launch");
}

template <int MB>
static int launch_gate_up(const MoeArgs& a, int cu_count, hipStream_t stream) {
    const int pairs = a.m * a.top_k, most = a.experts < pairs ? a.experts : pairs;
    const long long items = (long long)most * (a.inner / 16);
    const int steps = (a.hidden + 127) / 128, waves = steps >= 16 ? 8 : steps >= 8 ? 4 : steps >= 4 ? 2 : 1;
    const unsigned grid = items < 2ll * cu_count ? (unsigned)items : 2u * cu_count;
    const size_t lds = (size_t)moe_plan_layout(a.m, a.experts, a.top_k).dwords * 4 + (size_t)waves * 2 * MB * 1024;
    static LdsGranted granted;
    if (int rc = request_dynamic_lds(reinterpret_cast<const void*>(moe_gate_up_kernel<MB>), lds, granted)) return rc;
    moe_gate_up_kernel<MB><<<grid, 64 * waves, lds, stream>>>(a);
    return launched("moe_gate_up launch");
}

template <int MB>
static int launch_down(const MoeArgs& a, int cu_count, hipStream_t stream) {
    (void)cu_count;
    const int waves = 8;
    const size_t lds = (size_t)moe_plan_layout(a.m, a.experts, a.top_k).dwords * 4 + (size_t)waves * a.m * 64;
    static LdsGranted granted;
    if (int rc = request_dynamic_lds(reinterpret_cast<const void*>(moe_down_kernel<MB>), lds, granted)) return rc;
    moe_down_kernel<MB><<<a.hidden / 16, 64 * waves, lds, stream>>>(a);
    return launched("moe_down launch");
}

static int launch_experts(const MoeArgs& a, int cu_count, hipStream_t stream) {
    if (int rc = a.m <= 16 ? launch_gate_up<1>(a, cu_count, stream) : a.m <= 32 ? launch_gate_up<2>(a, cu_count, stream) : launch_gate_up<4>(a, cu_count, stream))
        return rc;
    return a.m <= 16 ? launch_down<1>(a, cu_count, stream) : a.m <= 32 ? launch_down<2>(a, cu_count, stream) : launch_down<4>(a, cu_count, stream);
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
    moe_plan_kernel<true, false><<<(unsigned)(m + 7) / 8, 512, 0, st>>>(a);
    return launched("moe_choose launch");
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
    moe_plan_kernel<false, true><<<1, 512, 0, st>>>(a);
    if (int rc = launched("moe_plan launch")) return rc;
    return launch_experts(a, dev->cu_count, st);
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
    moe_plan_kernel<true, true><<<1, 512, 0, st>>>(a);
    if (int rc = launched("moe_plan launch")) return rc;
    return launch_experts(a, dev->cu_count, st);
}

}  // extern "C"
