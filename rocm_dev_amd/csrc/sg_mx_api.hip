// C entry points of the MXFP4 operators (include/sgemm.h): every argument is checked here, before anything is launched.
#include "../../include/sgemm_debug.h"
#include "sg_mx.h"

using namespace sg;

namespace {
bool off16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

int gemm(bool fp4, int build, const uint8_t* A, const uint8_t* SA, const uint8_t* P, void* D, const float* scale,
         const float* row_scales, int m, int n, int k, void* stream) {
    if (!A || (fp4 && !SA) || !P || !D || m <= 0 || n <= 0 || k <= 0) return SG_BAD_ARGUMENT;
    if (k % kMxBlock) return SG_K_NOT_DIVISIBLE_BY_WARPTILE_K;
    if (off16(A) || off16(P) || (reinterpret_cast<uintptr_t>(D) & 7u)) return SG_BAD_ALIGNMENT;
    DeviceInfo* dev;
    if (int rc = get_device_info(&dev)) return rc;
    const MxLayout l = mx_layout(n, k);
    MxArgs a{};
    a.A = A;
    a.SA = SA;
    a.P = P;
    a.PS = P + l.scales_at;
    a.D = static_cast<uint16_t*>(D);
    a.scale = scale;
    a.row_scale = row_scales;
    a.m = m;
    a.n = n;
    a.k = k;
    a.tiles = l.tiles;
    a.steps = l.steps;
    a.quads = l.quads;
    a.pitch = l.pitch;
    return launch_mx_gemm(fp4, build, a, dev->cu_count, static_cast<hipStream_t>(stream));
}
}  // namespace

extern "C" {

int sg_mxfp4_encode_rows(const void* X, uint8_t* Q, uint8_t* S, int rows, int cols, void* stream) {
    if (!X || !Q || !S || rows <= 0 || cols <= 0 || cols % kMxBlock) return SG_BAD_ARGUMENT;
    if (off16(X) || off16(Q)) return SG_BAD_ALIGNMENT;
    DeviceInfo* dev;
    if (int rc = get_device_info(&dev)) return rc;
    return launch_mx_encode(X, Q, S, rows, cols, static_cast<hipStream_t>(stream));
}

int sg_mxfp4_decode_rows(const uint8_t* Q, const uint8_t* S, void* Y, int rows, int cols, void* stream) {
    if (!Q || !S || !Y || rows <= 0 || cols <= 0 || cols % kMxBlock) return SG_BAD_ARGUMENT;
    if (off16(Q) || off16(Y)) return SG_BAD_ALIGNMENT;
    DeviceInfo* dev;
    if (int rc = get_device_info(&dev)) return rc;
    return launch_mx_decode(Q, S, Y, rows, cols, static_cast<hipStream_t>(stream));
}

size_t sg_mxfp4_packed_bytes(int n, int k) { return n <= 0 || k <= 0 || k % kMxBlock ? 0 : mx_layout(n, k).bytes; }

int sg_mxfp4_pack(const uint8_t* B, const uint8_t* B_scales, uint8_t* P, int n, int k, int b_stride, void* stream) {
    if (!B || !B_scales || !P || n <= 0 || k <= 0 || b_stride < k / 2) return SG_BAD_ARGUMENT;
    if (k % kMxBlock) return SG_K_NOT_DIVISIBLE_BY_WARPTILE_K;
    if (off16(B) || (b_stride & 15) || off16(P)) return SG_BAD_ALIGNMENT;
    DeviceInfo* dev;
    if (int rc = get_device_info(&dev)) return rc;
    return launch_mx_pack(B, B_scales, P, n, k, b_stride, static_cast<hipStream_t>(stream));
}

int sg_mxfp4_gemm(const uint8_t* A, const uint8_t* A_scales, const uint8_t* P, void* D, const float* scale_tensor, int m, int n, int k,
                  void* stream) {
    return gemm(true, 0, A, A_scales, P, D, scale_tensor, nullptr, m, n, k, stream);
}

int sg_mxfp4_gemm_fp8act(const uint8_t* A, const uint8_t* P, void* D, const float* scale_tensor, const float* row_scales, int m, int n, int k,
                         void* stream) {
    return gemm(false, 0, A, nullptr, P, D, scale_tensor, row_scales, m, n, k, stream);
}

int sg_debug_mxfp4_gemm(const uint8_t* A, const uint8_t* A_scales, const uint8_t* P, void* D, const float* scale_tensor,
                        const float* row_scales, int m, int n, int k, int build, void* stream) {
    return gemm(A_scales != nullptr, build, A, A_scales, P, D, scale_tensor, row_scales, m, n, k, stream);
}

int sg_debug_mxfp4_choice(int fp4_activations, int m, int n, int k, int workspace) {
    if (m <= 0 || n <= 0 || k <= 0 || k % kMxBlock) return 0;
    return mx_choice(fp4_activations != 0, m, n, k, 256, workspace != 0);
}

int sg_debug_mxfp4_searches(void) { return mx_searches(); }

}  // extern "C"
