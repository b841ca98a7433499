// MXFP4 codec for gfx950: quantising bf16 rows, bringing codes back to bf16, and laying weights out for the matrix
// instruction (sg_mx.h).  The format's scale rule (OCP Microscaling v1.0, 6.3):
//
//   e    = floor(log2(absmax of the block)) - 2          (2 = exponent of E2M1's largest value)
//   S    = clamp(e + 127, 0, 254), 127 for a block of zeros, 255 for one with a NaN or an infinity (its codes are 0)
//   code = e2m1_rne_sat(x / 2^(S - 127))
//
// floor(log2) of a bf16 is its exponent field, so S = max(field - 2, 0) without a logarithm, and the largest magnitude is
// the largest bit pattern: packed 16-bit integer maxima.  Dividing by a power of two is exact; v_cvt_scalef32_pk_fp4_bf16
// divides, rounds to nearest even and saturates two values at once (all bf16 values checked against the formula under 14
// scales, both ends of the range among them), and v_cvt_scalef32_pk_bf16_fp4 is its exact inverse.
//
// Rows are contiguous and a block never crosses two, so both kernels see one sequence of blocks and no rows.  They are
// HBM-bound at 2 + 17/32 bytes a value: 28672 x 4096 there and back 89.6 us = 6.6 TB/s, decoding 4096 x 14336 24.7 us = 6.0.  Eight
// values a lane keep loads and stores contiguous over a wave (1 KB of bf16, 256 bytes of codes); with a block of 32 a lane
// the 64-byte pieces of neighbours would interleave, which costs such streams a third (sg_codec.hip).
//
// Packing reads 64 bytes of each of 16 rows for every KB it writes, and each byte of codes and scales is moved once: 28672 x 4096 28.2 us = 4.4 TB/s
// there and back, against 19 at the codec's rate; 57344 x 8192 120.5.  Once a weight matrix, so that the simple form stays.
#include "sg_mx.h"

namespace sg {

typedef __bf16 bf16v2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16v2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t max_halves(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16v2, a), __builtin_bit_cast(u16v2, b)));
}
// the float 2^(S - 127); 2^-127 is subnormal
__device__ __forceinline__ float mx_scale(unsigned S) { return __uint_as_float(S == 0 ? 0x00400000u : S << 23); }

// A lane takes 8 values of a chunk and four lanes a block; a wave's chunk is 512 values, 1 KB in and 256 bytes out.
constexpr int kMxChunks = 4;       // chunks of a wave: loads in flight

__global__ void __launch_bounds__(256) mx_encode_kernel(const u32x4* __restrict__ X, uint32_t* __restrict__ Q,
                                                        uint8_t* __restrict__ S, size_t blocks) {
    const int lane = lane_id();
    const size_t first = ((size_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * (16 * kMxChunks);      // the wave's first block
    u32x4 raw[kMxChunks];
#pragma unroll
    for (int c = 0; c < kMxChunks; c++) {
        const size_t block = first + c * 16 + (lane >> 2);
        // a lane beyond the end takes the last block again and stores nothing
        raw[c] = __builtin_nontemporal_load(X + (block < blocks ? block : blocks - 1) * 4 + (lane & 3));
    }
#pragma unroll
    for (int c = 0; c < kMxChunks; c++) {
        const size_t block = first + c * 16 + (lane >> 2);
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) top = max_halves(top, raw[c][j] & 0x7fff7fffu);
        top = max_halves(top, __builtin_amdgcn_update_dpp(0, top, 0xb1, 0xf, 0xf, false));     // quad_perm [1, 0, 3, 2]
        top = max_halves(top, __builtin_amdgcn_update_dpp(0, top, 0x4e, 0xf, 0xf, false));     // quad_perm [2, 3, 0, 1]
        const unsigned amax = (top & 0xffffu) > (top >> 16) ? (top & 0xffffu) : (top >> 16);
        const unsigned field = amax >> 7;
        const unsigned s = amax == 0 ? 127u : field == 255u ? 255u : field > 2u ? field - 2u : 0u;
        const float by = mx_scale(s == 255u ? 127u : s);
        const uint32_t w0 = raw[c].x, w1 = raw[c].y, w2 = raw[c].z, w3 = raw[c].w;   // (a bit cast of a vector's element takes the first)
        uint32_t q = 0;
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(bf16v2, w0), by, 0);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(bf16v2, w1), by, 1);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(bf16v2, w2), by, 2);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(bf16v2, w3), by, 3);
        if (s == 255u) q = 0;
        if (block < blocks) {
            Q[block * 4 + (lane & 3)] = q;
            if ((lane & 3) == 0) S[block] = (uint8_t)s;
        }
    }
}

__global__ void __launch_bounds__(256) mx_decode_kernel(const uint32_t* __restrict__ Q, const uint8_t* __restrict__ S,
                                                        u32x4* __restrict__ Y, size_t blocks) {
    const int lane = lane_id();
    const size_t first = ((size_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * (16 * kMxChunks);
    uint32_t q[kMxChunks];
    unsigned s[kMxChunks];
#pragma unroll
    for (int c = 0; c < kMxChunks; c++) {
        const size_t block = first + c * 16 + (lane >> 2), at = block < blocks ? block : blocks - 1;
        q[c] = __builtin_nontemporal_load(Q + at * 4 + (lane & 3));
        s[c] = S[at];
    }
#pragma unroll
    for (int c = 0; c < kMxChunks; c++) {
        const size_t block = first + c * 16 + (lane >> 2);
        const float by = mx_scale(s[c]);          // 255: a float of that exponent, which the conversion takes as NaN
        u32x4 y;
        y[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q[c], by, 0));
        y[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q[c], by, 1));
        y[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q[c], by, 2));
        y[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q[c], by, 3));
        if (block < blocks) __builtin_nontemporal_store(y, Y + block * 4 + (lane & 3));
    }
}

// One wave a step of a tile (1 KB of codes), and the scales of the four steps of a group with the first of them.
__global__ void __launch_bounds__(256) mx_pack_kernel(const uint8_t* __restrict__ B, const uint8_t* __restrict__ SB,
                                                      uint8_t* __restrict__ P, uint8_t* __restrict__ PS, int n, int k_blocks,
                                                      int pitch, int quads, int b_stride) {
    const int lane = lane_id(), r = lane & 15, g = lane >> 4;
    const size_t tile = blockIdx.x;
    const size_t row = tile * 16 + r;
    const bool live = row < (size_t)n;
    for (int step = blockIdx.y * 4 + (int)(threadIdx.x >> 6); step < pitch; step += gridDim.y * 4) {
        const int block = step * 4 + g;
        u32x4 codes = {0, 0, 0, 0};
        if (live && block < k_blocks) codes = *reinterpret_cast<const u32x4*>(B + row * (size_t)b_stride + (size_t)block * 16);
        *reinterpret_cast<u32x4*>(P + (tile * pitch + step) * kMxStepBytes + lane * 16) = codes;
        if (step % 4 == 0) {
            uint32_t s = 0;
#pragma unroll
            for (int t = 0; t < 4; t++) {
                const int b = block + 4 * t;
                s |= (uint32_t)(live && b < k_blocks ? SB[row * (size_t)k_blocks + b] : 127) << (8 * t);
            }
            *reinterpret_cast<uint32_t*>(PS + (tile * quads + step / 4) * kMxQuadBytes + lane * 4) = s;
        }
    }
}

// Block scales of activations on rows of whole groups of four steps, 16 bytes each, for the wide kernel's direct loads: 16 bytes a lane.
__global__ void __launch_bounds__(256) mx_scale_rows_kernel(const uint8_t* __restrict__ SA, u32x4* __restrict__ out, unsigned m, unsigned quads,
                                                            unsigned inv_quads, int k_blocks) {
    const unsigned at = blockIdx.x * 256 + threadIdx.x;
    const unsigned row = fast_div(at, quads, inv_quads), q = at - row * quads;
    if (row >= m) return;
    const uint8_t* s = SA + (size_t)row * k_blocks + 16 * (size_t)q;
    u32x4 v;
    if (16 * (int)q + 16 <= k_blocks) {
        __builtin_memcpy(&v, s, 16);
    } else {
        const int have = k_blocks - 16 * (int)q;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            v[e] = 0;
#pragma unroll
            for (int b = 0; b < 4; b++) v[e] |= (uint32_t)(4 * e + b < have ? s[4 * e + b] : 127) << (8 * b);
        }
    }
    out[at] = v;
}

int launch_mx_scale_rows(const uint8_t* SA, uint8_t* out, int m, int k, int quads, hipStream_t stream) {
    const unsigned pieces = (unsigned)m * (unsigned)quads;               // (the caller keeps it below 2^31)
    mx_scale_rows_kernel<<<(pieces + 255) / 256, 256, 0, stream>>>(SA, reinterpret_cast<u32x4*>(out), (unsigned)m, (unsigned)quads,
                                                                   div_reciprocal((unsigned)quads), k / kMxBlock);
    return report_hip("mx_scale_rows launch", hipGetLastError()) == hipSuccess ? SG_SUCCESS : SG_LAUNCH_FAILED;
}

static unsigned mx_codec_grid(size_t blocks) { return (unsigned)((blocks + 64 * kMxChunks - 1) / (64 * kMxChunks)); }

int launch_mx_encode(const void* X, uint8_t* Q, uint8_t* S, int rows, int cols, hipStream_t stream) {
    const size_t blocks = (size_t)rows * (size_t)(cols / kMxBlock);
    mx_encode_kernel<<<mx_codec_grid(blocks), 256, 0, stream>>>(static_cast<const u32x4*>(X), reinterpret_cast<uint32_t*>(Q), S, blocks);
    return report_hip("mx_encode launch", hipGetLastError()) == hipSuccess ? SG_SUCCESS : SG_LAUNCH_FAILED;
}

int launch_mx_decode(const uint8_t* Q, const uint8_t* S, void* Y, int rows, int cols, hipStream_t stream) {
    const size_t blocks = (size_t)rows * (size_t)(cols / kMxBlock);
    mx_decode_kernel<<<mx_codec_grid(blocks), 256, 0, stream>>>(reinterpret_cast<const uint32_t*>(Q), S, static_cast<u32x4*>(Y), blocks);
    return report_hip("mx_decode launch", hipGetLastError()) == hipSuccess ? SG_SUCCESS : SG_LAUNCH_FAILED;
}

int launch_mx_pack(const uint8_t* B, const uint8_t* SB, uint8_t* P, int n, int k, int b_stride, hipStream_t stream) {
    const MxLayout l = mx_layout(n, k);
    const unsigned gy = l.quads < 65535 ? (unsigned)l.quads : 65535u;
    mx_pack_kernel<<<dim3((unsigned)l.tiles, gy), 256, 0, stream>>>(B, SB, P, P + l.scales_at, n, k / kMxBlock, l.pitch, l.quads, b_stride);
    return report_hip("mx_pack launch", hipGetLastError()) == hipSuccess ? SG_SUCCESS : SG_LAUNCH_FAILED;
}

}  // namespace sg
