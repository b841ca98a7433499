// MXFP4 in this library: what its translation units share.
//
// Values: 32 neighbouring columns of a row share a scale 2^(S - 127), one byte S, 255 = NaN; every value is an E2M1 code
// (sign, exponent, mantissa: 0, 0.5, 1, 1.5, 2, 3, 4, 6), two a byte, the even column in the low nibble.
//
// Weights are multiplied from a packed buffer, laid out once when a program loads them.  v_mfma_scale_f32_16x16x128 takes
// 16 weight rows and 128 columns: lane l (row l % 16, block l / 16) holds the 16 bytes of one block of its row and its
// scale.  The buffer holds exactly that, so that a wave loads operands as they are, 1 KB contiguous at a time, without a
// pass through LDS:
//     codes   [n / 16][k / 128][64 lanes][16 bytes]    (an even number of 128-column steps)
//     scales  [n / 16][k / 512][64 lanes][4 bytes]     byte t of a lane: its block of step t of the 512 columns (op_sel)
// with n, k rounded up; what is beyond the matrix holds code 0 and scale 1.
#pragma once

#include "sg_device.h"
#include "sg_host.h"

namespace sg {

constexpr int kMxBlock = 32;       // columns that share a scale
constexpr int kMxStepBytes = 1024; // codes of 16 rows x 128 columns
constexpr int kMxQuadBytes = 256;  // scales of 16 rows x 512 columns

struct MxLayout {
    int tiles, steps, quads;       // 16-row tiles, 128-column steps with columns of the matrix, 512-column groups
    int pitch;                     // steps of a tile in the buffer
    size_t scales_at, bytes;
};
inline MxLayout mx_layout(int n, int k) {
    MxLayout l;
    l.tiles = (int)(((unsigned)n + 15) / 16);
    l.steps = (int)(((unsigned)k + 127) / 128);
    l.quads = (l.steps + 3) / 4;
    l.pitch = (l.steps + 1) / 2 * 2;
    l.scales_at = (size_t)l.tiles * l.pitch * kMxStepBytes;
    l.bytes = l.scales_at + (size_t)l.tiles * l.quads * kMxQuadBytes;
    return l;
}

struct MxArgs {
    const uint8_t* A;         // activations [m][k] E4M3, or [m][k / 2] codes
    const uint8_t* SA;        // [m][k / 32] scales of the codes
    const uint8_t* P;         // packed codes
    const uint8_t* PS;        // packed scales
    uint16_t* D;              // [m][n] bf16
    const float* scale;       // one factor, or NULL
    const float* row_scale;   // [m] factors, or NULL
    int m, n, k;
    int tiles, steps, quads, pitch;  // MxLayout
    const uint8_t* SX;        // the wide kernel's copy of SA: [m][quads * 16], or SA itself where that is its layout
    int n_groups, m_groups;   // workgroup tiles along n and m
    int splits;               // workgroups that share K of a tile, by whole groups of four steps
    float* ws;                // splits > 1: their sums, [split][m / 16][n / 16][64 lanes][4], added by a second launch
};

int launch_mx_encode(const void* X, uint8_t* Q, uint8_t* S, int rows, int cols, hipStream_t stream);
int launch_mx_decode(const uint8_t* Q, const uint8_t* S, void* Y, int rows, int cols, hipStream_t stream);
int launch_mx_pack(const uint8_t* B, const uint8_t* SB, uint8_t* P, int n, int k, int b_stride, hipStream_t stream);
int launch_mx_scale_rows(const uint8_t* SA, uint8_t* out, int m, int k, int quads, hipStream_t stream);
// fp4: activations in MXFP4, otherwise E4M3; build: 0 = the library's choice (sg_mx_gemm.hip)
int mx_choice(bool fp4, int m, int n, int k, int cu_count, bool workspace);
int mx_searches();
int launch_mx_gemm(bool fp4, int build, MxArgs& a, int cu_count, hipStream_t stream);

}  // namespace sg
