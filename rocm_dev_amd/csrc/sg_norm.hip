// Root-mean-square norm of bf16 rows, the residual added first, into E4M3 rows with a scale each (include/sgemm.h).
//
//   v = bf16(X + residual);   y = v * w * rstd,  rstd = 1 / sqrt(sum(v^2) / cols + eps);   s = absmax(y) / 448;   Q = e4m3(y / s)
//
// v * w is a product of two bf16 values, exact in fp32, and rstd is one factor of the whole row, so absmax(y) is rstd * max|v * w|
// to the bit: the sum of squares and the maximum come out of the same pass over the row and one reduction.  A row is held
// in registers between the reduction and the codes: it is read from memory once.
// fp32 throughout; roundings to fewer bits are the three outputs' own (v as bf16, since the next layer adds to what is
// stored; the codes; Y).  y / s is a product with 1 / s: y itself carries the rounding of its sum of squares, so that a correctly rounded
// quotient (as the encoder's, whose input is exact) would mean nothing here.
#include <cmath>

#include "sg_device.h"
#include "sg_host.h"
#include "sg_quant.h"

namespace sg {

struct NormArgs {
    const uint8_t* X;
    const uint8_t* residual;     // or NULL
    const uint8_t* weight;       // or NULL
    uint8_t* sum;                // or NULL
    uint8_t* Y;                  // or NULL
    uint8_t* Q;
    float* scales;
    float eps;
    int rows, cols;
};

// Of what a thread has seen of its row.
struct RowSums {
    float squares, top;          // sum of v^2, max |v * w|
};

struct RowFactors {
    float rstd, s, inv;
    bool divide;                 // 1 / s does not stand for s
};
__device__ __forceinline__ RowFactors row_factors(RowSums r, int cols, float eps) {
    RowFactors f;
    f.rstd = 1.0f / sqrtf(r.squares / (float)cols + eps);
    float top = r.top * f.rstd;
    if (!(top > 0.0f)) top = 0.0f;                       // also NaN: an infinity times zero, or a row that holds a NaN
    f.s = top == 0.0f ? 1.0f : __fdiv_rn(top, 448.0f);
    f.inv = __fdiv_rn(1.0f, f.s);
    f.divide = !(f.s >= 0x1p-120f && f.s <= 0x1p120f);
    return f;
}

// v of eight columns, as bf16 holds it
__device__ __forceinline__ u32x4 add_bf16(u32x4 x, u32x4 r) {
    u32x4 v;
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = pack_bf16x2(bf16_lo(x[j]) + bf16_lo(r[j]), bf16_hi(x[j]) + bf16_hi(r[j]));
    return v;
}
__device__ __forceinline__ void see(RowSums& r, u32x4 v, u32x4 w) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float lo = bf16_lo(v[j]), hi = bf16_hi(v[j]);
        r.squares = fmaf(lo, lo, r.squares);
        r.squares = fmaf(hi, hi, r.squares);
        r.top = fmaxf(r.top, fmaxf(fabsf(lo * bf16_lo(w[j])), fabsf(hi * bf16_hi(w[j]))));
    }
}
template <bool DIVIDE>
__device__ __forceinline__ u32x2 codes_of(const float (&y)[8], const RowFactors& f) {
    float q[8];
#pragma unroll
    for (int j = 0; j < 8; j++) q[j] = DIVIDE ? __fdiv_rn(y[j], f.s) : y[j] * f.inv;
    int w0 = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
    w0 = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], w0, true);
    int w1 = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], 0, false);
    w1 = __builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], w1, true);
    return u32x2{canonical_nan_codes(w0), canonical_nan_codes(w1)};
}
// codes and Y of eight columns, `at` chunks into the matrix
__device__ __forceinline__ void put(const NormArgs& a, size_t at, u32x4 v, u32x4 w, const RowFactors& f) {
    float y[8];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        y[2 * j] = bf16_lo(v[j]) * bf16_lo(w[j]) * f.rstd;
        y[2 * j + 1] = bf16_hi(v[j]) * bf16_hi(w[j]) * f.rstd;
    }
    reinterpret_cast<u32x2*>(a.Q)[at] = f.divide ? codes_of<true>(y, f) : codes_of<false>(y, f);
    if (a.Y) {
        u32x4 o;
#pragma unroll
        for (int j = 0; j < 4; j++) o[j] = pack_bf16x2(y[2 * j], y[2 * j + 1]);
        reinterpret_cast<u32x4*>(a.Y)[at] = o;
    }
}
constexpr unsigned kOnes = 0x3f803f80u;      // two bf16 ones

// A thread's chunks of its row: t, t + STEP, ...  One past the row's end takes the last chunk again, counts nothing and stores nothing.
template <int STEP, int CH>
struct RowChunks {
    u32x4 v[CH], w[CH];

    __device__ __forceinline__ RowSums load(const NormArgs& a, size_t row, int t, int nchunks) {
        const u32x4* const x = reinterpret_cast<const u32x4*>(a.X) + row * nchunks;
        const u32x4* const res = reinterpret_cast<const u32x4*>(a.residual) + row * nchunks;
        const u32x4* const wt = reinterpret_cast<const u32x4*>(a.weight);
        u32x4 r[CH];
#pragma unroll
        for (int c = 0; c < CH; c++) v[c] = __builtin_nontemporal_load(x + at(c, t, nchunks));
        if (a.residual) {
#pragma unroll
            for (int c = 0; c < CH; c++) r[c] = __builtin_nontemporal_load(res + at(c, t, nchunks));
        }
        if (a.weight) {
#pragma unroll
            for (int c = 0; c < CH; c++) w[c] = wt[at(c, t, nchunks)];
        } else {
#pragma unroll
            for (int c = 0; c < CH; c++) w[c] = u32x4{kOnes, kOnes, kOnes, kOnes};
        }
        if (a.residual) {
#pragma unroll
            for (int c = 0; c < CH; c++) v[c] = add_bf16(v[c], r[c]);
        }
        RowSums sums = {0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < CH; c++)
            if (c * STEP + t < nchunks) see(sums, v[c], w[c]);
        return sums;
    }
    __device__ __forceinline__ void store(const NormArgs& a, size_t row, int t, int nchunks, const RowFactors& f) {
#pragma unroll
        for (int c = 0; c < CH; c++)
            if (c * STEP + t < nchunks) {
                const size_t to = row * nchunks + c * STEP + t;
                if (a.sum) reinterpret_cast<u32x4*>(a.sum)[to] = v[c];
                put(a, to, v[c], w[c], f);
            }
    }
    static __device__ __forceinline__ int at(int c, int t, int nchunks) { return c * STEP + t < nchunks ? c * STEP + t : nchunks - 1; }
};

template <int LANES>
__device__ __forceinline__ RowSums over_lanes(RowSums r) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
        r.squares += __shfl_xor(r.squares, o);
        r.top = fmaxf(r.top, __shfl_xor(r.top, o));
    }
    return r;
}
// over a workgroup, in wave order
template <int THREADS>
__device__ __forceinline__ RowSums over_threads(RowSums r) {
    __shared__ RowSums of_wave[THREADS / 64];
    r = over_lanes<64>(r);
    if (THREADS == 64) return r;
    if (lane_id() == 0) of_wave[threadIdx.x >> 6] = r;
    __syncthreads();
    r = of_wave[0];
#pragma unroll
    for (int w = 1; w < THREADS / 64; w++) {
        r.squares += of_wave[w].squares;
        r.top = fmaxf(r.top, of_wave[w].top);
    }
    return r;
}

// One workgroup a row.
template <int THREADS, int CH>
__global__ void __launch_bounds__(THREADS) rmsnorm_row_kernel(const NormArgs a) {
    const int t = threadIdx.x, nchunks = a.cols >> 3;
    RowChunks<THREADS, CH> row;
    const RowSums sums = over_threads<THREADS>(row.load(a, blockIdx.x, t, nchunks));
    const RowFactors f = row_factors(sums, a.cols, a.eps);
    if (t == 0) a.scales[blockIdx.x] = f.s;
    row.store(a, blockIdx.x, t, nchunks, f);
}

// Short rows: LANES lanes of a wave share one.
template <int LANES, int CH>
__global__ void __launch_bounds__(256) rmsnorm_short_rows_kernel(const NormArgs a) {
    const unsigned mine = blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    const unsigned at = mine < (unsigned)a.rows ? mine : (unsigned)a.rows - 1;      // lanes past the last row store nothing
    const int t = (int)threadIdx.x % LANES, nchunks = a.cols >> 3;
    RowChunks<LANES, CH> row;
    const RowSums sums = over_lanes<LANES>(row.load(a, at, t, nchunks));
    if (mine >= (unsigned)a.rows) return;
    const RowFactors f = row_factors(sums, a.cols, a.eps);
    if (t == 0) a.scales[mine] = f.s;
    row.store(a, mine, t, nchunks, f);
}

// Rows beyond 65536 columns: two passes; v is read again where it is stored, and formed again where it is not.  (Its sum may
// lie where the residual was: a thread reads and writes the same chunks in both passes.)
__global__ void __launch_bounds__(1024) rmsnorm_long_rows_kernel(const NormArgs a) {
    const int t = threadIdx.x, nchunks = a.cols >> 3;
    const size_t first = (size_t)blockIdx.x * nchunks;
    const u32x4 ones = {kOnes, kOnes, kOnes, kOnes};
    RowSums sums = {0.0f, 0.0f};
    for (int c = t; c < nchunks; c += 1024) {
        u32x4 v = reinterpret_cast<const u32x4*>(a.X)[first + c];
        if (a.residual) v = add_bf16(v, reinterpret_cast<const u32x4*>(a.residual)[first + c]);
        if (a.sum) reinterpret_cast<u32x4*>(a.sum)[first + c] = v;
        see(sums, v, a.weight ? reinterpret_cast<const u32x4*>(a.weight)[c] : ones);
    }
    const RowFactors f = row_factors(over_threads<1024>(sums), a.cols, a.eps);
    if (t == 0) a.scales[blockIdx.x] = f.s;
    for (int c = t; c < nchunks; c += 1024) {
        u32x4 v;
        if (a.sum) {
            v = reinterpret_cast<const u32x4*>(a.sum)[first + c];
        } else {
            v = reinterpret_cast<const u32x4*>(a.X)[first + c];
            if (a.residual) v = add_bf16(v, reinterpret_cast<const u32x4*>(a.residual)[first + c]);
        }
        put(a, first + c, v, a.weight ? reinterpret_cast<const u32x4*>(a.weight)[c] : ones, f);
    }
}

static int launch(const NormArgs& a, hipStream_t stream) {
    const int nchunks = a.cols >> 3;
    const unsigned rows = (unsigned)a.rows;
#define SG_SHORT(LANES, CH) rmsnorm_short_rows_kernel<LANES, CH><<<(rows - 1) / (256 / LANES) + 1, 256, 0, stream>>>(a)
#define SG_ROW(THREADS, CH) rmsnorm_row_kernel<THREADS, CH><<<rows, THREADS, 0, stream>>>(a)
    if (nchunks <= 4) SG_SHORT(4, 1);
    else if (nchunks <= 16) SG_SHORT(16, 1);
    else if (nchunks <= 64) SG_SHORT(32, 2);
    else if (nchunks <= 128) SG_ROW(64, 2);
    else if (nchunks <= 256) SG_ROW(128, 2);
    else if (nchunks <= 512) SG_ROW(256, 2);
    else if (nchunks <= 1024) SG_ROW(512, 2);
    else if (nchunks <= 2048) SG_ROW(1024, 2);
    else if (nchunks <= 4096) SG_ROW(1024, 4);
    else if (nchunks <= 8192) SG_ROW(1024, 8);
    else rmsnorm_long_rows_kernel<<<rows, 1024, 0, stream>>>(a);
#undef SG_SHORT
#undef SG_ROW
    return report_hip("rmsnorm launch", hipGetLastError()) == hipSuccess ? SG_SUCCESS : SG_LAUNCH_FAILED;
}

}  // namespace sg

using namespace sg;

extern "C" int sg_rmsnorm_fp8_rows(const void* X, const void* residual, const void* weight, void* sum, void* Y, uint8_t* Q, float* scales,
                                   float eps, int rows, int cols, void* stream) {
    if (!X || !Q || !scales || rows <= 0 || cols <= 0 || cols % 16 || !(eps >= 0.0f) || !std::isfinite(eps)) return SG_BAD_ARGUMENT;
    for (const void* p : {X, residual, weight, static_cast<const void*>(sum), static_cast<const void*>(Y), static_cast<const void*>(Q)})
        if (reinterpret_cast<uintptr_t>(p) & 15u) return SG_BAD_ALIGNMENT;
    if (reinterpret_cast<uintptr_t>(scales) & 3u) return SG_BAD_ALIGNMENT;
    DeviceInfo* dev;
    if (int rc = get_device_info(&dev)) return rc;
    auto in = [](const void* p) { return static_cast<const uint8_t*>(p); };
    return launch(NormArgs{in(X), in(residual), in(weight), static_cast<uint8_t*>(sum), static_cast<uint8_t*>(Y), Q, scales, eps, rows, cols},
                  static_cast<hipStream_t>(stream));
}
