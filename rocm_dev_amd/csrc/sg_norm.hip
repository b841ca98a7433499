// Root-mean-square norm of bf16 rows, the residual added first, into E4M3 rows with a scale each (include/sgemm.h).
//
//   v = bf16(X + residual);   y = v * w * rstd,  rstd = 1 / sqrt(sum(v^2) / cols + eps);   s = absmax(y) / 448;   Q = e4m3(y / s)
//
// v * w is a product of two bf16 values, exact in fp32 (above 2^-133, or wherever |w| >= 2^-9), and rstd is one factor of the whole
// row, so absmax(y) is rstd * max|v * w| to the bit: the sum of squares and the maximum come out of the same pass over the row
// and one reduction.  A row is held in registers between the reduction and the codes: it is read from memory once.
// fp32 throughout; roundings to fewer bits are the three outputs' own (v as bf16, since the next layer adds to what is
// stored; the codes; Y).  y / s is one product, v * w with rstd / s: y itself carries the rounding of its sum of squares, so that a correctly rounded
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
    float rstd, s, code;         // code: rstd / s
    bool divide;                 // `code` does not stand for a quotient by s
};
__device__ __forceinline__ RowFactors row_factors(RowSums r, int cols, float eps) {
    RowFactors f;
    const float mean = r.squares / (float)cols + eps;
    // (with an eps as small, few values in a long row have a mean below fp32's normal range, though their squares are not: 2^64 times it)
    f.rstd = mean < 0x1p-100f ? 0x1p32f / sqrtf(r.squares * 0x1p64f / (float)cols + eps * 0x1p64f) : 1.0f / sqrtf(mean);
    float top = r.top * f.rstd;
    if (!(top > 0.0f)) top = 0.0f;                       // also NaN: an infinity times zero, or a row that holds a NaN
    f.s = __fdiv_rn(top, 448.0f);
    if (f.s == 0.0f) f.s = 1.0f;                         // also a top whose 448th part is nearer to zero than to 2^-149
    f.code = f.rstd * __fdiv_rn(1.0f, f.s);
    // code is about 448 / max|v * w|: a large rstd can lift s into the range whose reciprocals are normal while code itself overflows
    f.divide = !(f.s >= 0x1p-120f && f.s <= 0x1p120f && f.code <= 0x1p120f);
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
// codes and Y of eight columns, `at` chunks into the matrix
template <bool DIVIDE>
__device__ __forceinline__ void put_chunk(const NormArgs& a, size_t at, u32x4 v, u32x4 w, const RowFactors& f) {
    float p[8], q[8];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        p[2 * j] = bf16_lo(v[j]) * bf16_lo(w[j]);
        p[2 * j + 1] = bf16_hi(v[j]) * bf16_hi(w[j]);
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
        q[j] = DIVIDE ? __fdiv_rn(p[j] * f.rstd, f.s) : p[j] * f.code;
        // a scale of few steps of 2^-149 may be a third below the 448th part that it stands for
        if (DIVIDE) q[j] = q[j] > 448.0f ? 448.0f : q[j] < -448.0f ? -448.0f : q[j];
    }
    int w0 = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
    w0 = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], w0, true);
    int w1 = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], 0, false);
    w1 = __builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], w1, true);
    __builtin_nontemporal_store(u32x2{canonical_nan_codes(w0), canonical_nan_codes(w1)}, reinterpret_cast<u32x2*>(a.Q) + at);
    if (a.Y) {
        u32x4 o;
#pragma unroll
        for (int j = 0; j < 4; j++) o[j] = pack_bf16x2(p[2 * j] * f.rstd, p[2 * j + 1] * f.rstd);
        __builtin_nontemporal_store(o, reinterpret_cast<u32x4*>(a.Y) + at);
    }
}
__device__ __forceinline__ void put(const NormArgs& a, size_t at, u32x4 v, u32x4 w, const RowFactors& f) {
    if (f.divide) put_chunk<true>(a, at, v, w, f);
    else put_chunk<false>(a, at, v, w, f);
}
constexpr unsigned kOnes = 0x3f803f80u;      // two bf16 ones

// A thread's chunks of a row: t, t + STEP, ...  One past the row's end is the last chunk again, counts nothing and is not stored.
template <int STEP, int CH>
struct RowChunks {
    u32x4 x[CH], r[CH];

    static __device__ __forceinline__ int at(int c, int t, int nchunks) { return c * STEP + t < nchunks ? c * STEP + t : nchunks - 1; }
    __device__ __forceinline__ void load(const NormArgs& a, size_t row, int t, int nchunks) {
        const u32x4* const from = reinterpret_cast<const u32x4*>(a.X) + row * nchunks;
        const u32x4* const res = reinterpret_cast<const u32x4*>(a.residual) + row * nchunks;
#pragma unroll
        for (int c = 0; c < CH; c++) x[c] = __builtin_nontemporal_load(from + at(c, t, nchunks));
        if (a.residual)
#pragma unroll
            for (int c = 0; c < CH; c++) r[c] = __builtin_nontemporal_load(res + at(c, t, nchunks));
    }
    // x becomes v
    __device__ __forceinline__ void add(const NormArgs& a) {
        if (a.residual)
#pragma unroll
            for (int c = 0; c < CH; c++) x[c] = add_bf16(x[c], r[c]);
    }
};
__device__ __forceinline__ u32x4 weight_of(const NormArgs& a, int chunk) {
    return a.weight ? reinterpret_cast<const u32x4*>(a.weight)[chunk] : u32x4{kOnes, kOnes, kOnes, kOnes};
}
template <int STEP, int CH, class Weight>
__device__ __forceinline__ RowSums sums_of(const u32x4 (&v)[CH], int t, int nchunks, Weight&& weight) {
    RowSums sums = {0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < CH; c++)
        if (c * STEP + t < nchunks) see(sums, v[c], weight(c));
    return sums;
}
template <int STEP, int CH, class Weight>
__device__ __forceinline__ void put_row(const NormArgs& a, size_t row, const u32x4 (&v)[CH], int t, int nchunks, const RowFactors& f, Weight&& weight) {
#pragma unroll
    for (int c = 0; c < CH; c++)
        if (c * STEP + t < nchunks) {
            const size_t to = row * nchunks + c * STEP + t;
            if (a.sum) __builtin_nontemporal_store(v[c], reinterpret_cast<u32x4*>(a.sum) + to);
            put(a, to, v[c], weight(c), f);
        }
}

// Packed as they are, two values a register: the compiler would keep what it has unpacked.
template <int CH>
__device__ __forceinline__ void keep_packed(u32x4 (&v)[CH]) {
#pragma unroll
    for (int c = 0; c < CH; c++) asm volatile("" : "+v"(v[c]));
}

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

// A workgroup a row.  KEEP: the weight is asked for with the row and stays in registers; otherwise it is read where it is used, twice, out of
// the caches - later, but off the way of the first round of rows, and with fewer registers.
template <int THREADS, int CH, bool KEEP>
__global__ void __launch_bounds__(THREADS) rmsnorm_row_kernel(const NormArgs a) {
    const int t = threadIdx.x, nchunks = a.cols >> 3;
    RowChunks<THREADS, CH> row;
    u32x4 w[KEEP ? CH : 1];
    auto weight = [&](int c) { return KEEP ? w[KEEP ? c : 0] : weight_of(a, row.at(c, t, nchunks)); };
    row.load(a, blockIdx.x, t, nchunks);
    if (KEEP)
#pragma unroll
        for (int c = 0; c < CH; c++) w[KEEP ? c : 0] = weight_of(a, row.at(c, t, nchunks));
    row.add(a);
    RowSums sums = sums_of<THREADS>(row.x, t, nchunks, weight);
    keep_packed(row.x);
    if (KEEP) keep_packed(w);
    sums = over_threads<THREADS>(sums);
    const RowFactors f = row_factors(sums, a.cols, a.eps);
    if (t == 0) a.scales[blockIdx.x] = f.s;
    put_row<THREADS>(a, blockIdx.x, row.x, t, nchunks, f, weight);
}

// Short rows: LANES lanes of a wave share one.
template <int LANES, int CH>
__global__ void __launch_bounds__(256) rmsnorm_short_rows_kernel(const NormArgs a) {
    const unsigned mine = blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    const unsigned at = mine < (unsigned)a.rows ? mine : (unsigned)a.rows - 1;      // lanes past the last row store nothing
    const int t = (int)threadIdx.x % LANES, nchunks = a.cols >> 3;
    RowChunks<LANES, CH> row;
    u32x4 w[CH];
    auto weight = [&](int c) { return w[c]; };
    row.load(a, at, t, nchunks);
#pragma unroll
    for (int c = 0; c < CH; c++) w[c] = weight_of(a, row.at(c, t, nchunks));
    row.add(a);
    const RowSums sums = over_lanes<LANES>(sums_of<LANES>(row.x, t, nchunks, weight));
    if (mine >= (unsigned)a.rows) return;
    const RowFactors f = row_factors(sums, a.cols, a.eps);
    if (t == 0) a.scales[mine] = f.s;
    put_row<LANES>(a, mine, row.x, t, nchunks, f, weight);
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

template <int THREADS, int CH>
static void launch_row(const NormArgs& a, int cu_count, hipStream_t stream) {
    // Where all rows but a CU's first run at once, the weight is read late: us, late against kept, 1021 x 10944 11.7 - 15.2, 2048 x 4096 with
    // a residual 11.7 - 13.3, 1000 x 16384 20.6 - 23.7; a CU's first rows are waited for, and many rounds read it too often: 1 x 4096
    // 3.3 - 2.8, 256 x 8192 5.5 - 5.1, 8192 x 8192 86.8 - 83.2.
    const bool late = THREADS < 1024 && a.rows > cu_count && a.rows <= cu_count * (2048 / THREADS);
    if (late) rmsnorm_row_kernel<THREADS, CH, false><<<(unsigned)a.rows, THREADS, 0, stream>>>(a);
    else rmsnorm_row_kernel<THREADS, CH, true><<<(unsigned)a.rows, THREADS, 0, stream>>>(a);
}

static int launch(const NormArgs& a, int cu_count, hipStream_t stream) {
    const int nchunks = a.cols >> 3;
    const unsigned rows = (unsigned)a.rows;
    // the smallest group of threads that holds the row in two chunks each, with more rows in four (as the encoder of rows)
#define SG_SHORT(LANES, CH) rmsnorm_short_rows_kernel<LANES, CH><<<(rows - 1) / (256 / LANES) + 1, 256, 0, stream>>>(a)
    if (nchunks <= 4) SG_SHORT(4, 1);
    else if (nchunks <= 16) SG_SHORT(16, 1);
    else if (nchunks <= 64) SG_SHORT(32, 2);
    else if (nchunks <= 128) launch_row<64, 2>(a, cu_count, stream);
    else if (nchunks <= 256) launch_row<128, 2>(a, cu_count, stream);
    else if (nchunks <= 512) launch_row<256, 2>(a, cu_count, stream);
    else if (nchunks <= 1024 && a.rows <= 1024) launch_row<512, 2>(a, cu_count, stream);
    else if (nchunks <= 1024) launch_row<256, 4>(a, cu_count, stream);
    else if (nchunks <= 2048 && a.rows <= 256) launch_row<1024, 2>(a, cu_count, stream);
    else if (nchunks <= 2048) launch_row<512, 4>(a, cu_count, stream);
    else if (nchunks <= 4096) launch_row<1024, 4>(a, cu_count, stream);
    // (kept, the weight's registers would spill: 64 x 65536 19.0, 14.4 this way)
    else if (nchunks <= 8192) rmsnorm_row_kernel<1024, 8, false><<<rows, 1024, 0, stream>>>(a);
    else rmsnorm_long_rows_kernel<<<rows, 1024, 0, stream>>>(a);
#undef SG_SHORT
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
    NormArgs a{in(X), in(residual), in(weight), static_cast<uint8_t*>(sum), static_cast<uint8_t*>(Y), Q, scales, eps, rows, cols};
    constexpr int kMost = 1 << 21;      // a launch has fewer than 2^32 threads, a row up to 1024 of them
    for (int left = rows;; left -= kMost) {
        a.rows = left < kMost ? left : kMost;
        if (int rc = launch(a, dev->cu_count, static_cast<hipStream_t>(stream))) return rc;
        if (left <= kMost) return SG_SUCCESS;
        const size_t values = (size_t)kMost * cols;
        a.X += 2 * values;
        if (a.residual) a.residual += 2 * values;
        if (a.sum) a.sum += 2 * values;
        if (a.Y) a.Y += 2 * values;
        a.Q += values;
        a.scales += kMost;
    }
}
