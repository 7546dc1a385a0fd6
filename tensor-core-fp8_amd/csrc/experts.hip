// C ABI of the operators for layers with experts: products of rows grouped by expert and their weight
// gradient, quantisation of their operands, products with 4-bit weights (include/fp8gemm.h).  Validate,
// pick a kernel, launch asynchronously, return the launch status.
#include "fp8gemm.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "dispatch.h"
#include "kernel_quantize.h"
#include "w4_args.h"

namespace fp8gemm_detail {

extern template hipError_t dispatch_grouped<0, 0>(int, int, int, const uint8_t *, const uint8_t *, void *, int, const GroupSpec &, hipStream_t);
extern template hipError_t dispatch_grouped<0, 1>(int, int, int, const uint8_t *, const uint8_t *, void *, int, const GroupSpec &, hipStream_t);
extern template hipError_t dispatch_grouped<1, 0>(int, int, int, const uint8_t *, const uint8_t *, void *, int, const GroupSpec &, hipStream_t);
extern template hipError_t dispatch_grouped<1, 1>(int, int, int, const uint8_t *, const uint8_t *, void *, int, const GroupSpec &, hipStream_t);
extern template hipError_t dispatch_wgrad<0, 0>(int, int, int, const uint8_t *, const uint8_t *, void *, int, const GroupSpec &, hipStream_t);
extern template hipError_t dispatch_wgrad<0, 1>(int, int, int, const uint8_t *, const uint8_t *, void *, int, const GroupSpec &, hipStream_t);
extern template hipError_t dispatch_wgrad<1, 0>(int, int, int, const uint8_t *, const uint8_t *, void *, int, const GroupSpec &, hipStream_t);
extern template hipError_t dispatch_wgrad<1, 1>(int, int, int, const uint8_t *, const uint8_t *, void *, int, const GroupSpec &, hipStream_t);

// ------------------------------------------------------------------ planning
// Cost model in microseconds, as plan_tile's (fp8gemm.hip): a round of whole tiles is k_tiles * per_k_tile + per_item, a
// round that is not full costs its K tiles times idle + (1 - idle) * (share of its tiles), and no launch is faster than
// its bytes at stream_rate.  Fitted to 120 cuts (1 to 64 experts, 1 to 4096 rows each, k 256 to 8192, n 512 to 8192): the
// pick takes 2 % longer than the best of nine measured shapes on average.  The cut itself is known on the device
// only: an expert is taken to have the average of rows, and half a tile of rows in a tile that is not full.
struct GroupedCost {
    int variant, bm, bn, per_cu;
    bool overhang;                                            // compiled for a K that is not a multiple of 128
    double per_k_tile, per_item, stream_rate, idle;           // us, us, bytes per us
};
constexpr GroupedCost kGroupedCosts[] = {
    {13, 256, 256, 1, true, 1.44, 7.6, 4.65e6, 0.60},
    {14, 192, 256, 1, false, 1.18, 6.2, 4.9e6, 0.64},
    // two workgroups on a CU: 128 x 128 tiles, with the non-temporal hint on B and without; 64 x 128 with it
    {17, 128, 128, 2, false, 1.20, 2.2, 8.4e6, 0.44},
    {18, 128, 128, 2, true, 1.07, 2.25, 5.1e6, 0.30},
    {19, 64, 128, 2, true, 1.06, 1.4, 1e9, 0.23},
    // one workgroup on a CU, a deeper ring: no more tiles than CUs
    {15, 64, 128, 1, false, 0.466, 2.2, 6.2e6, 0.63},
};

int plan_grouped(int m, int k, int n, int groups)
{
    const double kt = (k + 127) / 128;
    const int busy = m < groups ? m : groups;
    const double average = (double)m / busy;
    const double bytes = (double)busy * n * k + (double)m * k + 2.0 * m * n;
    int pick = 18;
    double best = 1e30;
    for (const GroupedCost &c : kGroupedCosts) {
        if (k % 128 != 0 && !c.overhang) continue;
        if ((c.variant == 13 || c.variant == 14) && !p2h_ok(k, 1)) continue;
        const double rows_of_tiles = groups == 1 ? (double)((m + c.bm - 1) / c.bm) : busy * std::max(1.0, average / c.bm + 0.5);
        const double rounds = rows_of_tiles * ((n + c.bn - 1) / c.bn) / (256.0 * c.per_cu);
        const double whole = std::floor(rounds), rest = rounds - whole;
        double cost = whole * (kt * c.per_k_tile + c.per_item);
        if (rest > 1e-9) cost += kt * c.per_k_tile * (c.idle + (1.0 - c.idle) * rest) + c.per_item;
        cost = std::max(cost, bytes / c.stream_rate);
        if (cost < best) {
            best = cost;
            pick = c.variant;
        }
    }
    return pick;
}

// The weight gradient: the same model, with the bytes of C alone (every other one is read for a tile's K walk).  Fitted to 114 cuts
// (1 to 16 experts, 128 to 32768 rows, m and n 256 to 8192): the pick takes 0.6 % longer than the best of the four on
// average.  One tile shape for all: us of 13 / 18 / 19 / 15 for one expert of 16384 rows, 512 x 1024, 139 / 70 / 45 / 41, 4096 x 4096
// 174 / 242 / 332 / 338; for 16 experts of 131 rows, 2048 x 2048, 51 / 46 / 60 / 91.
constexpr GroupedCost kWgradCosts[] = {
    {13, 256, 256, 1, true, 1.327, 9.87, 6.4e7, 0.733},
    {18, 128, 128, 2, true, 0.913, 3.28, 3.39e6, 0.399},
    {19, 64, 128, 2, true, 0.668, 2.45, 2.53e6, 0.394},
    {15, 64, 128, 1, true, 0.337, 2.30, 1e9, 0.780},
};

int plan_wgrad(int rows, int m, int n, int groups)
{
    const double kt = groups == 1 ? (rows + 127) / 128 : (double)rows / groups / 128 + 0.5;
    int pick = 18;
    double best = 1e30;
    for (const GroupedCost &c : kWgradCosts) {
        const double rounds = (double)groups * ((m + c.bm - 1) / c.bm) * ((n + c.bn - 1) / c.bn) / (256.0 * c.per_cu);
        const double whole = std::floor(rounds), rest = rounds - whole, tiles = c.variant == 13 ? std::max(kt, 2.0) : kt;
        double cost = whole * (tiles * c.per_k_tile + c.per_item);
        if (rest > 1e-9) cost += tiles * c.per_k_tile * (c.idle + (1.0 - c.idle) * rest) + c.per_item;
        cost = std::max(cost, 2.0 * groups * m * n / c.stream_rate);
        if (cost < best) {
            best = cost;
            pick = c.variant;
        }
    }
    return pick;
}

}  // namespace fp8gemm_detail

namespace fp8gemm_detail {
extern template hipError_t launch_w4<true, kW4Int>(const W4Args &, hipStream_t, int *);
extern template hipError_t launch_w4<false, kW4Int>(const W4Args &, hipStream_t, int *);
extern template hipError_t launch_w4<true, kW4Fp4>(const W4Args &, hipStream_t, int *);
extern template hipError_t launch_w4<false, kW4Fp4>(const W4Args &, hipStream_t, int *);
extern template hipError_t launch_w4<false, kW4Fp4Scaled>(const W4Args &, hipStream_t, int *);
}  // namespace fp8gemm_detail

using namespace fp8gemm_detail;

namespace {

static_assert(kMaxGroups == FP8GEMM_MAX_GROUPS, "the header names the table's size");

// a number of rows, columns or k: with room for the rounding up that grids and kernels do in ints
bool size_ok(int n) { return n > 0 && n <= (1 << 30); }
bool fmt_ok(int f) { return f == FP8GEMM_E4M3 || f == FP8GEMM_E5M2; }
bool wide_ok(int t) { return t == FP8GEMM_OUT_F32 || t == FP8GEMM_OUT_BF16 || t == FP8GEMM_OUT_F16; }
bool aligned_to(const void *p, unsigned bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
// a place for elements of a wide type
bool wide_aligned(const void *p, int type) { return aligned_to(p, type == FP8GEMM_OUT_F32 ? 4 : 2); }

int grouped(int groups, int m, int k, int n, const int *row_offsets, const void *a, int a_fmt, const void *b, int b_fmt, void *out, int out_type,
            const float *a_scale, const float *b_scale, int b_scale_per_column, int variant, void *stream)
{
    if (groups <= 0 || groups > kMaxGroups || !size_ok(m) || !size_ok(k) || !size_ok(n) || !row_offsets || !a || !b || !out) return (int)hipErrorInvalidValue;
    if (!fmt_ok(a_fmt) || !fmt_ok(b_fmt) || !wide_ok(out_type) || !wide_aligned(out, out_type)) return (int)hipErrorInvalidValue;
    const uint8_t *pa = static_cast<const uint8_t *>(a), *pb = static_cast<const uint8_t *>(b);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const GroupSpec spec = {row_offsets, groups, m, a_scale, b_scale, b_scale_per_column != 0, out_type, 0};
    (void)hipGetLastError();
    if (a_fmt == FP8GEMM_E4M3 && b_fmt == FP8GEMM_E4M3) return (int)dispatch_grouped<0, 0>(m, k, n, pa, pb, out, variant, spec, s);
    if (a_fmt == FP8GEMM_E5M2 && b_fmt == FP8GEMM_E5M2) return (int)dispatch_grouped<1, 1>(m, k, n, pa, pb, out, variant, spec, s);
    if (a_fmt == FP8GEMM_E4M3) return (int)dispatch_grouped<0, 1>(m, k, n, pa, pb, out, variant, spec, s);
    return (int)dispatch_grouped<1, 0>(m, k, n, pa, pb, out, variant, spec, s);
}

int wgrad(int groups, int rows, int m, int n, const int *row_offsets, const void *a_t, int a_fmt, const void *b_t, int b_fmt, int ld, void *out,
          int out_type, const float *a_scale, const float *b_scale, int accumulate, int variant, void *stream)
{
    if (groups <= 0 || groups > kMaxGroups || rows <= 0 || !size_ok(m) || !size_ok(n) || !row_offsets || !a_t || !b_t || !out) return (int)hipErrorInvalidValue;
    if (!fmt_ok(a_fmt) || !fmt_ok(b_fmt) || !wide_ok(out_type) || !wide_aligned(out, out_type)) return (int)hipErrorInvalidValue;
    const int least = fp8gemm_grouped_ld(rows, groups);
    if (least == 0 || ld < least || ld % kTokenRun != 0 || ld > (1 << 23)) return (int)hipErrorInvalidValue;
    if (!aligned_to(a_t, 16) || !aligned_to(b_t, 16)) return (int)hipErrorInvalidValue;
    const uint8_t *pa = static_cast<const uint8_t *>(a_t), *pb = static_cast<const uint8_t *>(b_t);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const GroupSpec spec = {row_offsets, groups, rows, a_scale, b_scale, 1, out_type, accumulate != 0};
    (void)hipGetLastError();
    if (a_fmt == FP8GEMM_E4M3 && b_fmt == FP8GEMM_E4M3) return (int)dispatch_wgrad<0, 0>(m, ld, n, pa, pb, out, variant, spec, s);
    if (a_fmt == FP8GEMM_E5M2 && b_fmt == FP8GEMM_E5M2) return (int)dispatch_wgrad<1, 1>(m, ld, n, pa, pb, out, variant, spec, s);
    if (a_fmt == FP8GEMM_E4M3) return (int)dispatch_wgrad<0, 1>(m, ld, n, pa, pb, out, variant, spec, s);
    return (int)dispatch_wgrad<1, 0>(m, ld, n, pa, pb, out, variant, spec, s);
}

// ------------------------------------------------------------------ quantisation
constexpr int kRowsAtOnce = 1 << 23;                       // rows of one launch: 2^32 threads are too many for a grid

template <int TYPE, int FMT>
hipError_t launch_quantize_rows(int rows, int cols, const void *x, size_t stride, int x_rows, const int *index, uint8_t *codes, float *scales, hipStream_t s)
{
    const size_t elem = TYPE == FP8GEMM_OUT_F32 ? 4 : 2;
    for (; rows > 0; rows -= kRowsAtOnce) {
        const int now = std::min(rows, kRowsAtOnce);
#define ROWS_KERNEL(WAVES, HELD)                                                                                                            \
    hipLaunchKernelGGL((quantize_rows_kernel<TYPE, FMT, WAVES, HELD>), dim3((unsigned)((now + 4 / WAVES - 1) / (4 / WAVES))), dim3(256), 0, s, \
                       now, cols, x, stride, x_rows, index, codes, scales)
        // Four waves to a row, two or eight pieces of eight elements a lane; short rows get a wave each, for which four would be
        // half idle.  One wave with eight pieces for rows of up to 4096 is slower: 32768 rows of 4096 74.4 us against 68.0 (calls
        // one behind the other on three matrices), 3001 rows of 2048 8.0 against 7.7; but rows that are not whole pieces 16.2
        // against 18.0 (8192 of 1843).
        if (cols <= 1024)
            ROWS_KERNEL(1, 2);
        else if (cols <= 4096)
            ROWS_KERNEL(4, 2);
        else if (cols <= 16384)
            ROWS_KERNEL(4, 8);
        else
            hipLaunchKernelGGL((quantize_rows_any_kernel<TYPE, FMT>), dim3((unsigned)now), dim3(256), 0, s, cols, x, stride, x_rows, index, codes, scales);
#undef ROWS_KERNEL
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        if (index)
            index += now;
        else {
            x = static_cast<const char *>(x) + (size_t)now * stride * elem;
            x_rows -= now;
        }
        codes += (size_t)now * cols;
        scales += now;
    }
    return hipSuccess;
}

template <int TYPE, int FMT>
hipError_t launch_quantize_columns(const GroupSpec &grp, int cols, const void *x, size_t stride, int x_rows, const int *index, uint8_t *codes, size_t ld,
                                   float *scales, hipStream_t s)
{
    const long col_blocks = (cols + kColBlock - 1) / kColBlock;
#define COLUMNS_KERNEL(PART, WORKGROUPS)                                                                                                             \
    hipLaunchKernelGGL((quantize_columns_kernel<TYPE, FMT, PART>), dim3((unsigned)(WORKGROUPS)), dim3(kColThreads), 0, s, grp, cols, x, stride, x_rows, index, \
                       codes, ld, scales)
    const int busy = std::min(grp.rows, grp.groups);
    const long batches = grp.rows / col_rows(TYPE) + grp.groups;          // as many as any cut of the rows has
    if (col_blocks * std::max(batches, (long)grp.groups) > 0xFFFFFFFFL / kColThreads - col_blocks) return hipErrorInvalidValue;
    // Split over the rows where the whole walks leave CUs idle and take several batches (bf16, us split / whole: one expert of 16384
    // rows, 512 columns 22 / 144, 2000 rows 17.7 / 21.2; 3 of 2667, 2048 columns 29 / 48; but one of 1500, 4096 columns 20.6 / 18.6, 16 of
    // 512, 2048 columns 31 / 23, 32 of 1024, 4096 columns 186 / 120).
    if (col_blocks * busy < 256 && grp.rows / busy > 3 * col_rows(TYPE)) {
        const size_t count = (size_t)grp.groups * cols;
        hipLaunchKernelGGL(quantize_clear_kernel, dim3((unsigned)((count + 255) / 256)), dim3(256), 0, s, scales, count);
        COLUMNS_KERNEL(kColMaxima, col_blocks * batches);
        COLUMNS_KERNEL(kColCodes, col_blocks * (batches + 1));
    } else {
        COLUMNS_KERNEL(kColWhole, col_blocks * (grp.groups + 1));
    }
#undef COLUMNS_KERNEL
    return hipGetLastError();
}

bool quantize_source_ok(int rows, int cols, const void *x, int x_type, long long x_stride, int x_rows, const int *row_index, int fmt)
{
    if (!size_ok(rows) || !size_ok(cols) || x_rows <= 0 || !x || !wide_ok(x_type) || !fmt_ok(fmt) || x_stride < cols) return false;
    return (row_index || rows <= x_rows) && wide_aligned(x, x_type);
}

// ------------------------------------------------------------------ 4-bit weights
int gemv_w4(int groups, int m, int k, int n, const int *row_offsets, const void *x, int x_type, const float *x_scale, const void *w, int w_fmt, int run,
            const void *w_scales, int scale_type, const void *w_zeros, void *y, int y_type, void *stream, int *plan = nullptr)
{
    if (groups <= 0 || groups > kMaxGroups || !size_ok(m) || !size_ok(k) || !size_ok(n) || run <= 0 || !x || !w || !w_scales || !y) return (int)hipErrorInvalidValue;
    if (run % 32 != 0 || k % run != 0 || k > (1 << 23)) return (int)hipErrorInvalidValue;
    if (w_fmt != FP8GEMM_W4_INT && w_fmt != FP8GEMM_W4_E2M1) return (int)hipErrorInvalidValue;
    if (w_zeros && w_fmt != FP8GEMM_W4_INT) return (int)hipErrorInvalidValue;
    if (x_type != FP8GEMM_T_BF16 && x_type != FP8GEMM_T_F16 && x_type != FP8GEMM_T_E4M3 && x_type != FP8GEMM_T_E5M2) return (int)hipErrorInvalidValue;
    if (!wide_ok(scale_type) && scale_type != FP8GEMM_T_E8M0) return (int)hipErrorInvalidValue;
    if (!wide_ok(y_type) || !wide_aligned(y, y_type) || !aligned_to(x, 16) || !aligned_to(w, 16)) return (int)hipErrorInvalidValue;
    if (wide_ok(scale_type) && !wide_aligned(w_scales, scale_type)) return (int)hipErrorInvalidValue;
    const W4Args p = {row_offsets, groups, m, k, n, x, x_type, x_scale, static_cast<const uint8_t *>(w), w_scales, scale_type,
                      static_cast<const uint8_t *>(w_zeros), run, y, y_type, k / run, 0, 1, 0, 0, 0, 1, 0};
    hipStream_t s = static_cast<hipStream_t>(stream);
    (void)hipGetLastError();
    const bool f16 = x_type != FP8GEMM_T_BF16;
    hipError_t e;
    if (w_fmt == FP8GEMM_W4_INT)
        e = f16 ? launch_w4<true, kW4Int>(p, s, plan) : launch_w4<false, kW4Int>(p, s, plan);
    else if (f16)
        e = launch_w4<true, kW4Fp4>(p, s, plan);
    else
        e = scale_type == FP8GEMM_T_E8M0 ? launch_w4<false, kW4Fp4Scaled>(p, s, plan) : launch_w4<false, kW4Fp4>(p, s, plan);
    return (int)e;
}

}  // namespace

extern "C" {

int fp8gemm_grouped(int groups, int m, int k, int n, const int *row_offsets, const void *a, int a_fmt, const void *b, int b_fmt, void *out,
                    int out_type, const float *a_scale, const float *b_scale, int b_scale_per_column, void *stream)
{
    return grouped(groups, m, k, n, row_offsets, a, a_fmt, b, b_fmt, out, out_type, a_scale, b_scale, b_scale_per_column, -1, stream);
}

int fp8gemm_grouped_tuned(int groups, int m, int k, int n, const int *row_offsets, const void *a, int a_fmt, const void *b, int b_fmt, void *out,
                          int out_type, const float *a_scale, const float *b_scale, int b_scale_per_column, int variant, void *stream)
{
    return grouped(groups, m, k, n, row_offsets, a, a_fmt, b, b_fmt, out, out_type, a_scale, b_scale, b_scale_per_column, variant, stream);
}

int fp8gemm_grouped_ld(int rows, int groups)
{
    if (rows <= 0 || groups <= 0 || groups > kMaxGroups) return 0;
    const long long ld = ((long long)rows + (long long)(kTokenRun - 1) * groups) / kTokenRun * kTokenRun;
    return ld > (1 << 23) ? 0 : (int)ld;
}

int fp8gemm_grouped_wgrad(int groups, int rows, int m, int n, const int *row_offsets, const void *a_t, int a_fmt, const void *b_t, int b_fmt,
                          int ld, void *out, int out_type, const float *a_scale, const float *b_scale, int accumulate, void *stream)
{
    return wgrad(groups, rows, m, n, row_offsets, a_t, a_fmt, b_t, b_fmt, ld, out, out_type, a_scale, b_scale, accumulate, -1, stream);
}

int fp8gemm_grouped_wgrad_tuned(int groups, int rows, int m, int n, const int *row_offsets, const void *a_t, int a_fmt, const void *b_t,
                                int b_fmt, int ld, void *out, int out_type, const float *a_scale, const float *b_scale, int accumulate,
                                int variant, void *stream)
{
    return wgrad(groups, rows, m, n, row_offsets, a_t, a_fmt, b_t, b_fmt, ld, out, out_type, a_scale, b_scale, accumulate, variant, stream);
}

int fp8gemm_quantize_rows(int rows, int cols, const void *x, int x_type, long long x_stride, int x_rows, const int *row_index, int fmt,
                          void *codes, float *scales, void *stream)
{
    if (!codes || !scales || !quantize_source_ok(rows, cols, x, x_type, x_stride, x_rows, row_index, fmt)) return (int)hipErrorInvalidValue;
    uint8_t *pc = static_cast<uint8_t *>(codes);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const size_t stride = (size_t)x_stride;
    (void)hipGetLastError();
#define QUANT(TYPE)                                                                                                       \
    (fmt == FP8GEMM_E4M3 ? launch_quantize_rows<TYPE, 0>(rows, cols, x, stride, x_rows, row_index, pc, scales, s)         \
                         : launch_quantize_rows<TYPE, 1>(rows, cols, x, stride, x_rows, row_index, pc, scales, s))
    if (x_type == FP8GEMM_OUT_F32) return (int)QUANT(FP8GEMM_OUT_F32);
    if (x_type == FP8GEMM_OUT_BF16) return (int)QUANT(FP8GEMM_OUT_BF16);
    return (int)QUANT(FP8GEMM_OUT_F16);
#undef QUANT
}

int fp8gemm_quantize_columns(int groups, int rows, int cols, const int *row_offsets, const void *x, int x_type, long long x_stride, int x_rows,
                             const int *row_index, int fmt, void *codes_t, int ld, float *scales, void *stream)
{
    if (!codes_t || !scales || !row_offsets || !quantize_source_ok(rows, cols, x, x_type, x_stride, x_rows, row_index, fmt)) return (int)hipErrorInvalidValue;
    const int least = fp8gemm_grouped_ld(rows, groups);
    if (least == 0 || ld < least || ld % kTokenRun != 0 || ld > (1 << 23) || !aligned_to(codes_t, 16)) return (int)hipErrorInvalidValue;
    uint8_t *pc = static_cast<uint8_t *>(codes_t);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const size_t stride = (size_t)x_stride;
    const GroupSpec spec = {row_offsets, groups, rows, nullptr, nullptr, 0, 0, 0};
    (void)hipGetLastError();
#define QUANT(TYPE)                                                                                                         \
    (fmt == FP8GEMM_E4M3 ? launch_quantize_columns<TYPE, 0>(spec, cols, x, stride, x_rows, row_index, pc, ld, scales, s)    \
                         : launch_quantize_columns<TYPE, 1>(spec, cols, x, stride, x_rows, row_index, pc, ld, scales, s))
    if (x_type == FP8GEMM_OUT_F32) return (int)QUANT(FP8GEMM_OUT_F32);
    if (x_type == FP8GEMM_OUT_BF16) return (int)QUANT(FP8GEMM_OUT_BF16);
    return (int)QUANT(FP8GEMM_OUT_F16);
#undef QUANT
}

int fp8gemm_gemv_w4(int m, int k, int n, const void *x, int x_type, const float *x_scale, const void *w, int w_fmt, int run, const void *w_scales,
                    int scale_type, const void *w_zeros, void *y, int y_type, void *stream)
{
    return gemv_w4(1, m, k, n, nullptr, x, x_type, x_scale, w, w_fmt, run, w_scales, scale_type, w_zeros, y, y_type, stream);
}

int fp8gemm_grouped_w4(int groups, int m, int k, int n, const int *row_offsets, const void *x, int x_type, const float *x_scale, const void *w,
                       int w_fmt, int run, const void *w_scales, int scale_type, const void *w_zeros, void *y, int y_type, void *stream)
{
    if (!row_offsets) return (int)hipErrorInvalidValue;
    return gemv_w4(groups, m, k, n, row_offsets, x, x_type, x_scale, w, w_fmt, run, w_scales, scale_type, w_zeros, y, y_type, stream);
}

int fp8gemm_w4_plan(int groups, int m, int k, int n, int x_type, int w_fmt, int run, int scale_type, int plan[7])
{
    if (!plan) return (int)hipErrorInvalidValue;
    alignas(16) char some[16];                             // (stands for every operand: nothing is read)
    return gemv_w4(groups, m, k, n, nullptr, some, x_type, nullptr, some, w_fmt, run, some, scale_type, nullptr, some, FP8GEMM_OUT_F32, nullptr, plan);
}

}  // extern "C"
