// What the kernels for 4-bit weights (kernel_w4.h) are told, and how their launch code is reached.
#ifndef FP8GEMM_W4_ARGS_H
#define FP8GEMM_W4_ARGS_H

#include <hip/hip_runtime.h>
#include <stdint.h>

// how the weights become 16-bit numbers
constexpr int kW4Int = 0;           // 16 + q, corrected by a second MFMA
constexpr int kW4Fp4 = 1;           // e2m1, scales applied to sums
constexpr int kW4Fp4Scaled = 2;     // e2m1, power-of-two scales applied by the conversion (x in bf16, scales in bytes)

struct W4Args {
    const int *offsets;             // null: one group of all rows
    int groups, rows;
    int k, n;
    const void *x;
    int x_type;                     // FP8GEMM_T_*
    const float *x_scale;
    const uint8_t *w;
    const void *w_scale;
    int scale_type;
    const uint8_t *zeros;
    int run;
    void *y;
    int y_type;
    int per_row;                    // scales of a row of W
    // the layout, planned by the launch code
    int wk_shift;                   // 2^wk_shift waves along K (the rest side by side)
    int blocks;                     // blocks of columns a workgroup goes through
    int ring;                       // slots of a wave's ring
    int pass, plan_rows;            // blocks whose scales are staged at once with all of K, for up to plan_rows rows (0: as they fit)
    int part_rows;                  // rows that the partial sums have room for
    int stage_bytes;                // LDS for x and scales
};

namespace fp8gemm_detail {

// validated arguments -> kernel and launch (w4_pair.hip); the layout fields of `p` are filled in there.  With `plan` the
// layout is written there (fp8gemm_w4_plan) and nothing is launched.
template <bool F16, int MODE>
hipError_t launch_w4(const W4Args &p, hipStream_t s, int *plan);

}  // namespace fp8gemm_detail

#endif  // FP8GEMM_W4_ARGS_H
