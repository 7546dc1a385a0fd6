// Products with 4-bit weights, launch code of one pair of 16-bit type and way of expanding the weights.  Compiled five
// times, with -DFP8GEMM_W4_F16=<0|1> (x and the expanded weights in bf16 or f16) -DFP8GEMM_W4_MODE=<kW4...> (w4_args.h).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "dispatch.h"
#include "kernel_w4.h"

#if !defined(FP8GEMM_W4_F16) || !defined(FP8GEMM_W4_MODE)
#error "compile with -DFP8GEMM_W4_F16=<0|1> -DFP8GEMM_W4_MODE=<0|1|2>"
#endif

namespace fp8gemm_detail {

template <bool F16, int MODE, int RUN, int KIND>
struct W4KernelTag {};

constexpr int kW4MaxLds = 160 * 1024;

template <bool F16, int MODE, int RUN, int KIND>
hipError_t launch_w4_kernel(W4Args p, hipStream_t s, int *plan)
{
    // Rows of x that an expert has at a time, as far as the host can tell.
    const int busy = std::min(p.rows, p.groups);
    const int rows = std::min((p.rows + busy - 1) / busy, 16);
    const long col_tiles = (p.n + 15) / 16, row_bytes = p.k / 2;
    // How the eight waves are laid out, how many workgroups share a CU and how many blocks of columns each takes: the
    // least time in units of one ring stage of a workgroup -- one unit to add the waves along K up, one to start a pass, more to
    // stage the rows of x or where not all of x fits, and two workgroups on a CU hide 28 % of each other's time.  The experts that
    // will have rows are counted as if every row fell on any of them.  Fitted to 140 calls (integers in runs of 32 and 128, e2m1, 1 to
    // 14 rows of one matrix, 8 to 40 of 8 and 32 experts): the pick takes 0.7 % longer than the best of the eight layouts on
    // average, 12 % at worst.  Not among them, and slower than by the fit to fewer calls before it: 2 rows of 8192 x 28672 in runs of
    // 128 35.0 us (31.0), 8 rows of 28672 x 8192 35.9 (34.8); faster: 1 row of 28672 x 8192 in runs of 32 36.8 (43.6), 4 rows in runs
    // of 128 30.9 (33.9).
    constexpr int EB = w4_entry_bytes(MODE, KIND);
    const double active = p.groups > 1 ? p.groups * (1.0 - std::pow(1.0 - 1.0 / p.groups, p.rows)) : 1.0;
    double best = 1e30;
    int best_lds = 0;
    p.part_rows = std::min(p.rows, 16);
    for (int per_cu = 2; per_cu >= 1; --per_cu)
        for (int wk = 1; wk <= kW4Waves; wk *= 2) {
            if (wk > 1 && p.k <= (wk - 1) * kW4StageK) continue;
            const int wc = kW4Waves / wk, unit = kW4StageK * wk, slot = w4_ring_bytes(1);
            const long blocks = (col_tiles + wc - 1) / wc, whole = ((long)p.k + unit - 1) / unit * unit;
            long each = std::min(blocks, (blocks * busy + 256 * per_cu - 1) / (256 * per_cu));
            each = std::max(1L, std::min(each, ((1L << 31) - 1) / (16 * wc * row_bytes)));
            const long x_bytes = rows * (whole * 2 + 16), block_bytes = (long)16 * wc * (((whole / RUN) * EB + 15) / 16 + 1) * 16;
            const long fixed = w4_ring_bytes(kW4RingTwo) + w4_part_bytes(wk, p.part_rows);
            const long room = kW4MaxLds / per_cu - fixed;
            const long least = p.part_rows * w4_x_pitch(unit) + (long)16 * wc * (unit / RUN * EB + 31);
            if (room < least) continue;
            const bool fits = x_bytes + block_bytes <= room;
            // (K in pieces: a pass for every block and piece)
            const long at_once = fits ? std::min(each, (room - x_bytes) / block_bytes) : 1;
            const double passes = fits ? (double)((each + at_once - 1) / at_once) : (double)each * (x_bytes + block_bytes) / room;
            const double stages = (double)((p.k + unit - 1) / unit), staging = (fits ? 1.0 : (double)each) * rows * whole / 12500.0;
            const double on_a_cu = std::ceil((double)((blocks + each - 1) / each) * active / 256.0);
            const double cost = on_a_cu * (each * (stages + (wk > 1 ? 1.15 : 0.0)) + staging) * (on_a_cu > 1.0 && per_cu > 1 ? 0.72 : 1.0) +
                                std::max(1.0, on_a_cu / per_cu) * passes * 1.25 + (fits ? 0.0 : 1.7);
            if (cost < best) {
                best = cost;
                p.wk_shift = wk == 1 ? 0 : (wk == 2 ? 1 : (wk == 4 ? 2 : 3));
                p.pass = fits ? (int)at_once : 0;
                p.plan_rows = rows;
                p.blocks = (int)each;
                // (an expert may have more rows than the average: x gets the room that the CU has)
                p.stage_bytes = (int)(p.groups > 1 || !fits ? room : std::max(least, x_bytes + at_once * block_bytes));
                p.ring = room - p.stage_bytes >= (kW4RingFour - kW4RingTwo) * slot ? kW4RingFour : kW4RingTwo;
                best_lds = (int)fixed + (p.ring - kW4RingTwo) * slot + p.stage_bytes;
            }
        }
    if (best_lds == 0) return hipErrorInvalidValue;
    const int lds = best_lds, wc = kW4Waves >> p.wk_shift;
    if (plan) {
        const int layout[7] = {16, 1 << p.wk_shift, 16 * wc, p.blocks, p.pass, p.plan_rows, p.ring};
        std::copy(layout, layout + 7, plan);
        return hipSuccess;
    }
    auto kernel = gemv_w4_kernel<F16, MODE, RUN, KIND>;
    hipError_t e = allow_lds<W4KernelTag<F16, MODE, RUN, KIND>>(kernel, kW4MaxLds);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(kernel, dim3((unsigned)((col_tiles + wc * p.blocks - 1) / (wc * p.blocks)), (unsigned)p.groups), dim3(64 * kW4Waves), lds, s, p);
    return hipGetLastError();
}

template <bool F16, int MODE, int RUN, int MT, int KIND, int WK, int TN, bool CODES>
struct W4WideKernelTag {};

template <bool F16, int MODE, int RUN, int MT, int KIND, int WK, int TN, bool CODES>
hipError_t launch_w4_wide(const W4Args &p, hipStream_t s, int *plan)
{
    constexpr int COLS = w4_wide_cols(WK, TN), PIECE = w4_piece(WK), EB = w4_entry_bytes(MODE, KIND), ROOM = kW4MaxLds - w4_wide_x_bytes(MT, WK);
    // the scales of all of K, or of equal parts, whole turns of the weights' registers
    const int pieces = (p.k + PIECE - 1) / PIECE;
    auto bytes = [](int pieces_) { return COLS * w4_scale_pitch(pieces_ * (PIECE / RUN), EB); };
    static_assert(COLS * w4_scale_pitch(kW4Ahead * (PIECE / RUN), EB) <= ROOM, "no room for the scales");
    int parts = 1, scale_pieces;
    do {
        scale_pieces = ((pieces + parts - 1) / parts + kW4Ahead - 1) / kW4Ahead * kW4Ahead;
        ++parts;
    } while (bytes(scale_pieces) > ROOM);
    if (plan) {
        const int layout[7] = {16 * MT, WK, COLS, 1, scale_pieces * PIECE, 0, 0};
        std::copy(layout, layout + 7, plan);
        return hipSuccess;
    }
    auto kernel = gemm_w4_wide_kernel<F16, MODE, RUN, MT, KIND, WK, TN, CODES>;
    hipError_t e = allow_lds<W4WideKernelTag<F16, MODE, RUN, MT, KIND, WK, TN, CODES>>(kernel, kW4MaxLds);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(kernel, dim3((unsigned)((p.n + COLS - 1) / COLS), (unsigned)p.groups), dim3(64 * kW4Waves), w4_wide_x_bytes(MT, WK) + bytes(scale_pieces), s, p, scale_pieces);
    return hipGetLastError();
}

template <bool F16, int MODE, int RUN, int MT, int KIND>
hipError_t launch_w4_tall(const W4Args &p, int busy, hipStream_t s, int *plan)
{
    // Workgroups of 128 columns (two blocks of 16 a wave) where they still keep half the CUs busy (us for 64 / 128 columns: 64 x 4096 x
    // 16384 22.3 / 28.2, 32 x 4096 x 4096 15.2 / 21.8, 48 x 2048 x 24576 33.3 / 29.1, 17 x 8192 x 28672 49.0 / 40.7); else of 64; of 32
    // with twice the waves along K where 64 keep less than half busy and K has several turns of its pieces (64 / 32: 20 x 4096 x
    // 4096 14.8 / 11.5, 64 x 8192 x 2048 43 / 31, 30 x 2048 x 6000 10.7 / 9.6, but 40 x 1024 x 1024 9.6 / 11.2).
    const long columns = (long)busy * p.n;
    auto launch = [&](auto codes) {
        constexpr bool CODES = decltype(codes)::value;
        if (columns > 128 * 128) return launch_w4_wide<F16, MODE, RUN, MT, KIND, 2, 2, CODES>(p, s, plan);
        if (columns > 128 * 64 || p.k <= 1024) return launch_w4_wide<F16, MODE, RUN, MT, KIND, 2, 1, CODES>(p, s, plan);
        return launch_w4_wide<F16, MODE, RUN, MT, KIND, 4, 1, CODES>(p, s, plan);
    };
    if constexpr (F16)
        if (p.x_type != FP8GEMM_T_F16) return launch(std::true_type{});
    return launch(std::false_type{});
}

template <bool F16, int MODE, int RUN, int KIND>
hipError_t launch_w4_rows(const W4Args &p, hipStream_t s, int *plan)
{
    // Rows of x per pass over the weights; with experts, what an expert has on average (eight experts, us for gemv / 32 rows at a
    // time: 4096 x 4096 integers, 8 rows each 23.2 / 25.2, 12 rows 30.6 / 25.1; 2048 x 2048 e2m1, 8 rows 16.2 / 9.9).  The host knows no more than the average: 192 rows to 32
    // experts of 4096 x 4096 take 54 us in even parts and 390 all to one, whose weights are read for every 16 of them.
    const int busy = std::min(p.rows, p.groups), average = (p.rows + busy - 1) / busy;
    if (p.rows <= 16 || average <= 6) return launch_w4_kernel<F16, MODE, RUN, KIND>(p, s, plan);
    return p.rows <= 32 || average <= 16 ? launch_w4_tall<F16, MODE, RUN, 2, KIND>(p, busy, s, plan) : launch_w4_tall<F16, MODE, RUN, 4, KIND>(p, busy, s, plan);
}

template <bool F16, int MODE>
hipError_t launch_w4(const W4Args &p, hipStream_t s, int *plan)
{
    const bool long_runs = p.run % 128 == 0;
    if constexpr (MODE == kW4Fp4Scaled) {
        return long_runs ? launch_w4_rows<F16, MODE, 128, kW4ScaleByte>(p, s, plan) : launch_w4_rows<F16, MODE, 32, kW4ScaleByte>(p, s, plan);
    } else {
        if (p.scale_type == FP8GEMM_T_F32) return long_runs ? launch_w4_rows<F16, MODE, 128, kW4ScaleF32>(p, s, plan) : launch_w4_rows<F16, MODE, 32, kW4ScaleF32>(p, s, plan);
        if (p.scale_type == FP8GEMM_T_F16) return long_runs ? launch_w4_rows<F16, MODE, 128, kW4ScaleF16>(p, s, plan) : launch_w4_rows<F16, MODE, 32, kW4ScaleF16>(p, s, plan);
        return long_runs ? launch_w4_rows<F16, MODE, 128, kW4ScaleBf16>(p, s, plan) : launch_w4_rows<F16, MODE, 32, kW4ScaleBf16>(p, s, plan);
    }
}

template hipError_t launch_w4<FP8GEMM_W4_F16 != 0, FP8GEMM_W4_MODE>(const W4Args &, hipStream_t, int *);

}  // namespace fp8gemm_detail
