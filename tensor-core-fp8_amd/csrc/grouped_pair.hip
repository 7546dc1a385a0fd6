// Products grouped by expert, launch code of one operand pairing.  Compiled four times, with
// -DFP8GEMM_PAIR_A=<0|1> -DFP8GEMM_PAIR_B=<0|1> (0 = E4M3, 1 = E5M2).
#include "dispatch.h"
#include "kernel_grouped.h"

#if !defined(FP8GEMM_PAIR_A) || !defined(FP8GEMM_PAIR_B)
#error "compile with -DFP8GEMM_PAIR_A=<0|1> -DFP8GEMM_PAIR_B=<0|1>"
#endif

namespace fp8gemm_detail {

// two workgroups on a CU (their epilogues and first loads overlap the other's K loop): a 3 x 24 KiB ring of the
// 64 x 128 tile; the quarter tile's 2 x 32 KiB ring fits as it is
using TileE3 = TileShape<64, 128, 128, 1, 4, 3, 3>;

template <class S, int AF, int BF, bool KOVER, bool BSTREAM, bool NOPF, int GROUPED, int PER_CU>
struct PtileGroupedKernelTag {};

template <class S, int AF, int BF, bool KOVER, bool BSTREAM, bool NOPF, int GROUPED, int PER_CU>
static hipError_t launch_grouped_shape(int m, int k, int n, const uint8_t *a, const uint8_t *b, void *out, int rotate, const GroupSpec &grp, hipStream_t stream)
{
    constexpr int kFixedLds = S::PTILE_LDS_BYTES + kGroupTableOffset + 2 * (S::BM + S::BN) * 4;
    static_assert(kFixedLds + kGroupTableBytes <= S::LDS_MAX, "the group table does not fit behind the ring");
    static_assert((kFixedLds + 2 * 257 * 4) * PER_CU <= S::LDS_MAX, "two workgroups of up to 256 groups do not fit a CU");
    const int tiles_m = (m + S::BM - 1) / S::BM, tiles_n = (n + S::BN - 1) / S::BN;
    // tile numbers are ints (the rows of every group may leave a tile of their own)
    const long tiles = GROUPED == kGroupedRows ? ((long)tiles_m + grp.groups) * tiles_n : (long)tiles_m * tiles_n * grp.groups;
    if (tiles > (1L << 30)) return hipErrorInvalidValue;
    const int lds = kFixedLds + 2 * (grp.groups + 1) * 4;
    auto kernel = gemm_ptile_grouped_kernel<S, AF, BF, KOVER, BSTREAM, NOPF, GROUPED, PER_CU>;
    hipError_t e = allow_lds<PtileGroupedKernelTag<S, AF, BF, KOVER, BSTREAM, NOPF, GROUPED, PER_CU>>(kernel, kFixedLds + kGroupTableBytes);
    if (e != hipSuccess) return e;
    const unsigned grid = tiles < 256 * PER_CU ? (unsigned)((tiles + 7) / 8 * 8) : 256u * PER_CU;
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(S::THREADS), lds, stream, m, k, n, a, b, out, tiles_m, tiles_n, rotate, grp);
    return hipGetLastError();
}

// OVERHANG_TOO: this shape is also compiled for a K that is not a multiple of its K tile.
template <class S, int AF, int BF, bool BSTREAM, bool NOPF, int PER_CU, bool OVERHANG_TOO>
static hipError_t launch_grouped_rows(int m, int k, int n, const uint8_t *a, const uint8_t *b, void *out, const GroupSpec &grp, hipStream_t stream)
{
    // (a K walk of its own for every tile column where the rows of A are few, for every XCD and round otherwise)
    const int rotate = (size_t)m * k <= ((size_t)2 << 20) ? 1 : 2;
    if (k % 128 == 0) return launch_grouped_shape<S, AF, BF, false, BSTREAM, NOPF, kGroupedRows, PER_CU>(m, k, n, a, b, out, rotate, grp, stream);
    if constexpr (OVERHANG_TOO) return launch_grouped_shape<S, AF, BF, true, BSTREAM, NOPF, kGroupedRows, PER_CU>(m, k, n, a, b, out, rotate, grp, stream);
    return hipErrorInvalidValue;
}

template <int AF, int BF>
hipError_t dispatch_grouped(int m, int k, int n, const uint8_t *a, const uint8_t *b, void *out, int variant, const GroupSpec &grp, hipStream_t stream)
{
    const bool aligned = k % 16 == 0 && k <= (1 << 23) && ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) % 16) == 0;
    if (variant < 0) variant = aligned ? plan_grouped(m, k, n, grp.groups) : kGroupedDirect;
    if (variant != kGroupedDirect && !aligned) return hipErrorInvalidValue;
    switch (variant) {
    case kGroupedDirect: {
        const long tiles_m = (m + 31) / 32, tiles_n = (n + 31) / 32;
        if (tiles_m * tiles_n > 0xFFFFFFFFL / 64) return hipErrorInvalidValue;          // (a grid holds fewer than 2^32 threads)
        hipLaunchKernelGGL((gemm_grouped_direct_kernel<AF, BF>), dim3((unsigned)(tiles_m * tiles_n)), dim3(64), 0, stream, k, n, a, b, out, (int)tiles_n,
                           aligned ? 1 : 0, grp);
        return hipGetLastError();
    }
    case 13:
        if (!p2h_ok(k, 1)) return hipErrorInvalidValue;
        return launch_grouped_rows<TileP2h, AF, BF, false, false, 1, true>(m, k, n, a, b, out, grp, stream);
    case 14:
        if (!p2h_ok(k, 1)) return hipErrorInvalidValue;
        return launch_grouped_rows<TileT2h, AF, BF, false, false, 1, false>(m, k, n, a, b, out, grp, stream);
    case 15: return launch_grouped_rows<TileE5, AF, BF, true, true, 1, false>(m, k, n, a, b, out, grp, stream);
    case 17: return launch_grouped_rows<TileQ2, AF, BF, true, true, 2, false>(m, k, n, a, b, out, grp, stream);
    case 18: return launch_grouped_rows<TileQ2, AF, BF, false, false, 2, true>(m, k, n, a, b, out, grp, stream);
    case 19: return launch_grouped_rows<TileE3, AF, BF, true, true, 2, true>(m, k, n, a, b, out, grp, stream);
    default: return hipErrorInvalidValue;
    }
}

template <int AF, int BF>
hipError_t dispatch_wgrad(int m, int ld, int n, const uint8_t *a_t, const uint8_t *b_t, void *out, int variant, const GroupSpec &grp, hipStream_t stream)
{
    if (variant < 0) variant = plan_wgrad(grp.rows, m, n, grp.groups);
    switch (variant) {
    case 13: return launch_grouped_shape<TileP2h, AF, BF, false, false, false, kGroupedK, 1>(m, ld, n, a_t, b_t, out, 2, grp, stream);
    case 18: return launch_grouped_shape<TileQ2, AF, BF, false, false, false, kGroupedK, 2>(m, ld, n, a_t, b_t, out, 2, grp, stream);
    case 19: return launch_grouped_shape<TileE3, AF, BF, false, false, false, kGroupedK, 2>(m, ld, n, a_t, b_t, out, 2, grp, stream);
    case 15: return launch_grouped_shape<TileE5, AF, BF, false, false, true, kGroupedK, 1>(m, ld, n, a_t, b_t, out, 2, grp, stream);
    default: return hipErrorInvalidValue;
    }
}

template hipError_t dispatch_grouped<FP8GEMM_PAIR_A, FP8GEMM_PAIR_B>(int, int, int, const uint8_t *, const uint8_t *, void *, int, const GroupSpec &, hipStream_t);
template hipError_t dispatch_wgrad<FP8GEMM_PAIR_A, FP8GEMM_PAIR_B>(int, int, int, const uint8_t *, const uint8_t *, void *, int, const GroupSpec &, hipStream_t);

}  // namespace fp8gemm_detail
