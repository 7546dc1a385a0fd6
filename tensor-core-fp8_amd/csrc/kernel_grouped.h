// Products of rows grouped by expert for any k, n and pointer alignment: one wave per 32 x 32 tile of C,
// operands straight from global memory into MFMA registers (as kernel_direct.h).  The tiled kernel
// (kernel_ptile.h) takes over wherever rows of A and B are whole 16-byte pieces.
//
// A tile's 32 rows may belong to several groups: every group that has rows in it is multiplied on its own,
// with the other groups' rows read as zeros, and stores only its own rows.  (Adding the groups' products
// into one accumulator would let a NaN in one group's matrix reach another group's rows: 0 * NaN.)
#ifndef FP8GEMM_KERNEL_GROUPED_H
#define FP8GEMM_KERNEL_GROUPED_H

#include "group_table.h"
#include "kernel_direct.h"

template <int AF, int BF>
__global__ __launch_bounds__(64) void gemm_grouped_direct_kernel(int K, int N, const uint8_t *__restrict__ A, const uint8_t *__restrict__ B,
                                                                 void *__restrict__ C, int tiles_n, int vec_ok, GroupSpec grp)
{
    const int lane = threadIdx.x;
    const int i = lane & 31;
    const int g = lane >> 5;
    const int m0 = (int)(blockIdx.x / (unsigned)tiles_n) * 32;
    const int n0 = (int)(blockIdx.x % (unsigned)tiles_n) * 32;
    int begin = group_offset(grp, 0);
    for (int e = 0; e < grp.groups && begin < m0 + 32; ++e) {
        int end = group_offset(grp, e + 1);
        end = end > begin ? end : begin;
        const int first = begin;
        begin = end;
        if (end <= m0 || first == end) continue;                       // (uniform)
        v16f acc;
        for (int r = 0; r < 16; ++r) acc[r] = 0.0f;
        const uint8_t *Be = B + (size_t)e * N * K;
        // (rows in front of the group: a row number at the end of the matrix, which reads as zeros)
        const int arow = m0 + i < first ? end : m0 + i;
        for (int k0 = 0; k0 < K; k0 += 64) {
            const int kk = k0 + g * 32;
            const v8i a = direct_load32(A, arow, end, kk, K, vec_ok != 0);
            const v8i b = direct_load32(Be, n0 + i, N, kk, K, vec_ok != 0);
            acc = mfma_32x32x64<AF, BF>(a, b, acc);
        }
        const int col = n0 + i;
        if (col < N) {
            const float sb = grp.b_scale ? grp.b_scale[grp.b_per_column ? (size_t)e * N + col : (size_t)e] : 1.0f;
            for (int r = 0; r < 16; ++r) {
                const int row = m0 + 8 * (r >> 2) + 4 * g + (r & 3);
                if (row >= first && row < end) store_out(C, (size_t)row * N + col, acc[r] * (grp.a_scale ? grp.a_scale[row] : 1.0f) * sb, grp.type);
            }
        }
    }
}

#endif  // FP8GEMM_KERNEL_GROUPED_H
