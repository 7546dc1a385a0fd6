// Rows grouped by expert: what the grouped kernels are told, and the table that turns a tile number
// into a group, built by every workgroup from the row offsets (which live on the device: the host
// lays out no work list and never waits for them).
//
// Group g owns rows [offsets[g], offsets[g + 1]) of a matrix of `rows` rows.  Every offset is clamped to
// [0, rows] and raised to the largest one before it, so that no content of the array can send a kernel
// outside its operands: what the table describes is always a cut of at most `rows` rows.
#ifndef FP8GEMM_GROUP_TABLE_H
#define FP8GEMM_GROUP_TABLE_H

#include "device_common.h"

constexpr int kNotGrouped = 0;
constexpr int kGroupedRows = 1;      // C[rows of g] = A[rows of g] * B[g]^T
constexpr int kGroupedK = 2;         // C[g] = A[:, tokens of g] * B[:, tokens of g]^T

constexpr int kMaxGroups = 1024;     // the table has to fit the LDS that the largest ring leaves
// the table lies behind the LDS of the tiled kernel, its prefetch landing place and its flag, and two sets of scales
constexpr int kGroupTableOffset = 256 + 16;
constexpr int kGroupTableBytes = 2 * (kMaxGroups + 1) * 4;

// A group's tokens fill whole runs of this many columns of a transposed operand: whole K tiles, so
// that no K tile holds tokens of two groups and none needs a test for its end.
constexpr int kTokenRun = 128;

struct GroupSpec {
    const int *offsets;              // groups + 1 row numbers
    int groups;
    int rows;
    const float *a_scale;            // kGroupedRows: one per row; kGroupedK: groups x M; null for 1
    const float *b_scale;            // groups x N, or one per group; null for 1
    int b_per_column;
    int type;                        // of C (FP8GEMM_DEV_OUT_*)
    int accumulate;                  // C += instead of C =
};

__device__ __forceinline__ int group_offset(const GroupSpec &g, int i)
{
    int v = g.offsets[i];
    v = v < 0 ? 0 : v;
    return v > g.rows ? g.rows : v;
}

// Fills tab_tile[0 .. groups] (number of the first tile of each group, and the total) and tab_row[0 .. groups]:
//   tiles_m == 0 (the groups cut the rows into tiles of UNIT): tab_row = row offsets;
//   tiles_m > 0 (every group has tiles_m x tiles_n tiles): tab_row = first run of UNIT tokens of each group in the
//   padded token axis.
// Returns the total.  Called by all threads; ends in a barrier.
template <int UNIT>
__device__ __forceinline__ int build_group_table(const GroupSpec &g, int tiles_m, int tiles_n, __attribute__((address_space(3))) int *tab_tile,
                                                 __attribute__((address_space(3))) int *tab_row)
{
    if (threadIdx.x < 64) {
        const int lane = threadIdx.x;
        int carry = 0;                                   // runs of UNIT rows in the groups before this chunk
        int highest = 0;                                 // largest offset before this chunk
        for (int c = 0; c < g.groups; c += 64) {
            const int i = c + lane;
            const bool mine = i < g.groups;
            int first = mine ? group_offset(g, i) : 0, end = mine ? group_offset(g, i + 1) : 0;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const int v = __shfl_up(first, off, 64);
                first = lane >= off && v > first ? v : first;
            }
            first = first > highest ? first : highest;
            end = end > first ? end : first;
            highest = __shfl(end, 63, 64);
            const int count = (end - first + UNIT - 1) / UNIT;
            int sum = count;                             // inclusive scan over the wave
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const int v = __shfl_up(sum, off, 64);
                sum += lane >= off ? v : 0;
            }
            const int before = carry + sum - count;
            if (mine) {
                tab_tile[i] = tiles_m > 0 ? i * tiles_m * tiles_n : before * tiles_n;
                tab_row[i] = tiles_m > 0 ? before : first;
                if (i == g.groups - 1) {
                    const int all = before + count;
                    tab_tile[i + 1] = tiles_m > 0 ? g.groups * tiles_m * tiles_n : all * tiles_n;
                    tab_row[i + 1] = tiles_m > 0 ? all : end;
                }
            }
            carry += __shfl(sum, 63, 64);
        }
    }
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(tab_tile[g.groups]);
}

// The group of tile number t < total: the last one whose first tile is not behind t (empty groups share
// their first tile with the next one).  Whole waves only.
__device__ __forceinline__ int group_of_tile(int groups, const __attribute__((address_space(3))) int *tab_tile, int t)
{
    const int lane = threadIdx.x & 63;
    int n = 0;
    for (int c = 0; c < groups; c += 64) {
        const int i = c + lane;
        n += __popcll(__ballot(i < groups && tab_tile[i < groups ? i : 0] <= t));
    }
    return __builtin_amdgcn_readfirstlane(n - 1);
}

#endif  // FP8GEMM_GROUP_TABLE_H
