// Wide numbers (fp32, bf16, fp16) to fp8 codes with power-of-two scales, row by row or transposed.
//
// The scale of a run of numbers is the smallest power of two s (2^-126 at least) with
// max|x| <= s * (largest finite code); both formats' largest codes are 1.75 * 2^e, so s follows from the
// exponent of the maximum and one comparison of its mantissa, and x / s is exact: the only rounding is the
// code's own, to nearest even, done by the conversion instructions.  Infinities and NaNs do not enter the
// maximum; +-Inf becomes the largest finite code and NaN 0x7F, as in the host codec (fp8.h).
#ifndef FP8GEMM_KERNEL_QUANTIZE_H
#define FP8GEMM_KERNEL_QUANTIZE_H

#include "group_table.h"

// biased exponent of the scale for a largest finite magnitude (given by its bits)
template <int FMT>
__device__ __forceinline__ int quant_scale_exponent(uint32_t amax_bits)
{
    if (amax_bits == 0) return 127;
    const int top = FMT == 0 ? 8 : 15;                    // 448 = 1.75 * 2^8, 57344 = 1.75 * 2^15
    const int e = (int)(amax_bits >> 23) - top + ((amax_bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return e < 1 ? 1 : e;
}
__device__ __forceinline__ float quant_scale(int e) { return __builtin_bit_cast(float, (uint32_t)e << 23); }
__device__ __forceinline__ float quant_inverse(int e) { return __builtin_bit_cast(float, (uint32_t)(254 - e) << 23); }

// the codes of two scaled numbers, in the low or the high half of a word
template <int FMT, bool HIGH>
__device__ __forceinline__ uint32_t quant_pair(float a, float b, uint32_t old)
{
    return FMT == 0 ? (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, (int)old, HIGH) : (uint32_t)__builtin_amdgcn_cvt_pk_bf8_f32(a, b, (int)old, HIGH);
}

// four scaled numbers -> one word of codes; `rough`: infinities and NaNs may be among them
template <int FMT>
__device__ __forceinline__ uint32_t quant_four(float a, float b, float c, float d, bool rough)
{
    uint32_t nan = 0;
    if (rough) {
        const float top = FMT == 0 ? 448.0f : 57344.0f;
        nan = (a != a ? 0x7Fu : 0u) | (b != b ? 0x7F00u : 0u) | (c != c ? 0x7F0000u : 0u) | (d != d ? 0x7F000000u : 0u);
        a = fminf(fmaxf(a, -top), top);                   // (a NaN becomes a number here; its code is replaced below)
        b = fminf(fmaxf(b, -top), top);
        c = fminf(fmaxf(c, -top), top);
        d = fminf(fmaxf(d, -top), top);
    }
    uint32_t w = quant_pair<FMT, true>(c, d, quant_pair<FMT, false>(a, b, 0));
    if (rough) {
        const uint32_t byte = ((nan & 0x01010101u) * 0xFFu);
        w = (w & ~byte) | nan;
    }
    return w;
}

// eight consecutive elements from a 16-byte aligned place
template <int TYPE>
__device__ __forceinline__ void quant_load8(const void *base, size_t index, float v[8])
{
    if (TYPE == FP8GEMM_DEV_OUT_F32) {
        const v4f *p = reinterpret_cast<const v4f *>(static_cast<const float *>(base) + index);
        const v4f a = p[0], b = p[1];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = a[i];
            v[4 + i] = b[i];
        }
    } else {
        const v4i w = *reinterpret_cast<const v4i *>(static_cast<const unsigned short *>(base) + index);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (TYPE == FP8GEMM_DEV_OUT_BF16) {
                v[2 * i] = __builtin_bit_cast(float, (uint32_t)w[i] << 16);
                v[2 * i + 1] = __builtin_bit_cast(float, (uint32_t)w[i] & 0xFFFF0000u);
            } else {
                v[2 * i] = (float)__builtin_bit_cast(_Float16, (unsigned short)((uint32_t)w[i] & 0xFFFFu));
                v[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (unsigned short)((uint32_t)w[i] >> 16));
            }
        }
    }
}

// folds |x| into the running maximum of finite magnitudes; whether x is an infinity or a NaN
__device__ __forceinline__ bool quant_fold(float x, uint32_t &amax_bits)
{
    const uint32_t b = __builtin_bit_cast(uint32_t, x) & 0x7FFFFFFFu;
    const bool odd = b >= 0x7F800000u;
    amax_bits = !odd && b > amax_bits ? b : amax_bits;      // (non-negative floats order like their bits)
    return odd;
}

// Row r of codes = row (row_index ? row_index[r] : r) of x; a row_index outside [0, x_rows) gives a row of zeros with
// scale 1.  WAVES waves to a row, 4 / WAVES rows to a workgroup.  HBM bound: every wide element is read once, held in
// registers (HELD pieces of eight elements a lane) until the row's maximum is known, and its code written.
template <int TYPE, int FMT, int WAVES, int HELD>
__global__ __launch_bounds__(256) void quantize_rows_kernel(int rows, int cols, const void *__restrict__ x, size_t x_stride, int x_rows,
                                                            const int *__restrict__ row_index, uint8_t *__restrict__ codes, float *__restrict__ scales)
{
    __shared__ uint32_t part[4];
    __shared__ int part_odd[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long row = (long)blockIdx.x * (4 / WAVES) + wave / WAVES;
    const int sub = wave % WAVES;
    if (WAVES == 1 && row >= rows) return;                 // (with four waves to a row the grid is exactly the rows)
    const long src = row_index ? (long)row_index[row] : row;
    const bool there = src >= 0 && src < x_rows;
    float v[HELD][8];
    uint32_t amax = 0;
    bool odd = false;
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
        const int c = ((h * WAVES + sub) * 64 + lane) * 8;
        if (there && c < cols) {
            quant_load8<TYPE>(x, (size_t)src * x_stride + c, v[h]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[h][i] = 0.0f;
        }
    }
#pragma unroll
    for (int h = 0; h < HELD; ++h)
#pragma unroll
        for (int i = 0; i < 8; ++i) odd |= quant_fold(v[h][i], amax);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const uint32_t o = (uint32_t)__shfl_xor((int)amax, off, 64);
        amax = o > amax ? o : amax;
    }
    bool rough = __any(odd);
    if (WAVES > 1) {
        if (lane == 0) {
            part[wave] = amax;
            part_odd[wave] = rough;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            amax = part[w] > amax ? part[w] : amax;
            rough |= part_odd[w] != 0;
        }
    }
    const int e = quant_scale_exponent<FMT>(amax);
    const float inv = quant_inverse(e);
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
        const int c = ((h * WAVES + sub) * 64 + lane) * 8;
        if (c < cols) {
            v2u w;
            w[0] = quant_four<FMT>(v[h][0] * inv, v[h][1] * inv, v[h][2] * inv, v[h][3] * inv, rough);
            w[1] = quant_four<FMT>(v[h][4] * inv, v[h][5] * inv, v[h][6] * inv, v[h][7] * inv, rough);
            *reinterpret_cast<v2u *>(codes + (size_t)row * cols + c) = w;
        }
    }
    if (lane == 0 && sub == 0) scales[row] = quant_scale(e);
}

// The same for any row length, stride and alignment: a workgroup to a row, which is read twice.
template <int TYPE, int FMT>
__global__ __launch_bounds__(256) void quantize_rows_any_kernel(int cols, const void *__restrict__ x, size_t x_stride, int x_rows,
                                                                const int *__restrict__ row_index, uint8_t *__restrict__ codes, float *__restrict__ scales)
{
    __shared__ uint32_t part[4];
    __shared__ int part_odd[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const size_t row = blockIdx.x;
    const long src = row_index ? (long)row_index[row] : (long)row;
    const bool there = src >= 0 && src < x_rows;
    uint32_t amax = 0;
    bool odd = false;
    if (there)
        for (int c = threadIdx.x; c < cols; c += 256) odd |= quant_fold(load_in(x, (size_t)src * x_stride + c, TYPE), amax);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const uint32_t o = (uint32_t)__shfl_xor((int)amax, off, 64);
        amax = o > amax ? o : amax;
    }
    if (lane == 0) {
        part[wave] = amax;
    }
    const bool any_odd = __any(odd);
    if (lane == 0) part_odd[wave] = any_odd;
    __syncthreads();
    bool rough = false;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        amax = part[w] > amax ? part[w] : amax;
        rough |= part_odd[w] != 0;
    }
    const int e = quant_scale_exponent<FMT>(amax);
    const float inv = quant_inverse(e);
    for (int c = threadIdx.x; c < cols; c += 256) {
        const float v = there ? load_in(x, (size_t)src * x_stride + c, TYPE) * inv : 0.0f;
        codes[row * cols + c] = (uint8_t)quant_four<FMT>(v, v, v, v, rough);
    }
    if (threadIdx.x == 0) scales[row] = quant_scale(e);
}

// ---- transposed, grouped -------------------------------------------------------------------
// codes_t (cols x ld): the tokens of group g, a column each, from its first run of kTokenRun columns on (group_table.h), zeros
// behind its last token and behind the last group; scales (groups x cols).  A workgroup takes kColBlock columns
// of one group, reads them twice (once for the maxima), and turns 128 x 64 pieces around in LDS so that every
// column's 128 codes leave as one whole line.
constexpr int kColBlock = 64;
constexpr int kColPitch = kTokenRun + 4;       // bytes of a column in LDS: 33 words, so that eight columns x eight words hit 64 banks

template <int TYPE, bool VEC>
__device__ __forceinline__ void quant_load_cols(const void *x, size_t at, int c, int cols, float v[8])
{
    if (VEC) {
        if (c < cols) {
            quant_load8<TYPE>(x, at + c, v);
            return;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c + i < cols ? load_in(x, at + c + i, TYPE) : 0.0f;
    }
}

template <int TYPE, int FMT, bool VEC>
__global__ __launch_bounds__(256) void quantize_columns_kernel(GroupSpec grp, int cols, const void *__restrict__ x, size_t x_stride, int x_rows,
                                                               const int *__restrict__ row_index, uint8_t *__restrict__ codes_t, size_t ld,
                                                               float *__restrict__ scales)
{
    using lds_int = __attribute__((address_space(3))) int;
    __shared__ int table[2 * (kMaxGroups + 1)];
    __shared__ uint32_t amax_of[32][kColBlock];
    __shared__ uint8_t turn[kColBlock * kColPitch];
    lds_int *tab_run = (lds_int *)table, *tab_row = (lds_int *)table + kMaxGroups + 1;
    build_group_table<kTokenRun>(grp, 0, 1, tab_run, tab_row);
    const int col_blocks = (cols + kColBlock - 1) / kColBlock;
    const int g = (int)(blockIdx.x / (unsigned)col_blocks);
    const int c0 = (int)(blockIdx.x % (unsigned)col_blocks) * kColBlock;
    const int cc = threadIdx.x & 7, slot = threadIdx.x >> 3;       // eight columns, one of 32 rows
    const int c = c0 + cc * 8;
    // the place of 16 codes in the write-out: column, piece
    const int wcol = threadIdx.x >> 3, wpiece = threadIdx.x & 7;
    if (g == grp.groups) {
        // behind the last group: zeros
        for (size_t at = (size_t)tab_run[g] * kTokenRun; at < ld; at += kTokenRun)
            for (int j = wcol; j < kColBlock; j += 32)
                if (c0 + j < cols) *reinterpret_cast<v4i *>(codes_t + (size_t)(c0 + j) * ld + at + wpiece * 16) = v4i{0, 0, 0, 0};
        return;
    }
    const int first = tab_row[g], end = tab_row[g + 1];
    const auto source = [&](int r) -> long { return row_index ? (long)row_index[r] : (long)r; };
    // ---- the columns' largest magnitudes
    uint32_t amax[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    bool odd = false;
    for (int r = first + slot; r < end; r += 32) {
        const long src = source(r);
        if (src < 0 || src >= x_rows) continue;
        float v[8];
        quant_load_cols<TYPE, VEC>(x, (size_t)src * x_stride, c, cols, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) odd |= quant_fold(v[i], amax[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) amax_of[slot][cc * 8 + i] = amax[i];
    const bool rough = __syncthreads_or(odd) != 0;
    float inv[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        uint32_t m = 0;
        for (int s = 0; s < 32; ++s) {
            const uint32_t o = amax_of[s][cc * 8 + i];
            m = o > m ? o : m;
        }
        const int e = quant_scale_exponent<FMT>(m);
        inv[i] = quant_inverse(e);
        if (slot == 0 && c + i < cols) scales[(size_t)g * cols + c + i] = quant_scale(e);
    }
    // ---- the codes, a run of tokens at a time: a thread has four tokens of its eight columns
    for (int r0 = first; r0 < end; r0 += kTokenRun) {
        float v[4][8];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int r = r0 + slot * 4 + u;
            const long src = r < end ? source(r) : -1;
            if (src >= 0 && src < x_rows) {
                quant_load_cols<TYPE, VEC>(x, (size_t)src * x_stride, c, cols, v[u]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[u][i] = 0.0f;
            }
        }
        __syncthreads();                                  // (the run before has been written out)
#pragma unroll
        for (int i = 0; i < 8; ++i)
            *reinterpret_cast<uint32_t *>(turn + (cc * 8 + i) * kColPitch + slot * 4) =
                quant_four<FMT>(v[0][i] * inv[i], v[1][i] * inv[i], v[2][i] * inv[i], v[3][i] * inv[i], rough);
        __syncthreads();
        const size_t at = ((size_t)tab_run[g] + (size_t)(r0 - first) / kTokenRun) * kTokenRun;
#pragma unroll
        for (int j = wcol; j < kColBlock; j += 32)
            if (c0 + j < cols) {
                const uint32_t *p = reinterpret_cast<const uint32_t *>(turn + j * kColPitch + wpiece * 16);
                *reinterpret_cast<v4i *>(codes_t + (size_t)(c0 + j) * ld + at + wpiece * 16) = v4i{(int)p[0], (int)p[1], (int)p[2], (int)p[3]};
            }
    }
}

#endif  // FP8GEMM_KERNEL_QUANTIZE_H
