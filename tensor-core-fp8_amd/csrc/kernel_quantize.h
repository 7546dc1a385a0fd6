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

// eight consecutive elements as they are stored (a 16-bit type fills the first half)
struct QuantRaw {
    v4i lo, hi;
};
template <int TYPE>
__device__ __forceinline__ QuantRaw quant_load8_raw(const void *base, size_t index)      // from a 16-byte aligned place
{
    QuantRaw r = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    if (TYPE == FP8GEMM_DEV_OUT_F32) {
        const v4i *p = reinterpret_cast<const v4i *>(static_cast<const float *>(base) + index);
        r.lo = p[0];
        r.hi = p[1];
    } else {
        r.lo = *reinterpret_cast<const v4i *>(static_cast<const unsigned short *>(base) + index);
    }
    return r;
}
template <int TYPE>
__device__ __forceinline__ void quant_unpack8(const QuantRaw &r, float v[8])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t lo = (uint32_t)r.lo[i], hi = (uint32_t)r.hi[i];
        if (TYPE == FP8GEMM_DEV_OUT_F32) {
            v[i] = __builtin_bit_cast(float, lo);
            v[4 + i] = __builtin_bit_cast(float, hi);
        } else if (TYPE == FP8GEMM_DEV_OUT_BF16) {
            v[2 * i] = __builtin_bit_cast(float, lo << 16);
            v[2 * i + 1] = __builtin_bit_cast(float, lo & 0xFFFF0000u);
        } else {
            v[2 * i] = (float)__builtin_bit_cast(_Float16, (unsigned short)(lo & 0xFFFFu));
            v[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (unsigned short)(lo >> 16));
        }
    }
}
template <int TYPE>
__device__ __forceinline__ void quant_load8(const void *base, size_t index, float v[8])
{
    const QuantRaw r = quant_load8_raw<TYPE>(base, index);
    quant_unpack8<TYPE>(r, v);
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
// registers (HELD pieces of eight elements a lane) until the row's maximum is known, and its code written: 32768 rows
// of 4096 bf16 gathered from 16384 take 74 us.
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
// behind its last token and behind the last group; scales (groups x cols).  HBM bound.  A workgroup takes kColBlock
// columns (a line of 16-bit numbers) of one group, 256 or 512 rows at a time, quads of rows of eight columns a thread: a first walk
// finds the maxima, the second one goes backwards, so that it starts with the rows that are still in registers (all of
// them, for a group of no more rows) and goes on with those that are still cached.  128 x 64 pieces are turned
// around in LDS, so that every column's 128 codes leave as one whole line.
constexpr int kColBlock = 64;
constexpr int kColThreads = 512;
// rows at a time: four or eight a thread, which are 32 registers of either
__host__ __device__ constexpr int col_rows(int type) { return kColThreads / 8 * (type == FP8GEMM_DEV_OUT_F32 ? 4 : 8); }
constexpr int kColPitch = kTokenRun + 4;       // bytes of a column in LDS: 33 words, so that eight columns x eight words hit 64 banks

// elements at + c .. at + c + 7, those from `cols` on as zeros
template <int TYPE, bool VEC>
__device__ __forceinline__ QuantRaw quant_load_cols(const void *x, size_t at, int c, int cols)
{
    QuantRaw r = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    if (VEC) {
        if (c < cols) r = quant_load8_raw<TYPE>(x, at + c);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (c + i >= cols) continue;
            if (TYPE == FP8GEMM_DEV_OUT_F32) {
                const int w = static_cast<const int *>(x)[at + c + i];
                if (i < 4)
                    r.lo[i & 3] = w;
                else
                    r.hi[i & 3] = w;
            } else {
                const uint32_t h = static_cast<const unsigned short *>(x)[at + c + i];
                r.lo[i / 2] = (int)((uint32_t)r.lo[i / 2] | (h << (16 * (i & 1))));
            }
        }
    }
    return r;
}

template <int TYPE, int FMT, bool VEC>
__global__ __launch_bounds__(kColThreads) void quantize_columns_kernel(GroupSpec grp, int cols, const void *__restrict__ x, size_t x_stride, int x_rows,
                                                                       const int *__restrict__ row_index, uint8_t *__restrict__ codes_t, size_t ld,
                                                                       float *__restrict__ scales)
{
    using lds_int = __attribute__((address_space(3))) int;
    constexpr int WAVES = kColThreads / 64, ROWS = col_rows(TYPE), RUNS = ROWS / kTokenRun, QUADS = ROWS / (kColThreads / 2);
    __shared__ int table[2 * (kMaxGroups + 1)];
    __shared__ uint32_t amax_of[WAVES][kColBlock];
    __shared__ uint8_t turn[RUNS][kColBlock * kColPitch];
    lds_int *tab_run = (lds_int *)table, *tab_row = (lds_int *)table + kMaxGroups + 1;
    build_group_table<kTokenRun>(grp, 0, 1, tab_run, tab_row);
    const int col_blocks = (cols + kColBlock - 1) / kColBlock;
    const int g = (int)(blockIdx.x / (unsigned)col_blocks);
    const int c0 = (int)(blockIdx.x % (unsigned)col_blocks) * kColBlock;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int cc = threadIdx.x & 7, slot = threadIdx.x >> 3;       // eight columns, four of the rows
    const int c = c0 + cc * 8;
    // the place of 16 codes in the write-out: one of the runs written at once, column, piece of the run
    constexpr int AT_ONCE = kColThreads / (8 * kColBlock);
    const int wrun = threadIdx.x / (8 * kColBlock), wcol = (threadIdx.x >> 3) % kColBlock, wpiece = threadIdx.x & 7;
    if (g == grp.groups) {
        // behind the last group: zeros
        for (size_t at = ((size_t)tab_run[g] + wrun) * kTokenRun; at < ld; at += AT_ONCE * kTokenRun)
            if (c0 + wcol < cols) *reinterpret_cast<v4i *>(codes_t + (size_t)(c0 + wcol) * ld + at + wpiece * 16) = v4i{0, 0, 0, 0};
        return;
    }
    const int first = tab_row[g], end = tab_row[g + 1];
    const int batches = end > first ? (end - first + ROWS - 1) / ROWS : 0;
    QuantRaw raw[QUADS][4];
    auto load = [&](int batch) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < QUADS; ++q) {
            const int r0 = first + batch * ROWS + q * (kColThreads / 2) + slot * 4;
            long src[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) src[u] = r0 + u < end ? (row_index ? (long)row_index[r0 + u] : (long)(r0 + u)) : -1;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                raw[q][u] = QuantRaw{{0, 0, 0, 0}, {0, 0, 0, 0}};
                if (src[u] >= 0 && src[u] < x_rows) raw[q][u] = quant_load_cols<TYPE, VEC>(x, (size_t)src[u] * x_stride, c, cols);
            }
        }
    };
    // ---- the columns' largest magnitudes
    uint32_t amax[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    bool odd = false;
    for (int b = 0; b < batches; ++b) {
        load(b);
#pragma unroll
        for (int q = 0; q < QUADS; ++q)
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                float v[8];
                quant_unpack8<TYPE>(raw[q][u], v);
#pragma unroll
                for (int i = 0; i < 8; ++i) odd |= quant_fold(v[i], amax[i]);
            }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
        for (int off = 8; off < 64; off <<= 1) {
            const uint32_t o = (uint32_t)__shfl_xor((int)amax[i], off, 64);
            amax[i] = o > amax[i] ? o : amax[i];
        }
        if (lane < 8) amax_of[wave][cc * 8 + i] = amax[i];
    }
    const bool rough = __syncthreads_or(odd) != 0;
    float inv[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        uint32_t m = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const uint32_t o = amax_of[w][cc * 8 + i];
            m = o > m ? o : m;
        }
        const int e = quant_scale_exponent<FMT>(m);
        inv[i] = quant_inverse(e);
        if (slot == 0 && c + i < cols) scales[(size_t)g * cols + c + i] = quant_scale(e);
    }
    // ---- the codes
    for (int b = batches - 1; b >= 0; --b) {
        if (b < batches - 1) load(b);
        __syncthreads();                                  // (the runs before have been written out)
#pragma unroll
        for (int q = 0; q < QUADS; ++q) {
            float v[4][8];
#pragma unroll
            for (int u = 0; u < 4; ++u) quant_unpack8<TYPE>(raw[q][u], v[u]);
            uint8_t *to = turn[q * (kColThreads / 256) + slot / 32] + cc * 8 * kColPitch + slot % 32 * 4;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                *reinterpret_cast<uint32_t *>(to + i * kColPitch) = quant_four<FMT>(v[0][i] * inv[i], v[1][i] * inv[i], v[2][i] * inv[i], v[3][i] * inv[i], rough);
        }
        __syncthreads();
#pragma unroll
        for (int run = wrun; run < RUNS; run += AT_ONCE) {
            const int r = b * RUNS + run;                 // run of the group
            if (first + r * kTokenRun >= end || c0 + wcol >= cols) continue;
            const uint32_t *p = reinterpret_cast<const uint32_t *>(turn[run] + wcol * kColPitch + wpiece * 16);
            *reinterpret_cast<v4i *>(codes_t + (size_t)(c0 + wcol) * ld + ((size_t)tab_run[g] + r) * kTokenRun + wpiece * 16) = v4i{(int)p[0], (int)p[1], (int)p[2], (int)p[3]};
        }
    }
}

#endif  // FP8GEMM_KERNEL_QUANTIZE_H
