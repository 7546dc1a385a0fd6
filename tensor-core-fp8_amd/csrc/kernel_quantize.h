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

// Eight consecutive elements as they are stored (a 16-bit type fills the first half), from any element's place: global memory
// takes 16 bytes at once from every address, only lines that are touched twice cost something.
typedef int quant_v4i __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t quant_v2u __attribute__((ext_vector_type(2), aligned(1)));
struct QuantRaw {
    v4i lo, hi;
};
template <int TYPE>
__device__ __forceinline__ QuantRaw quant_load8_raw(const void *base, size_t index)
{
    QuantRaw r = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    if (TYPE == FP8GEMM_DEV_OUT_F32) {
        const quant_v4i *p = reinterpret_cast<const quant_v4i *>(static_cast<const float *>(base) + index);
        r.lo = p[0];
        r.hi = p[1];
    } else {
        r.lo = *reinterpret_cast<const quant_v4i *>(static_cast<const unsigned short *>(base) + index);
    }
    return r;
}
// the first `count` < 8 of them, zeros behind
template <int TYPE>
__device__ __forceinline__ QuantRaw quant_load_some(const void *base, size_t index, int count)
{
    QuantRaw r = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
    for (int i = 0; i < 7; ++i) {
        if (i >= count) continue;
        if (TYPE == FP8GEMM_DEV_OUT_F32) {
            const int w = static_cast<const int *>(base)[index + i];
            if (i < 4)
                r.lo[i & 3] = w;
            else
                r.hi[i & 3] = w;
        } else {
            const uint32_t h = static_cast<const unsigned short *>(base)[index + i];
            r.lo[i / 2] = (int)((uint32_t)r.lo[i / 2] | (h << (16 * (i & 1))));
        }
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
// of 4096 bf16 that no cache holds take 62 us (6.5 TB/s), gathered from 16384 67, 8192 rows of 1843 18.
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
        QuantRaw raw = {{0, 0, 0, 0}, {0, 0, 0, 0}};
        if (there && c + 8 <= cols) raw = quant_load8_raw<TYPE>(x, (size_t)src * x_stride + c);
        quant_unpack8<TYPE>(raw, v[h]);
    }
    if (cols % 8 != 0) {                                   // the last piece of a row is a part of one
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
            const int c = ((h * WAVES + sub) * 64 + lane) * 8;
            if (there && c < cols && c + 8 > cols) quant_unpack8<TYPE>(quant_load_some<TYPE>(x, (size_t)src * x_stride + c, cols - c), v[h]);
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
            uint8_t *to = codes + (size_t)row * cols + c;
            if (c + 8 <= cols)
                *reinterpret_cast<quant_v2u *>(to) = w;
            else
                for (int i = 0; i < cols - c; ++i) to[i] = (uint8_t)(w[i / 4] >> (8 * (i & 3)));
        }
    }
    if (lane == 0 && sub == 0) scales[row] = quant_scale(e);
}

// The same for any row length: a workgroup to a row, which is read twice, an element a lane and load: 4096 rows of 28672 bf16
// 223 us, a single one 35, where 4096 rows of 16384 take 34 above.
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
// around in LDS, so that every column's 128 codes leave as one whole line.  32768 rows of 4096 bf16 in 32 uneven groups: 125 us, 5 TB/s
// of the 625 MB that move (three quarters of the rows are read a second time; 108 us in even groups), 4099 rows of 2048 in 8: 15.
constexpr int kColBlock = 64;
constexpr int kColThreads = 512;
// rows at a time: four or eight a thread, which are 32 registers of either
__host__ __device__ constexpr int col_rows(int type) { return kColThreads / 8 * (type == FP8GEMM_DEV_OUT_F32 ? 4 : 8); }
constexpr int kColPitch = kTokenRun + 4;       // bytes of a column in LDS: 33 words, so that eight columns x eight words hit 64 banks

// Where few blocks of columns and few groups leave CUs without work, the walks are split over the rows: a kernel for the
// maxima (PART 1: a workgroup takes the rows of one batch and raises the scales, cleared before, to its own -- a power of two
// orders like its bits, so the order of the workgroups does not matter) and one for the codes (PART 2).  16384 rows of 512 columns
// of one group take 22 us, in one walk 144.
constexpr int kColWhole = 0, kColMaxima = 1, kColCodes = 2;

__global__ __launch_bounds__(256) void quantize_clear_kernel(float *scales, size_t count)
{
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i < count) scales[i] = 0.0f;
}

template <int TYPE, int FMT, int PART>
__global__ __launch_bounds__(kColThreads) void quantize_columns_kernel(GroupSpec grp, int cols, const void *__restrict__ x, size_t x_stride, int x_rows,
                                                                       const int *__restrict__ row_index, uint8_t *__restrict__ codes_t, size_t ld,
                                                                       float *__restrict__ scales)
{
    using lds_int = __attribute__((address_space(3))) int;
    constexpr int WAVES = kColThreads / 64, ROWS = col_rows(TYPE), RUNS = ROWS / kTokenRun, QUADS = ROWS / (kColThreads / 2);
    __shared__ int table[2 * (kMaxGroups + 1)];
    __shared__ int batch_table[PART == kColWhole ? 1 : kMaxGroups + 1];
    __shared__ uint32_t amax_of[WAVES][kColBlock];
    __shared__ uint8_t turn[PART == kColMaxima ? 1 : RUNS][kColBlock * kColPitch];
    lds_int *tab_run = (lds_int *)table, *tab_row = (lds_int *)table + kMaxGroups + 1;
    const int col_blocks = (cols + kColBlock - 1) / kColBlock;
    int g = (int)(blockIdx.x / (unsigned)col_blocks), batch0 = 0;
    if constexpr (PART != kColWhole) {
        // (a group without rows gets no batch here: its scales of 1 are written below)
        const int total = build_group_table<ROWS>(grp, 0, 1, (lds_int *)batch_table, tab_row);
        if (g < total) {
            const int batch = g;
            g = group_of_tile(grp.groups, (lds_int *)batch_table, batch);
            batch0 = batch - __builtin_amdgcn_readfirstlane(batch_table[g]);
        } else {
            // the last workgroups: what lies behind the last group, and the groups without rows
            if (PART == kColMaxima || g < (int)(gridDim.x / (unsigned)col_blocks) - 1) return;
            g = grp.groups;
        }
        __syncthreads();
    }
    build_group_table<kTokenRun>(grp, 0, 1, tab_run, tab_row);
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
        if (PART == kColCodes)
            for (int e = threadIdx.x / kColBlock; e < grp.groups; e += kColThreads / kColBlock) {
                const int col = c0 + threadIdx.x % kColBlock;
                if (tab_row[e + 1] <= tab_row[e] && col < cols) scales[(size_t)e * cols + col] = 1.0f;
            }
        return;
    }
    // the rows of this workgroup: all of the group's, or those of one batch
    const int first = tab_row[g] + batch0 * ROWS, group_end = tab_row[g + 1];
    const int end = PART == kColWhole || group_end < first + ROWS ? group_end : first + ROWS;
    const int batches = end > first ? (end - first + ROWS - 1) / ROWS : 0;
    const bool tail = c0 + kColBlock > cols && cols % 8 != 0;      // a thread's eight columns may end behind the last one
    QuantRaw raw[QUADS][4];
    auto load = [&](int batch) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < QUADS; ++q) {
            if (first + batch * ROWS + q * (kColThreads / 2) >= end) continue;       // (uniform)
            const int r0 = first + batch * ROWS + q * (kColThreads / 2) + slot * 4;
            long src[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) src[u] = r0 + u < end ? (row_index ? (long)row_index[r0 + u] : (long)(r0 + u)) : -1;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                raw[q][u] = QuantRaw{{0, 0, 0, 0}, {0, 0, 0, 0}};
                if (src[u] >= 0 && src[u] < x_rows && c + 8 <= cols) raw[q][u] = quant_load8_raw<TYPE>(x, (size_t)src[u] * x_stride + c);
            }
            if (tail)
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (src[u] >= 0 && src[u] < x_rows && c < cols && c + 8 > cols) raw[q][u] = quant_load_some<TYPE>(x, (size_t)src[u] * x_stride + c, cols - c);
        }
    };
    // ---- the columns' largest magnitudes
    uint32_t amax[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    bool odd = false;
    for (int b = 0; b < batches; ++b) {
        load(b);
#pragma unroll
        for (int q = 0; q < QUADS; ++q) {
            if (first + b * ROWS + q * (kColThreads / 2) >= end) continue;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                float v[8];
                quant_unpack8<TYPE>(raw[q][u], v);
#pragma unroll
                for (int i = 0; i < 8; ++i) odd |= quant_fold(v[i], amax[i]);
            }
        }
    }
    if constexpr (PART != kColCodes) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
#pragma unroll
            for (int off = 8; off < 64; off <<= 1) {
                const uint32_t o = (uint32_t)__shfl_xor((int)amax[i], off, 64);
                amax[i] = o > amax[i] ? o : amax[i];
            }
            if (lane < 8) amax_of[wave][cc * 8 + i] = amax[i];
        }
    }
    const bool rough = __syncthreads_or(odd) != 0;
    if constexpr (PART == kColMaxima) {
        if (threadIdx.x < kColBlock && c0 + (int)threadIdx.x < cols) {
            uint32_t m = 0;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                const uint32_t o = amax_of[w][threadIdx.x];
                m = o > m ? o : m;
            }
            if (m != 0) atomicMax(reinterpret_cast<int *>(scales) + (size_t)g * cols + c0 + threadIdx.x, quant_scale_exponent<FMT>(m) << 23);
        }
        return;
    }
    float inv[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        int e = 127;
        if constexpr (PART == kColCodes) {
            // (0: no number but zeros.  The first batch writes the scale of 1 that stands for it, which reads as the same.)
            if (c + i < cols) {
                const int bits = __builtin_nontemporal_load(reinterpret_cast<const int *>(scales) + (size_t)g * cols + c + i);
                e = bits == 0 ? 127 : bits >> 23;
            }
        } else {
            uint32_t m = 0;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                const uint32_t o = amax_of[w][cc * 8 + i];
                m = o > m ? o : m;
            }
            e = quant_scale_exponent<FMT>(m);
        }
        inv[i] = quant_inverse(e);
        if (batch0 == 0 && slot == 0 && c + i < cols) scales[(size_t)g * cols + c + i] = quant_scale(e);
    }
    // ---- the codes
    for (int b = batches - 1; b >= 0; --b) {
        if (b < batches - 1) load(b);
        __syncthreads();                                  // (the runs before have been written out)
#pragma unroll
        for (int q = 0; q < QUADS; ++q) {
            if (first + b * ROWS + q * (kColThreads / 2) >= end) continue;
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
            *reinterpret_cast<v4i *>(codes_t + (size_t)(c0 + wcol) * ld + ((size_t)tab_run[g] + batch0 * RUNS + r) * kTokenRun + wpiece * 16) = v4i{(int)p[0], (int)p[1], (int)p[2], (int)p[3]};
        }
    }
}

#endif  // FP8GEMM_KERNEL_QUANTIZE_H
