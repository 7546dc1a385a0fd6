// y = W x for few rows of x and a W of 4-bit numbers, one scale per run of a row: HBM bound, W is the traffic.
//
//     y[i][j] = x_scale[i] * sum_t x[i][t] * (q[j][t] - zero[j][t / run]) * scale[j][t / run]
//
// A wave streams 16 rows of W (columns of y) through a private LDS ring with direct loads, as kernel_skinny.h
// does for 8-bit codes, expands them to 16 bits in registers and multiplies on v_mfma_f32_16x16x32: even with one
// row of x the matrix unit does in 16 clocks what 512 multiply-adds would take, and the vector unit is left
// to the expansion, one instruction per weight:
//   integers: a nibble q is masked into the mantissa of 16.0, which makes 16 + q; a second MFMA on the same x
//     with -(16 + zero) in place of W takes the excess out (all exact: small integers in 16 bits, sums in fp32),
//     so zero points cost no instruction per weight;
//   e2m1: the conversion instruction, two weights at a time, which also applies power-of-two scales where
//     x is bf16 (exact: bf16 has fp32's exponents).
// Other scales multiply the fp32 sum of a run, so neither weights nor scales are rounded.
//
// Which 8 of 32 consecutive k a lane holds is free as long as x agrees.  Runs of whole 128 k: a lane takes 32
// consecutive weights with one 16-byte LDS read.  Shorter runs: the four lanes of a row share 32 consecutive
// weights, so that an MFMA stays inside one run.
//
// A workgroup of four waves is WC waves side by side (16 columns each) times WK waves along K, whose sums are
// added in wave order through LDS at the end: few columns still fill the chip.  x and the scales of `chunk` k
// at a time are staged in LDS for all four.
#ifndef FP8GEMM_KERNEL_W4_H
#define FP8GEMM_KERNEL_W4_H

#include "kernel_ptile.h"
#include "kernel_skinny.h"

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));

constexpr int kW4Waves = 4;
constexpr int kW4RowBytes = 128;                       // of a row of W per ring stage: 256 weights
constexpr int kW4Stages = 5;
constexpr int kW4StageK = 2 * kW4RowBytes;
constexpr int kW4StageBytes = 16 * kW4RowBytes;
constexpr int kW4StageLoads = kW4StageBytes / 1024;
constexpr int kW4RingBytes = kW4Waves * kW4Stages * kW4StageBytes;

// how the weights become 16-bit numbers
constexpr int kW4Int = 0;           // 16 + q, corrected by a second MFMA
constexpr int kW4Fp4 = 1;           // e2m1, scales applied to sums
constexpr int kW4Fp4Scaled = 2;     // e2m1, power-of-two scales applied by the conversion (bf16 only)

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
    int chunk;                      // k staged at a time: a multiple of kW4StageK * WK
    int wk;
};

// one scale as a float
__device__ __forceinline__ float w4_scale(const void *p, size_t i, int type)
{
    if (type == FP8GEMM_T_E8M0) {
        const uint32_t b = static_cast<const uint8_t *>(p)[i];
        return __builtin_bit_cast(float, b == 0 ? 0x00400000u : (b == 255 ? 0x7FC00000u : b << 23));
    }
    return load_in(p, i, type);
}

template <bool F16, int MODE>
__device__ __forceinline__ v4i w4_expand(uint32_t w, float scale)
{
    v4i r;
    if constexpr (MODE == kW4Int) {
        // the nibbles of each 16-bit half, lowest first, into the mantissa's top four bits of 16.0
        if constexpr (F16) {
            r[0] = (int)(((w << 6) & 0x03C003C0u) | 0x4C004C00u);
            r[1] = (int)(((w << 2) & 0x03C003C0u) | 0x4C004C00u);
            r[2] = (int)(((w >> 2) & 0x03C003C0u) | 0x4C004C00u);
            r[3] = (int)(((w >> 6) & 0x03C003C0u) | 0x4C004C00u);
        } else {
            r[0] = (int)(((w << 3) & 0x00780078u) | 0x41804180u);
            r[1] = (int)(((w >> 1) & 0x00780078u) | 0x41804180u);
            r[2] = (int)(((w >> 5) & 0x00780078u) | 0x41804180u);
            r[3] = (int)(((w >> 9) & 0x00780078u) | 0x41804180u);
        }
    } else if constexpr (F16) {
        r[0] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 0));
        r[1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 1));
        r[2] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 2));
        r[3] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 3));
    } else {
        r[0] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0));
        r[1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1));
        r[2] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2));
        r[3] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3));
    }
    return r;
}

template <bool F16>
__device__ __forceinline__ v4f w4_mfma(v4i a, v4i b, v4f c)
{
    if constexpr (F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}

// eight consecutive numbers of x as 16-bit ones (f16 from fp8 codes: exact)
template <bool F16>
__device__ __forceinline__ v4i w4_load_x(const void *x, size_t index, int type)
{
    if (!F16 || type == FP8GEMM_T_F16) return *reinterpret_cast<const v4i *>(static_cast<const unsigned short *>(x) + index);
    const v2u c = *reinterpret_cast<const v2u *>(static_cast<const uint8_t *>(x) + index);
    v4i r;
    if (type == FP8GEMM_T_E5M2) {                       // the upper byte of an f16
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            r[2 * h] = (int)(((c[h] & 0xFFu) << 8) | ((c[h] & 0xFF00u) << 16));
            r[2 * h + 1] = (int)(((c[h] >> 8) & 0xFF00u) | (c[h] & 0xFF000000u));
        }
    } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[h], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[h], true);
            const _Float16 f[4] = {(_Float16)lo[0], (_Float16)lo[1], (_Float16)hi[0], (_Float16)hi[1]};
            r[2 * h] = (int)((uint32_t)__builtin_bit_cast(unsigned short, f[0]) | ((uint32_t)__builtin_bit_cast(unsigned short, f[1]) << 16));
            r[2 * h + 1] = (int)((uint32_t)__builtin_bit_cast(unsigned short, f[2]) | ((uint32_t)__builtin_bit_cast(unsigned short, f[3]) << 16));
        }
    }
    return r;
}

// LDS behind the ring for `rows` rows of x, `chunk` k and wc waves side by side; scales once per RUN k
constexpr int w4_stage_bytes(int rows, int chunk, int wc, int run_k, bool zeros)
{
    return rows * chunk * 2 + (chunk / run_k) * 16 * wc * 4 * (zeros ? 2 : 1);
}

// F16: x and the expanded weights are f16 (else bf16).  RUN: 128 or 32, the k between two scales of the staged table.
// MT: blocks of 16 rows of x held at once.
template <bool F16, int MODE, int RUN, int MT>
__global__ __launch_bounds__(64 * kW4Waves) void gemv_w4_kernel(W4Args p)
{
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const uint32_t lds_base = (uint32_t)(uintptr_t)(LDS_AS uint8_t *)lds;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int wc_count = kW4Waves / p.wk;
    const int wc = wave % wc_count, wk = wave / wc_count;
    const int g = blockIdx.y;
    const int block_cols = 16 * wc_count;
    const int block_n0 = blockIdx.x * block_cols;
    const int n0 = block_n0 + 16 * wc;
    int first = 0, end = p.rows;
    if (p.offsets) {
        // the group's rows: offsets clamped to the matrix and raised to the largest before them (group_table.h)
        GroupSpec spec = {};
        spec.offsets = p.offsets;
        spec.rows = p.rows;
        int most = 0;
        for (int i = lane; i <= g; i += 64) {
            const int v = group_offset(spec, i);
            most = v > most ? v : most;
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) {
            const int v = __shfl_xor(most, off, 64);
            most = v > most ? v : most;
        }
        first = __builtin_amdgcn_readfirstlane(most);
        end = __builtin_amdgcn_readfirstlane(group_offset(spec, g + 1));
        if (end <= first) return;
    }
    const int fi = lane & 15, fq = lane >> 4;

    // ---- ring of this wave: 16 rows of W, kW4RowBytes of each a stage, 16-byte pieces swizzled by row
    const size_t row_bytes = (size_t)p.k / 2;
    const int rows_w = p.n - n0 < 16 ? (p.n - n0 < 0 ? 0 : p.n - n0) : 16;
    // (rows past the last column of y, and bytes past the end of the last row, fall outside the extent and read as zeros;
    // bytes past the end of other rows are the next row's: x is zero there)
    const v4i rs = make_buffer_resource(p.w + ((size_t)g * p.n + (rows_w ? n0 : 0)) * row_bytes, (unsigned long long)rows_w * row_bytes);
    uint32_t ld_off[kW4StageLoads];
#pragma unroll
    for (int j = 0; j < kW4StageLoads; ++j) {
        const int row = j * 8 + (lane >> 3);
        ld_off[j] = (uint32_t)row * (uint32_t)row_bytes + (uint32_t)(((lane & 7) ^ (skinny_swizzle<kW4RowBytes>(row) & 7)) * 16);
    }
    const uint32_t ring = lds_base + (uint32_t)(wave * kW4Stages * kW4StageBytes);
    const uint8_t *ring_ptr = lds + wave * kW4Stages * kW4StageBytes;
    const int sw = skinny_swizzle<kW4RowBytes>(fi) & 7;
    auto issue = [&](int k0, int stage) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < kW4StageLoads; ++j)
            buffer_load_lds_b128_stream(rs, ring + (uint32_t)(stage * kW4StageBytes + j * 1024), ld_off[j] + (uint32_t)(k0 / 2), 0u);
    };

    uint8_t *xs = lds + kW4RingBytes;
    const int slice = p.chunk / p.wk;                     // k of a chunk that this wave multiplies
    for (int m0 = first; m0 < end; m0 += 16 * MT) {
        const int rows = end - m0 < 16 * MT ? end - m0 : 16 * MT;
        v4f total[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) total[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        for (int c0 = 0; c0 < p.k; c0 += p.chunk) {
            const int kw0 = c0 + wk * slice;
            const int left = p.k - kw0 < slice ? p.k - kw0 : slice;
            const int T = left > 0 ? (left + kW4StageK - 1) / kW4StageK : 0;
            __syncthreads();                              // (the staged x and scales of the chunk before are done with)
#pragma unroll
            for (int t = 0; t < kW4Stages - 1; ++t)
                if (t < T) issue(kw0 + t * kW4StageK, t);
            // ---- x and the scales of the chunk
            const int units = p.chunk / 8;                // eight numbers of a row; laid out [unit][row]
            for (int u = threadIdx.x; u < units * rows; u += 64 * kW4Waves) {
                const int unit = u / rows, row = u - unit * rows;
                const int kk = c0 + unit * 8;
                v4i v = {0, 0, 0, 0};
                if (kk < p.k) v = w4_load_x<F16>(p.x, (size_t)(m0 + row) * p.k + kk, p.x_type);
                if (MODE == kW4Int) {
                    // in the order of the expanded nibbles: 0 4, 1 5, 2 6, 3 7
                    const v4i o = v;
                    v[0] = (int)(((uint32_t)o[0] & 0xFFFFu) | ((uint32_t)o[2] << 16));
                    v[1] = (int)(((uint32_t)o[0] >> 16) | ((uint32_t)o[2] & 0xFFFF0000u));
                    v[2] = (int)(((uint32_t)o[1] & 0xFFFFu) | ((uint32_t)o[3] << 16));
                    v[3] = (int)(((uint32_t)o[1] >> 16) | ((uint32_t)o[3] & 0xFFFF0000u));
                }
                *reinterpret_cast<v4i *>(xs + (size_t)u * 16) = v;
            }
            float *ss = reinterpret_cast<float *>(xs + (size_t)units * rows * 16);
            uint32_t *zs = reinterpret_cast<uint32_t *>(ss + (p.chunk / RUN) * block_cols);
            const int runs = p.chunk / RUN, per_row = p.k / p.run;
            for (int u = threadIdx.x; u < runs * block_cols; u += 64 * kW4Waves) {
                const int col = u / runs, r = u - col * runs;
                const int kk = c0 + r * RUN;
                float s = MODE == kW4Fp4Scaled ? 1.0f : 0.0f;
                uint32_t z = 0;
                if (kk < p.k && block_n0 + col < p.n) {
                    const size_t at = ((size_t)g * p.n + block_n0 + col) * per_row + kk / p.run;
                    s = w4_scale(p.w_scale, at, p.scale_type);
                    if (MODE == kW4Int && p.zeros) z = p.zeros[at] & 15u;
                }
                ss[r * block_cols + col] = s;
                if (MODE == kW4Int && p.zeros) {
                    const float c = -(16.0f + (float)z);
                    const uint32_t h = out_bits16(c, F16 ? FP8GEMM_DEV_OUT_F16 : FP8GEMM_DEV_OUT_BF16);
                    zs[r * block_cols + col] = h | (h << 16);
                }
            }
            __syncthreads();
            // ---- this wave's slice of the chunk
            for (int t = 0; t < T; ++t) {
                if (t + kW4Stages - 1 < T) {
                    issue(kw0 + (t + kW4Stages - 1) * kW4StageK, (t + kW4Stages - 1) % kW4Stages);
                    wait_vmcnt<kW4StageLoads *(kW4Stages - 1)>();
                } else {
                    wait_vmcnt<0>();
                }
                asm volatile("" ::: "memory");            // (the ring is written behind the compiler's back)
                const uint8_t *st = ring_ptr + (t % kW4Stages) * kW4StageBytes + fi * kW4RowBytes;
#pragma unroll
                for (int h = 0; h < kW4StageK / 128; ++h) {           // 128 k: 64 bytes of a row, four 16-byte pieces
                    const int k128 = (kw0 - c0 + t * kW4StageK) / 128 + h;
                    uint32_t w[4];
                    if constexpr (RUN == 128 || MODE == kW4Fp4Scaled) {
                        const v4i v = *reinterpret_cast<const v4i *>(st + ((h * 4 + fq) ^ sw) * 16);
#pragma unroll
                        for (int d = 0; d < 4; ++d) w[d] = (uint32_t)v[d];
                    } else {
#pragma unroll
                        for (int d = 0; d < 4; ++d) w[d] = *reinterpret_cast<const uint32_t *>(st + ((h * 4 + d) ^ sw) * 16 + fq * 4);
                    }
                    constexpr bool PER_LANE = RUN == 128 || MODE == kW4Fp4Scaled;     // a lane has 32 consecutive weights
                    v4f sum[MT];
                    float lane_scale = 1.0f;
                    if constexpr (MODE == kW4Fp4Scaled) lane_scale = ss[(RUN == 128 ? k128 : k128 * 4 + fq) * block_cols + 16 * wc + fi];
#pragma unroll
                    for (int d = 0; d < 4; ++d) {
                        const v4i b = w4_expand<F16, MODE>(w[d], lane_scale);
                        const int unit = k128 * 16 + (PER_LANE ? 4 * fq + d : 4 * d + fq);
                        const bool open = RUN == 32 || d == 0;         // a new run of the staged scales begins
                        v4i zc;
                        if constexpr (MODE == kW4Int) {
                            int one = F16 ? (int)0xCE00CE00u : (int)0xC1C0C1C0u;       // -24
                            if (p.zeros) one = (int)zs[(RUN == 128 ? k128 : k128 * 4 + d) * block_cols + 16 * wc + fi];
                            zc = v4i{one, one, one, one};
                        }
#pragma unroll
                        for (int i = 0; i < MT; ++i) {
                            int row = i * 16 + fi;
                            row = row < rows ? row : rows - 1;
                            const v4i a = *reinterpret_cast<const v4i *>(xs + ((size_t)unit * rows + row) * 16);
                            if constexpr (MODE == kW4Fp4Scaled) {
                                total[i] = w4_mfma<F16>(a, b, total[i]);
                            } else {
                                sum[i] = w4_mfma<F16>(a, b, open ? v4f{0.0f, 0.0f, 0.0f, 0.0f} : sum[i]);
                                if constexpr (MODE == kW4Int) sum[i] = w4_mfma<F16>(a, zc, sum[i]);
                            }
                        }
                        if (MODE != kW4Fp4Scaled && (RUN == 32 || d == 3)) {
                            const float s = ss[(RUN == 128 ? k128 : k128 * 4 + d) * block_cols + 16 * wc + fi];
#pragma unroll
                            for (int i = 0; i < MT; ++i)
#pragma unroll
                                for (int r = 0; r < 4; ++r) total[i][r] += s * sum[i][r];
                        }
                    }
                }
                // all reads of this stage have returned before it is refilled
                wait_lgkmcnt0();
                asm volatile("" ::: "memory");
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        // ---- the waves along K, added in wave order; register r of lane (fi, fq) holds y[16 i + 4 fq + r][n0 + fi]
        if (p.wk > 1) {
            __syncthreads();
            v4f *part = reinterpret_cast<v4f *>(xs);
            if (wk > 0)
#pragma unroll
                for (int i = 0; i < MT; ++i) part[(((wk - 1) * wc_count + wc) * MT + i) * 64 + lane] = total[i];
            __syncthreads();
            if (wk == 0)
                for (int o = 1; o < p.wk; ++o)
#pragma unroll
                    for (int i = 0; i < MT; ++i) total[i] += part[(((o - 1) * wc_count + wc) * MT + i) * 64 + lane];
        }
        if (wk == 0 && n0 + fi < p.n) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = i * 16 + 4 * fq + r;
                    if (row < rows) {
                        const float s = p.x_scale ? p.x_scale[m0 + row] : 1.0f;
                        store_out(p.y, (size_t)(m0 + row) * p.n + n0 + fi, total[i][r] * s, p.y_type);
                    }
                }
        }
    }
}

#endif  // FP8GEMM_KERNEL_W4_H
