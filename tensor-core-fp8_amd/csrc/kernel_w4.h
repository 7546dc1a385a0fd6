// y = W x for few rows of x and a W of 4-bit numbers, one scale per run of a row: HBM bound, W is the traffic.
//
//     y[i][j] = x_scale[i] * sum_t x[i][t] * (q[j][t] - zero[j][t / run]) * scale[j][t / run]
//
// A wave streams 16 rows of W (columns of y) through a private LDS ring with direct loads, as kernel_skinny.h
// does for 8-bit codes, expands them to 16 bits in registers and multiplies on v_mfma_f32_16x16x32: even with one
// row of x the matrix unit does in 16 clocks what 512 multiply-adds would take, and the vector unit is left
// to the expansion, one instruction per weight:
//   integers: a nibble q is masked into the mantissa of 16.0, which makes 16 + q; a second MFMA on the same x
//     with -(16 + zero) in place of W takes the excess out (exact factors: small integers in 16 bits; sums in fp32,
//     so that x from 2^116 on, an infinity among them, can overflow both to a NaN),
//     and zero points cost no instruction per weight (taking it out as (16 + zero) times the sum of the run's x
//     saves those MFMAs and loses more at the staging of x, from four rows on by a factor);
//   e2m1: the conversion instruction, two weights at a time, which also applies power-of-two scales where
//     x is bf16 (exact but for weights of 2^128 and more, byte 253 on: bf16 has fp32's exponents, down to 2^-133).
// Other scales multiply the fp32 sum of a run, so neither weights nor scales are rounded.
//
// Which 8 of 32 consecutive k a lane holds is free as long as x agrees.  Runs of whole 128 k: a lane takes 32
// consecutive weights with one 16-byte LDS read.  Shorter runs: the four lanes of a row share 32 consecutive
// weights, so that an MFMA stays inside one run.
//
// A workgroup of eight waves is WC waves side by side (16 columns each) times WK waves along K, whose sums are
// added in wave order through LDS: few columns still fill the chip.  It goes through several blocks of columns;
// x and the scales of all of them are staged in LDS once, then the waves' rings run without a break over all blocks.
// One row, 28672 x 8192 integers in runs of 128: 27 us, 4.5 TB/s; runs of 32 37 us.  By the counters the vector unit is what is
// busiest, 64 and 70 % of the CUs' time, start and end of the launch included (matrix unit 28 and 18, LDS 26 and 30).
#ifndef FP8GEMM_KERNEL_W4_H
#define FP8GEMM_KERNEL_W4_H

#include "kernel_ptile.h"
#include "kernel_skinny.h"
#include "w4_args.h"

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));

constexpr int kW4Waves = 8, kW4WavesShift = 3;         // of a workgroup
constexpr int kW4RowBytes = 128;                       // of a row of W per ring stage: 256 weights
constexpr int kW4StageK = 2 * kW4RowBytes;
constexpr int kW4StageBytes = 16 * kW4RowBytes;
constexpr int kW4StageLoads = kW4StageBytes / 1024;
constexpr int kW4RingTwo = 2, kW4RingFour = 4;          // slots of a wave's ring: what fits
__host__ __device__ constexpr int w4_ring_bytes(int slots) { return kW4Waves * slots * kW4StageBytes; }

// how the scales lie in LDS: as they are stored, bytes as bf16 (the same powers of two) where a sum is multiplied
constexpr int kW4ScaleF32 = 0, kW4ScaleBf16 = 1, kW4ScaleF16 = 2, kW4ScaleByte = 3;

template <bool F16, int MODE>
__device__ __forceinline__ v4i w4_expand(uint32_t w, float scale)
{
    v4i r;
    if constexpr (MODE == kW4Int) {
        // the nibbles of each 16-bit half, lowest first, into the mantissa's top four bits of 16.0
        // (mask and exponent kept in registers, one of each kind: the and-or takes no literals)
        uint32_t mask = F16 ? 0x03C003C0u : 0x00780078u, sixteen = F16 ? 0x4C004C00u : 0x41804180u;
        asm("" : "+s"(mask));
        asm("" : "+v"(sixteen));
        constexpr int UP = F16 ? 6 : 3;                   // from bit 0 to the mantissa's top
        r[0] = (int)(((w << UP) & mask) | sixteen);
        r[1] = (int)(((UP >= 4 ? w << (UP >= 4 ? UP - 4 : 0) : w >> (UP >= 4 ? 0 : 4 - UP)) & mask) | sixteen);
        r[2] = (int)(((w >> (8 - UP)) & mask) | sixteen);
        r[3] = (int)(((w >> (12 - UP)) & mask) | sixteen);
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

// eight codes of x as f16 numbers (exact); both formats are expanded and one picked, so that the callers' loops stay without branches
__device__ __forceinline__ v4i w4_widen(v2u c, int type)
{
    v4i r;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int lo = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)c[h], 1.0f, false));
        const int hi = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)c[h], 1.0f, true));
        // (e5m2: the upper byte of an f16)
        r[2 * h] = type == FP8GEMM_T_E5M2 ? (int)__builtin_amdgcn_perm(0u, c[h], 0x010C000Cu) : lo;
        r[2 * h + 1] = type == FP8GEMM_T_E5M2 ? (int)__builtin_amdgcn_perm(0u, c[h], 0x030C020Cu) : hi;
    }
    return r;
}

// Staged x and scales.  x: a row behind the other, 16 bytes apart in the banks; scales: a column behind the other, an entry per run
// of RUN k -- the scale and, for integers, -(16 + zero) beside it in 16 bits -- odd counts of 16 bytes apart.  A lane's reads
// then differ by constants that the instructions carry, and 16 lanes read 16 rows or columns without a conflict.
__host__ __device__ constexpr int w4_entry_bytes(int mode, int kind)
{
    return kind == kW4ScaleByte ? 1 : (kind == kW4ScaleF32 ? 4 : 2) * (mode == kW4Int ? 2 : 1);
}
__host__ __device__ constexpr int w4_x_pitch(int chunk) { return chunk * 2 + 16; }
__host__ __device__ constexpr int w4_scale_pitch(int runs, int entry) { return ((runs * entry + 15) / 16 | 1) * 16; }
// two sets of the partial sums of the waves along K: rows x 16 floats a wave
__host__ __device__ constexpr int w4_part_bytes(int wk, int rows) { return wk > 1 ? 2 * (wk - 1) * (kW4Waves / wk) * rows * 64 : 0; }

// eight numbers of x as the weights are expanded: integers 0 4, 1 5, 2 6, 3 7
template <int MODE>
__device__ __forceinline__ v4i w4_order(v4i t)
{
    if (MODE != kW4Int) return t;
    return v4i{(int)__builtin_amdgcn_perm((uint32_t)t[2], (uint32_t)t[0], 0x05040100u), (int)__builtin_amdgcn_perm((uint32_t)t[2], (uint32_t)t[0], 0x07060302u),
               (int)__builtin_amdgcn_perm((uint32_t)t[3], (uint32_t)t[1], 0x05040100u), (int)__builtin_amdgcn_perm((uint32_t)t[3], (uint32_t)t[1], 0x07060302u)};
}

// Stages `units` pieces of eight numbers of each of `rows` rows of x, row m0 on, from k = c0 on (zeros behind the last k), by the
// first `threads` threads: piece after piece, row after row, kW4XLoads loads of a thread in flight.  CODES: x in fp8.
constexpr int kW4XLoads = 4;
template <int MODE, bool CODES>
__device__ __forceinline__ void w4_stage_x(const W4Args &p, int m0, int rows, int c0, int units, LDS_AS uint8_t *xs, int x_pitch, int threads)
{
    int row = 0, u = threadIdx.x;
    while (u >= units) {
        u -= units;
        ++row;
    }
    while (row < rows) {
        v4i v[kW4XLoads];
        int at[kW4XLoads];
        bool there[kW4XLoads];
#pragma unroll
        for (int b = 0; b < kW4XLoads; ++b) {
            at[b] = row < rows ? row * x_pitch + u * 16 : -1;
            there[b] = row < rows && c0 + u * 8 < p.k;
            // (a place outside reads the first numbers instead: no branch holds up the loads behind it)
            const size_t from = there[b] ? (size_t)(m0 + row) * p.k + c0 + u * 8 : 0;
            if (CODES) {
                const v2u c = *reinterpret_cast<const v2u *>(static_cast<const uint8_t *>(p.x) + from);
                v[b] = v4i{(int)c[0], (int)c[1], 0, 0};
            } else {
                v[b] = *reinterpret_cast<const v4i *>(static_cast<const unsigned short *>(p.x) + from);
            }
            u += threads;
            while (u >= units) {
                u -= units;
                ++row;
            }
        }
#pragma unroll
        for (int b = 0; b < kW4XLoads; ++b) {
            v4i o = w4_order<MODE>(CODES ? w4_widen(v2u{(uint32_t)v[b][0], (uint32_t)v[b][1]}, p.x_type) : v[b]);
            if (!there[b]) o = v4i{0, 0, 0, 0};
            if (at[b] >= 0) *reinterpret_cast<LDS_AS v4i *>(xs + at[b]) = o;
        }
    }
}

// -(16 + z) in 16 bits, twice: z in the top of the mantissa of -16
template <bool F16>
__device__ __forceinline__ uint32_t w4_excess(uint32_t z)
{
    return F16 ? 0xCC00CC00u | (z << 6) | (z << 22) : 0xC180C180u | (z << 3) | (z << 19);
}
// the staged entry of a stored scale (its bits) and zero point (fp32 scales: the scale alone)
template <bool F16, int MODE, int KIND, int ES>
__device__ __forceinline__ uint32_t w4_pack_entry(uint32_t bits, uint32_t z)
{
    // (a byte b stands for 2^(b - 127); as bf16 that is b << 7, 0 the subnormal 0x0040 and 255 a NaN.  The conversion takes
    // the byte as it is.)
    if (ES == 1 && KIND == kW4ScaleBf16) bits = bits == 0 ? 0x0040u : (bits == 255 ? 0x7FC0u : bits << 7);
    if (MODE == kW4Int && KIND != kW4ScaleF32) bits |= w4_excess<F16>(z) & 0xFFFF0000u;
    return bits;
}

// Stages the scales (and zero points) of `block_cols` columns for k from first_k on, `runs` staged runs each, by `threads` threads.
// ES: bytes of a stored scale; VEC: a stored run is a staged run and 16 bytes of scales can be read at once.  Columns from
// `cols` on and what lies behind the last k are staged as zeros (x is zero there, or nothing is stored).
template <bool F16, int MODE, int RUN, int KIND, int ES, bool VEC>
__device__ __forceinline__ void w4_stage_scales(const W4Args &p, size_t at0, int first_k, int runs, int cols, int block_cols, LDS_AS uint8_t *out, int tid, int threads)
{
    constexpr int EB = w4_entry_bytes(MODE, KIND);
    constexpr int E = VEC ? 16 / ES : 1;                  // scales a thread takes at once
    constexpr int BATCH = 2;                              // ... and how many such loads it has in flight
    const int pitch = w4_scale_pitch(runs, EB);
    const int units = (runs + E - 1) / E;                 // of a column, dealt to a power of two of threads
    const int shift = units > 32 ? 6 : (units > 1 ? 32 - __builtin_clz(units - 1) : 0);
    const int sub = tid & ((1 << shift) - 1), cols_at_once = threads >> shift;
    for (int unit = sub; unit < units; unit += 1 << shift)
        for (int col0 = tid >> shift; col0 < block_cols; col0 += BATCH * cols_at_once) {
            const int at_k = first_k + unit * E * RUN;
            const size_t at_row = VEC ? (size_t)(first_k / RUN + unit * E) : (size_t)(at_k / p.run);
            v4i raw[BATCH], z[BATCH];                     // (not VEC: one scale, one zero point, in the lowest bits)
#pragma unroll
            for (int b = 0; b < BATCH; ++b) {
                const int col = col0 + b * cols_at_once;
                raw[b] = z[b] = v4i{0, 0, 0, 0};
                if (col < cols && at_k < p.k) {           // (VEC: E divides what a row holds, all of them or none)
                    const size_t at = at0 + (size_t)col * p.per_row + at_row;
                    const uint8_t *from = static_cast<const uint8_t *>(p.w_scale) + at * ES;
                    if constexpr (VEC)
                        raw[b] = *reinterpret_cast<const v4i *>(from);
                    else
                        raw[b][0] = ES == 4 ? *reinterpret_cast<const int *>(from) : (ES == 2 ? *reinterpret_cast<const unsigned short *>(from) : *from);
                    if (MODE == kW4Int) {
                        if (!p.zeros) {
                            z[b] = v4i{0x08080808, 0x08080808, 0x08080808, 0x08080808};
                        } else if constexpr (E == 1) {
                            z[b][0] = p.zeros[at];
                        } else if constexpr (E == 4) {
                            z[b][0] = *reinterpret_cast<const int *>(p.zeros + at);
                        } else if constexpr (E == 8) {
                            const v2u t = *reinterpret_cast<const v2u *>(p.zeros + at);
                            z[b][0] = (int)t[0];
                            z[b][1] = (int)t[1];
                        } else {
                            z[b] = *reinterpret_cast<const v4i *>(p.zeros + at);
                        }
                    }
                }
            }
#pragma unroll
            for (int b = 0; b < BATCH; ++b) {
                const int col = col0 + b * cols_at_once;
                if (col >= block_cols) continue;
                LDS_AS uint8_t *to = out + col * pitch + unit * E * EB;
                if constexpr (KIND == kW4ScaleByte) {     // the bytes as they are
                    if constexpr (VEC)
                        *reinterpret_cast<LDS_AS v4i *>(to) = raw[b];
                    else
                        *to = (uint8_t)raw[b][0];
                    continue;
                }
                // (VEC: a column's pitch has room for whole units)
                v4i word = {0, 0, 0, 0};
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const uint32_t part = (uint32_t)raw[b][e * ES / 4] >> (8 * (e * ES % 4));
                    const uint32_t bits = ES == 4 ? part : part & (ES == 2 ? 0xFFFFu : 0xFFu);
                    const uint32_t zero = ((uint32_t)z[b][e / 4] >> (8 * (e & 3))) & 15u;
                    const uint32_t entry = w4_pack_entry<F16, MODE, KIND, ES>(bits, zero);
                    if constexpr (EB == 8) {
                        word[2 * (e & 1)] = (int)entry;
                        word[2 * (e & 1) + 1] = (int)w4_excess<F16>(zero);
                        if (!VEC) *reinterpret_cast<LDS_AS v2u *>(to) = v2u{(uint32_t)word[0], (uint32_t)word[1]};
                        if (VEC && (e & 1)) *reinterpret_cast<LDS_AS v4i *>(to + (e - 1) * EB) = word;
                    } else if constexpr (EB == 4) {
                        word[e & 3] = (int)entry;
                        if (!VEC) *reinterpret_cast<LDS_AS uint32_t *>(to) = entry;
                        if (VEC && (e & 3) == 3) *reinterpret_cast<LDS_AS v4i *>(to + (e - 3) * EB) = word;
                    } else {
                        if (!VEC) *reinterpret_cast<LDS_AS unsigned short *>(to) = (unsigned short)entry;
                        if (VEC) {
                            word[(e & 7) / 2] = (e & 1) ? (int)((uint32_t)word[(e & 7) / 2] | (entry << 16)) : (int)entry;
                            if ((e & 7) == 7) *reinterpret_cast<LDS_AS v4i *>(to + (e - 7) * EB) = word;
                        }
                    }
                }
            }
        }
}

// an entry of the staged scales: the scale, and for integers the 16-bit -(16 + zero) twice
template <int MODE, int KIND>
__device__ __forceinline__ void w4_entry(const LDS_AS uint8_t *at, float &scale, uint32_t &excess)
{
    uint32_t bits;
    if constexpr (MODE == kW4Int && KIND == kW4ScaleF32) {
        const v2u e = *reinterpret_cast<const LDS_AS v2u *>(at);
        bits = e[0];
        excess = e[1];
    } else if constexpr (MODE == kW4Int) {
        bits = *reinterpret_cast<const LDS_AS uint32_t *>(at);
        excess = __builtin_amdgcn_perm(bits, bits, 0x03020302u);
    } else if constexpr (KIND == kW4ScaleF32) {
        bits = *reinterpret_cast<const LDS_AS uint32_t *>(at);
    } else if constexpr (KIND == kW4ScaleByte) {
        bits = *at;
    } else {
        bits = *reinterpret_cast<const LDS_AS unsigned short *>(at);
    }
    if constexpr (KIND == kW4ScaleF32)
        scale = __builtin_bit_cast(float, bits);
    else if constexpr (KIND == kW4ScaleBf16)
        scale = __builtin_bit_cast(float, bits << 16);
    else if constexpr (KIND == kW4ScaleF16)
        scale = (float)__builtin_bit_cast(_Float16, (unsigned short)bits);
    else
        scale = __builtin_bit_cast(float, bits << 23);
}

// the scales staged from the stored type, 16 bytes at a time where runs and addresses allow it
template <bool F16, int MODE, int RUN, int KIND>
__device__ __forceinline__ void w4_stage_scales_any(const W4Args &p, size_t at0, int first_k, int runs, int cols, int block_cols, LDS_AS uint8_t *out, int tid, int threads)
{
    const int es = p.scale_type == FP8GEMM_T_E8M0 ? 1 : (p.scale_type == FP8GEMM_T_F32 ? 4 : 2), last = 16 / es - 1;
    const bool vec = p.run == RUN && ((p.per_row | runs | (first_k / RUN)) & last) == 0 && reinterpret_cast<uintptr_t>(p.w_scale) % 16 == 0 &&
                     (!p.zeros || reinterpret_cast<uintptr_t>(p.zeros) % 16 == 0);
#define W4_STAGE(ES) \
    (vec ? w4_stage_scales<F16, MODE, RUN, KIND, ES, true>(p, at0, first_k, runs, cols, block_cols, out, tid, threads) \
         : w4_stage_scales<F16, MODE, RUN, KIND, ES, false>(p, at0, first_k, runs, cols, block_cols, out, tid, threads))
    if constexpr (KIND == kW4ScaleF32) {
        W4_STAGE(4);
    } else if constexpr (KIND == kW4ScaleByte) {
        W4_STAGE(1);
    } else {
        if (KIND == kW4ScaleBf16 && es == 1)
            W4_STAGE(1);
        else
            W4_STAGE(2);
    }
#undef W4_STAGE
}

// the rows of group g: offsets clamped to the matrix and raised to the largest before them (group_table.h)
__device__ __forceinline__ void w4_group_rows(const W4Args &p, int g, int &first, int &end)
{
    first = 0;
    end = p.rows;
    if (!p.offsets) return;
    GroupSpec spec = {};
    spec.offsets = p.offsets;
    spec.rows = p.rows;
    int most = 0;
    for (int i = threadIdx.x & 63; i <= g; i += 64) {
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
}

// an extent of `bytes` (2^32 - 16 at most) from `base` on
__device__ __forceinline__ __amdgpu_buffer_rsrc_t w4_rsrc(const void *base, size_t bytes)
{
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), 0, (int)(uint32_t)(bytes > 0xFFFFFFF0u ? 0xFFFFFFF0u : bytes), 0x00020000);
}

// Four lanes 16 apart hold 16 consecutive bytes each: afterwards word d of lane q is word q of lane d.
__device__ __forceinline__ void w4_turn(uint32_t w[4])
{
    const auto a = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false), b = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
    const auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false), d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    w[0] = c[0];
    w[1] = c[1];
    w[2] = d[0];
    w[3] = d[1];
}

// F16: x and the expanded weights are f16 (else bf16).  RUN: 128 or 32, the k between two scales of the staged table.
// KIND: how the scales are staged.
template <bool F16, int MODE, int RUN, int KIND>
__global__ __launch_bounds__(64 * kW4Waves, 4) void gemv_w4_kernel(W4Args p)
{
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const uint32_t lds_base = (uint32_t)(uintptr_t)(LDS_AS uint8_t *)lds;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int wk_count = 1 << p.wk_shift, wc_count = kW4Waves >> p.wk_shift;
    const int wc = wave & (wc_count - 1), wk = wave >> (kW4WavesShift - p.wk_shift);
    const int g = blockIdx.y;
    const int block_cols = 16 * wc_count;
    // this workgroup's blocks of columns, one behind the other
    const int block_n0 = blockIdx.x * block_cols * p.blocks;
    const int blocks = p.n - block_n0 < p.blocks * block_cols ? (p.n - block_n0 + block_cols - 1) >> (4 + kW4WavesShift - p.wk_shift) : p.blocks;
    const int n0 = block_n0 + 16 * wc;
    int first, end;
    w4_group_rows(p, g, first, end);
    if (end <= first) return;
    const int fi = lane & 15, fq = lane >> 4;

    // ---- ring of this wave: 16 rows of W, kW4RowBytes of each a stage, 16-byte pieces swizzled by row
    const size_t row_bytes = (size_t)p.k / 2;
    const int rows_w = p.n - n0 < 0 ? 0 : p.n - n0;
    // (rows past the last column of y, and bytes past the end of the last row, fall outside the extent and read as zeros;
    // bytes past the end of other rows are the next row's: x is zero there)
    const v4i rs = make_buffer_resource(p.w + ((size_t)g * p.n + (rows_w ? n0 : 0)) * row_bytes, (unsigned long long)rows_w * row_bytes);
    uint32_t ld_off[kW4StageLoads];
#pragma unroll
    for (int j = 0; j < kW4StageLoads; ++j) {
        const int row = j * 8 + (lane >> 3);
        ld_off[j] = (uint32_t)row * (uint32_t)row_bytes + (uint32_t)(((lane & 7) ^ (skinny_swizzle<kW4RowBytes>(row) & 7)) * 16);
    }
    const uint32_t ring = lds_base + (uint32_t)(wave * p.ring * kW4StageBytes);
    const int sw = skinny_swizzle<kW4RowBytes>(fi) & 7;
    const LDS_AS uint8_t *ring_ptr = (const LDS_AS uint8_t *)lds + wave * p.ring * kW4StageBytes + fi * kW4RowBytes;
    LDS_AS float *parts = (LDS_AS float *)((LDS_AS uint8_t *)lds + w4_ring_bytes(p.ring));
    LDS_AS uint8_t *xs = (LDS_AS uint8_t *)lds + w4_ring_bytes(p.ring) + w4_part_bytes(wk_count, p.part_rows);
    constexpr bool PER_LANE = RUN == 128 || MODE == kW4Fp4Scaled;     // a lane has 32 consecutive weights
    constexpr int EB = w4_entry_bytes(MODE, KIND), RUNS128 = 128 / RUN;
    const int unit = kW4StageK << p.wk_shift;
    const int whole = (p.k + unit - 1) & ~(unit - 1);
    int flushed = 0;                                      // tiles added up so far: which of the two sets of partial sums is next

    for (int m0 = first; m0 < end; m0 += 16) {
        const int rows = end - m0 < 16 ? end - m0 : 16;
        // Staged at a time: all of K of x, and the scales of as many blocks of columns as fit beside it; where not even one
        // does, a block at a time with K in equal pieces, whole ring stages for every wave along K (the host leaves room
        // for one), whole multiples of 2048 if they are longer.
        // (as planned, unless an expert has more rows than the plan took it to have)
        int chunk = whole, pass = p.pass;
        if (rows > p.plan_rows || pass == 0) {
            pass = (p.stage_bytes - rows * w4_x_pitch(whole)) / (block_cols * w4_scale_pitch(whole / RUN, EB));
            if (pass < 1) {
                // (what a run takes, and the padding of rows and columns)
                const int per_run = rows * RUN * 2 + block_cols * EB;
                const int most_k = (p.stage_bytes - rows * 16 - block_cols * 31) / per_run * RUN;
                const int step = most_k >= 2048 ? 2048 : unit;
                const int most = most_k / step * step, pieces = (p.k + most - 1) / most;
                chunk = ((p.k + pieces - 1) / pieces + step - 1) / step * step;
                pass = 1;
            }
        }
        chunk = __builtin_amdgcn_readfirstlane(chunk);
        pass = __builtin_amdgcn_readfirstlane(pass);
        const int runs = chunk / RUN, x_pitch = w4_x_pitch(chunk), s_pitch = w4_scale_pitch(runs, EB);
        // this lane's place in the staged x (past the last row: that one again)
        const int x_row = (fi < rows ? fi : rows - 1) * x_pitch + (PER_LANE ? 4 * fq : fq) * 16;
        float x_scale[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) x_scale[r] = p.x_scale && 4 * fq + r < rows ? p.x_scale[m0 + 4 * fq + r] : 1.0f;
        v4f total = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int b0 = 0; b0 < blocks; b0 += pass) {
            const int nb = blocks - b0 < pass ? blocks - b0 : pass;
            for (int c0 = 0; c0 < p.k; c0 += chunk) {
                // Ring stages of K are dealt to the waves along K in turn, so that they read neighbouring lines; every workgroup
                // starts at its own one (workgroups in step would ask the same HBM channels at the same time).
                const int ks = ((p.k - c0 < chunk ? p.k - c0 : chunk) + kW4StageK - 1) / kW4StageK;
                const int T = ks > wk ? (ks - wk + wk_count - 1) >> p.wk_shift : 0;
                const int rot = T > 1 ? (int)(((((unsigned)(blockIdx.x + b0) * 2654435761u) >> 16) * (unsigned)T) >> 16) : 0;      // < T
                int next_b = 0, next_t = 0, left = nb * T;   // the next stage to load, and how many are left
                auto issue = [&](int stage) __attribute__((always_inline)) {
                    int t = next_t + rot;
                    t = t >= T ? t - T : t;
                    const uint32_t at = (uint32_t)(b0 + next_b) * (uint32_t)block_cols * (uint32_t)row_bytes + (uint32_t)((c0 + ((t << p.wk_shift) + wk) * kW4StageK) / 2);
#pragma unroll
                    for (int j = 0; j < kW4StageLoads; ++j)
                        buffer_load_lds_b128_stream(rs, ring + (uint32_t)(stage * kW4StageBytes + j * 1024), ld_off[j] + at, 0u);
                    --left;
                    if (++next_t == T) {
                        next_t = 0;
                        ++next_b;
                    }
                };
                __syncthreads();                          // (what was staged before is done with)
#pragma unroll
                for (int t = 0; t < kW4RingFour; ++t)
                    if (t < p.ring && left > 0) issue(t);
                // x and the scales: little of x by the lower half of the waves and the scales by the upper half at the same time, more by
                // all of them
                const bool with_x = b0 == 0 || chunk < whole;
                const int half = 32 * kW4Waves;
                const bool apart = rows * (chunk / 8) <= 2 * half * kW4XLoads;      // (two rounds of loads at most)
                const int x_threads = apart ? half : 2 * half;
                if (with_x && threadIdx.x < x_threads) {
                    if (F16 && p.x_type != FP8GEMM_T_F16)
                        w4_stage_x<MODE, true>(p, m0, rows, c0, chunk / 8, xs, x_pitch, x_threads);
                    else
                        w4_stage_x<MODE, false>(p, m0, rows, c0, chunk / 8, xs, x_pitch, x_threads);
                }
                LDS_AS uint8_t *ss = xs + rows * x_pitch;
                if (!with_x || !apart || threadIdx.x >= half) {
                    const int col0 = block_n0 + b0 * block_cols, staged = nb * block_cols;
                    const int cols = p.n - col0 < staged ? p.n - col0 : staged;
                    const size_t at0 = ((size_t)g * p.n + col0) * p.per_row;
                    const int tid = with_x && apart ? threadIdx.x - half : threadIdx.x, threads = with_x && apart ? half : 2 * half;
                    w4_stage_scales_any<F16, MODE, RUN, KIND>(p, at0, c0, runs, cols, staged, ss, tid, threads);
                }
                // (every load has landed: said here, so that the compiler does not wait for all of them inside the loop)
                wait_vmcnt<0>();
                __syncthreads();
                // The weights of a stage are read from the ring into registers while those of the stage before are multiplied:
                // the slot is free for another as soon as they are there.
                uint32_t now[kW4StageK / 32], next[kW4StageK / 32];
                auto read_stage = [&](int stage, uint32_t *w) __attribute__((always_inline)) {
                    asm volatile("" ::: "memory");        // (the ring is written behind the compiler's back)
                    const LDS_AS uint8_t *st = ring_ptr + stage * kW4StageBytes;
#pragma unroll
                    for (int h = 0; h < kW4StageK / 128; ++h) {       // 128 k: 64 bytes of a row, four 16-byte pieces
                        if constexpr (PER_LANE) {
                            const v4i v = *reinterpret_cast<const LDS_AS v4i *>(st + ((h * 4 + fq) ^ sw) * 16);
#pragma unroll
                            for (int d = 0; d < 4; ++d) w[4 * h + d] = (uint32_t)v[d];
                        } else {
#pragma unroll
                            for (int d = 0; d < 4; ++d) w[4 * h + d] = *reinterpret_cast<const LDS_AS uint32_t *>(st + ((h * 4 + d) ^ sw) * 16 + fq * 4);
                        }
                    }
                };
                int stage = 0, todo = nb * T;
                // (every load has landed, see above)
                if (todo > 0) read_stage(0, now);
                wait_lgkmcnt0();
                for (int b = 0; b < nb; ++b) {
                    if (c0 == 0) total = v4f{0.0f, 0.0f, 0.0f, 0.0f};
                    const LDS_AS uint8_t *s_block = ss + (b * block_cols + 16 * wc + fi) * s_pitch + (MODE == kW4Fp4Scaled && RUN == 32 ? fq : 0) * EB;
                    for (int t0 = 0; t0 < T; ++t0) {
                        if (left > 0) {
                            issue(stage);
                            if (p.ring == kW4RingTwo)
                                wait_vmcnt<(kW4RingTwo - 1) * kW4StageLoads>();
                            else
                                wait_vmcnt<(kW4RingFour - 1) * kW4StageLoads>();
                        } else {
                            wait_vmcnt<0>();
                        }
                        stage = stage == p.ring - 1 ? 0 : stage + 1;
                        if (--todo > 0) read_stage(stage, next);
                        int t = t0 + rot;
                        t = t >= T ? t - T : t;
                        const int k_at = ((t << p.wk_shift) + wk) * kW4StageK;
                        const LDS_AS uint8_t *x_at = xs + k_at * 2, *s_at = s_block + k_at / RUN * EB;
#pragma unroll
                        for (int h = 0; h < kW4StageK / 128; ++h) {
                            const uint32_t *w = now + 4 * h;
                            v4f sum, excess;
                            float lane_scale = 1.0f, s = 0.0f;
                            uint32_t pair = 0;
                            v4i minus;
                            if constexpr (MODE == kW4Fp4Scaled) w4_entry<MODE, KIND>(s_at + h * RUNS128 * EB, lane_scale, pair);
#pragma unroll
                            for (int d = 0; d < 4; ++d) {
                                const v4i wide = w4_expand<F16, MODE>(w[d], lane_scale);
                                const bool open = RUN == 32 || d == 0;         // a new run of the staged scales begins
                                if constexpr (MODE != kW4Fp4Scaled)
                                    if (open) {
                                        w4_entry<MODE, KIND>(s_at + (h * RUNS128 + (RUN == 32 ? d : 0)) * EB, s, pair);
                                        minus = v4i{(int)pair, (int)pair, (int)pair, (int)pair};
                                    }
                                const v4i a = *reinterpret_cast<const LDS_AS v4i *>(x_at + x_row + h * 256 + (PER_LANE ? d : 4 * d) * 16);
                                if constexpr (MODE == kW4Fp4Scaled) {
                                    total = w4_mfma<F16>(a, wide, total);
                                } else {
                                    // (the excess in a chain of its own: the two do not wait for each other)
                                    sum = w4_mfma<F16>(a, wide, open ? v4f{0.0f, 0.0f, 0.0f, 0.0f} : sum);
                                    if constexpr (MODE == kW4Int) excess = w4_mfma<F16>(a, minus, open ? v4f{0.0f, 0.0f, 0.0f, 0.0f} : excess);
                                }
                                if (MODE != kW4Fp4Scaled && (RUN == 32 || d == 3)) {
#pragma unroll
                                    for (int r = 0; r < 4; ++r) total[r] += s * (MODE == kW4Int ? sum[r] + excess[r] : sum[r]);
                                }
                            }
                        }
                        // all reads of the next stage have returned before its slot is refilled
                        wait_lgkmcnt0();
                        asm volatile("" ::: "memory");
                        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                        for (int d = 0; d < kW4StageK / 32; ++d) now[d] = next[d];
                    }
                    if (c0 + chunk < p.k) continue;
                    // ---- the waves along K, added in wave order (two sets of partial sums in turn: one barrier a tile);
                    // register r of lane (fi, fq) holds y[4 fq + r][column fi]
                    if (wk_count > 1) {
                        LDS_AS float *set = parts + (flushed & 1) * ((wk_count - 1) * wc_count * p.part_rows * 16);
                        ++flushed;
                        if (wk > 0)
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                if (4 * fq + r < rows) set[(((wk - 1) * wc_count + wc) * p.part_rows + 4 * fq + r) * 16 + fi] = total[r];
                        wait_lgkmcnt0();
                        asm volatile("" ::: "memory");
                        __builtin_amdgcn_s_barrier();     // (the loads in flight go on)
                        asm volatile("" ::: "memory");
                        if (wk == 0)
                            for (int o = 1; o < wk_count; ++o)
#pragma unroll
                                for (int r = 0; r < 4; ++r)
                                    if (4 * fq + r < rows) total[r] += set[(((o - 1) * wc_count + wc) * p.part_rows + 4 * fq + r) * 16 + fi];
                    }
                    const int col = n0 + (b0 + b) * block_cols + fi;
                    if (wk == 0 && col < p.n) {
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (4 * fq + r < rows) store_out(p.y, (size_t)(m0 + 4 * fq + r) * p.n + col, total[r] * x_scale[r], p.y_type);
                    }
                }
            }
        }
    }
}

// The same for more rows of x than one block of 16 (16 * MT at a time), where x no longer fits LDS and the waves would wait for
// it: K goes by in pieces, x through two LDS buffers and two sets of registers (a piece is read three pieces ahead), the
// weights straight into registers four pieces ahead, the scales staged for as many pieces as fit.  A wave takes TN blocks of
// 16 columns, so that a read of x from LDS feeds TN products: with one the LDS is what bounds 64 rows.  Two waves along K, or four
// where the columns are few.
//
// Where the four lanes of a row have to share 32 consecutive weights (see above) their 16-byte loads are turned around by
// swaps between lanes.  64 rows, integers in runs of 128: 4096 x 4096 17 us (the kernel above, in blocks of 64 rows, 69),
// 17536 x 6784 with 58 rows 55 (100): the matrix unit, LDS and the vector unit take 0.4 to 0.8 us of a piece's 1.7 each, and two
// waves on a SIMD in step overlap little of it.  Reading x a step ahead, or starting every workgroup at another piece, gains
// nothing.  What few columns cost besides is idle CUs: 64 rows of 4096 x 4096 have 128 workgroups, and the blocks of an expert's
// rows go by one behind the other in the same ones (1024 rows of 4096 x 4096 238 us).
constexpr int kW4Ahead = 4;
// WK waves along K: a piece has 128 k of each, a workgroup 16 * TN columns of the others side by side
__host__ __device__ constexpr int w4_piece(int wk) { return 128 * wk; }
__host__ __device__ constexpr int w4_wide_cols(int wk, int tn) { return 16 * tn * (kW4Waves / wk); }
__host__ __device__ constexpr int w4_wide_x_bytes(int mt, int wk) { return 2 * 16 * mt * w4_x_pitch(w4_piece(wk)); }

template <bool F16, int MODE, int RUN, int MT, int KIND, int WK, int TN, bool CODES>
__global__ __launch_bounds__(64 * kW4Waves) void gemm_w4_wide_kernel(W4Args p, int scale_pieces)
{
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    constexpr bool PER_LANE = RUN == 128 || MODE == kW4Fp4Scaled;
    constexpr int EB = w4_entry_bytes(MODE, KIND), WC = kW4Waves / WK, COLS = w4_wide_cols(WK, TN), PIECE = w4_piece(WK), PITCH = w4_x_pitch(PIECE);
    constexpr int UNITS = PIECE / 8, X_ROWS = 64 * kW4Waves / UNITS, XT = 16 * MT / X_ROWS;      // a thread stages every X_ROWS-th row's eight numbers
    static_assert(XT * X_ROWS == 16 * MT && kW4Ahead % 2 == 0, "whole turns");
    const int lane = threadIdx.x & 63, fi = lane & 15, fq = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), wc = wave % WC, wk = wave / WC;
    const int g = blockIdx.y, n0 = blockIdx.x * COLS;
    int first, end;
    w4_group_rows(p, g, first, end);
    if (end <= first) return;
    const size_t row_bytes = (size_t)p.k / 2;
    // (rows past the last column of y, and bytes past the end of the last row, fall outside the extent and read as zeros;
    // bytes past the end of other rows are the next row's: x is zero there)
    const __amdgpu_buffer_rsrc_t rw = w4_rsrc(p.w + ((size_t)g * p.n + n0) * row_bytes, (size_t)(p.n - n0 < COLS ? p.n - n0 : COLS) * row_bytes);
    uint32_t w_at[TN];
#pragma unroll
    for (int c = 0; c < TN; ++c) w_at[c] = (uint32_t)(16 * (TN * wc + c) + fi) * (uint32_t)row_bytes + (uint32_t)(wk * 64 + fq * 16);
    const int pieces = (p.k + PIECE - 1) / PIECE;
    constexpr uint32_t elem = CODES ? 1 : 2;
    LDS_AS uint8_t *xs = (LDS_AS uint8_t *)lds, *ss = xs + w4_wide_x_bytes(MT, WK);
    const int x_unit = threadIdx.x % UNITS, x_first = threadIdx.x / UNITS;       // this thread's eight columns and first row of a piece
    const int runs = scale_pieces * (PIECE / RUN), s_pitch = w4_scale_pitch(runs, EB);
    const LDS_AS uint8_t *s_lane[TN];
#pragma unroll
    for (int c = 0; c < TN; ++c) s_lane[c] = ss + (16 * (TN * wc + c) + fi) * s_pitch + (wk * (128 / RUN) + (MODE == kW4Fp4Scaled && RUN == 32 ? fq : 0)) * EB;
    const LDS_AS uint8_t *x_lane = xs + fi * PITCH + wk * 256 + (PER_LANE ? 4 * fq : fq) * 16;

    for (int m0 = first; m0 < end; m0 += 16 * MT) {
        const int rows = end - m0 < 16 * MT ? end - m0 : 16 * MT;
        const __amdgpu_buffer_rsrc_t rx = w4_rsrc(static_cast<const uint8_t *>(p.x) + (size_t)m0 * p.k * elem, (size_t)rows * p.k * elem);
        v4i x_raw[2][XT], w_raw[kW4Ahead][TN];
        auto load_x = [&](v4i (&r)[XT], int piece) __attribute__((always_inline)) {
            const int k = piece * PIECE + x_unit * 8;
#pragma unroll
            for (int i = 0; i < XT; ++i) {
                const uint32_t at = k < p.k ? ((uint32_t)(X_ROWS * i + x_first) * (uint32_t)p.k + (uint32_t)k) * elem : 0xFFFFFFF0u;
                if constexpr (CODES) {
                    const v2u c = __builtin_amdgcn_raw_buffer_load_b64(rx, (int)at, 0, 0);
                    r[i] = v4i{(int)c[0], (int)c[1], 0, 0};
                } else {
                    r[i] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rx, (int)at, 0, 0));
                }
            }
        };
        auto store_x = [&](const v4i (&r)[XT], int buffer) __attribute__((always_inline)) {
            LDS_AS uint8_t *to = xs + buffer * (16 * MT * PITCH) + x_first * PITCH + x_unit * 16;
#pragma unroll
            for (int i = 0; i < XT; ++i)
                *reinterpret_cast<LDS_AS v4i *>(to + X_ROWS * i * PITCH) = w4_order<MODE>(CODES ? w4_widen(v2u{(uint32_t)r[i][0], (uint32_t)r[i][1]}, p.x_type) : r[i]);
        };
        auto load_w = [&](v4i (&r)[TN], int piece) __attribute__((always_inline)) {
#pragma unroll
            for (int c = 0; c < TN; ++c)
                r[c] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rw, piece < pieces ? (int)(w_at[c] + (uint32_t)piece * (PIECE / 2)) : -16, 0, 2));
        };
        v4f total[MT][TN];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int c = 0; c < TN; ++c) total[i][c] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        load_x(x_raw[0], 0);
#pragma unroll
        for (int u = 0; u < kW4Ahead; ++u) load_w(w_raw[u], u);
        __syncthreads();                                  // (the rows before are done with)
        store_x(x_raw[0], 0);
        load_x(x_raw[0], 1);
        load_x(x_raw[1], 2);
        for (int s0 = 0; s0 < pieces; s0 += scale_pieces) {
            const int cols = p.n - n0 < COLS ? p.n - n0 : COLS;
            w4_stage_scales_any<F16, MODE, RUN, KIND>(p, ((size_t)g * p.n + n0) * p.per_row, s0 * PIECE, runs, cols, COLS, ss, threadIdx.x, 64 * kW4Waves);
            wait_lgkmcnt0();
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            const int s_end = pieces - s0 < scale_pieces ? pieces : s0 + scale_pieces;
            for (int q0 = s0; q0 < s_end; q0 += kW4Ahead) {
#pragma unroll
                for (int u = 0; u < kW4Ahead; ++u) {
                    const int q = q0 + u;
                    store_x(x_raw[u & 1], (u + 1) & 1);
                    __builtin_amdgcn_sched_barrier(0);    // (a load stays behind the last use of its registers: otherwise it gets others, and
                    load_x(x_raw[u & 1], q + 3);          // the copy back at the end of the loop waits for it)
                    uint32_t w[TN][4];
#pragma unroll
                    for (int c = 0; c < TN; ++c) {
#pragma unroll
                        for (int d = 0; d < 4; ++d) w[c][d] = (uint32_t)w_raw[u][c][d];
                        if constexpr (!PER_LANE) w4_turn(w[c]);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    const LDS_AS uint8_t *x_at = x_lane + (u & 1) * (16 * MT * PITCH);
                    const int s_at = (q - s0) * (PIECE / RUN) * EB;
                    v4f sum[MT][TN];
                    float s[TN];
                    v4i minus[TN];
#pragma unroll
                    for (int c = 0; c < TN; ++c) {
                        s[c] = 1.0f;
                        uint32_t pair = 0;
                        if constexpr (MODE == kW4Fp4Scaled) w4_entry<MODE, KIND>(s_lane[c] + s_at, s[c], pair);
                    }
#pragma unroll
                    for (int d = 0; d < 4; ++d) {
                        const bool open = RUN == 32 || d == 0;         // a new run of the staged scales begins
                        v4i a[MT];
#pragma unroll
                        for (int i = 0; i < MT; ++i) a[i] = *reinterpret_cast<const LDS_AS v4i *>(x_at + 16 * i * PITCH + (PER_LANE ? d : 4 * d) * 16);
#pragma unroll
                        for (int c = 0; c < TN; ++c) {
                            if constexpr (MODE != kW4Fp4Scaled)
                                if (open) {
                                    uint32_t pair = 0;
                                    w4_entry<MODE, KIND>(s_lane[c] + s_at + (RUN == 32 ? d : 0) * EB, s[c], pair);
                                    minus[c] = v4i{(int)pair, (int)pair, (int)pair, (int)pair};
                                }
                            const v4i wide = w4_expand<F16, MODE>(w[c][d], MODE == kW4Fp4Scaled ? s[c] : 1.0f);
#pragma unroll
                            for (int i = 0; i < MT; ++i) {
                                if constexpr (MODE == kW4Fp4Scaled) {
                                    total[i][c] = w4_mfma<F16>(a[i], wide, total[i][c]);
                                } else {
                                    sum[i][c] = w4_mfma<F16>(a[i], wide, open ? v4f{0.0f, 0.0f, 0.0f, 0.0f} : sum[i][c]);
                                }
                            }
                            if constexpr (MODE == kW4Int)
#pragma unroll
                                for (int i = 0; i < MT; ++i) sum[i][c] = w4_mfma<F16>(a[i], minus[c], sum[i][c]);
                        }
                        if (MODE != kW4Fp4Scaled && (RUN == 32 || d == 3)) {
#pragma unroll
                            for (int c = 0; c < TN; ++c)
#pragma unroll
                                for (int i = 0; i < MT; ++i)
#pragma unroll
                                    for (int r = 0; r < 4; ++r) total[i][c][r] += s[c] * sum[i][c][r];
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    load_w(w_raw[u], q + kW4Ahead);
                    wait_lgkmcnt0();
                    asm volatile("" ::: "memory");
                    __builtin_amdgcn_s_barrier();         // (the loads in flight go on)
                    asm volatile("" ::: "memory");
                }
            }
        }
        // ---- the waves along K, in order; register r of lane (fi, fq) holds y[16 i + 4 fq + r][column fi]
        static_assert((WK - 1) * WC * TN * MT * 1024 <= w4_wide_x_bytes(MT, WK), "no room for the partial sums");
        LDS_AS float *part = (LDS_AS float *)xs + lane * 4;
        if (wk > 0) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int c = 0; c < TN; ++c) *reinterpret_cast<LDS_AS v4f *>(part + ((((wk - 1) * WC + wc) * MT + i) * TN + c) * 256) = total[i][c];
        }
        __syncthreads();
        if (wk == 0) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int c = 0; c < TN; ++c) {
                    v4f y = total[i][c];
#pragma unroll
                    for (int o = 0; o < WK - 1; ++o) y += *reinterpret_cast<const LDS_AS v4f *>(part + (((o * WC + wc) * MT + i) * TN + c) * 256);
                    const int col = n0 + 16 * (TN * wc + c) + fi;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int row = i * 16 + 4 * fq + r;
                        if (row < rows && col < p.n)
                            store_out(p.y, (size_t)(m0 + row) * p.n + col, y[r] * (p.x_scale ? p.x_scale[m0 + row] : 1.0f), p.y_type);
                    }
                }
        }
    }
}

#endif  // FP8GEMM_KERNEL_W4_H
