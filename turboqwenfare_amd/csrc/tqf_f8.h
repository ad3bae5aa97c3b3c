// tqf_f8.h -- the e4m3 block-128 format on the device (not ABI).
//
// A matrix [rows x cols] of OCP e4m3 values with one f32 scale for each block
// of 128 x 128: W[r][k] = q[r][k] * s[r / 128][k / 128].  Device layout: tiles
// of 32 rows, four to a row of scale blocks (rows are padded to 128, columns
// to 128, with zeros), each tile's K blocks one after the other:
//   [tile][K block][8 chunks of 16 columns][32 rows][16 bytes]      (4 KiB a K block)
// then the scales [rows / 128][K blocks].  A wavefront's 16-byte loads of a
// tile are whole, contiguous KiB, and what lane l gets is an MFMA operand as it
// stands: rows l % 32 of chunks 2 j + l / 32 for the 32-row instructions, rows
// l % 16 of chunks 4 j + l / 16 for the 16-row ones (the order in which an
// MFMA takes its K elements is free, so long as both operands have the same).
//
// Rows of activations are quantised in blocks of 128 (f8_factors, f8_pack4) and kept
// by K block, for the form that reads them (t rows, t32: rounded up to 32):
//   tiles         [K block][t][128 bytes], scales [K block][t]; so is h, by position
//   split K       [K block][t32 / 32][8 chunks][32 rows][16 bytes], the matrices'
//                 order, scales [K block][t32]
// The forms for up to 16 rows and for few slots keep them in LDS.
#pragma once

#include "tqf_device.h"
#include "tqf_batch.h"

namespace tqf {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// e4m3's largest value, and the magnitude below which a block is all zero (its
// 448 / a would not be a finite f32).
constexpr float kF8Max = 448.0f;
constexpr float kF8Tiny = 0x1p-100f;

// The two factors of a block whose largest magnitude is a: values are stored as
// e4m3(x * inv) (to nearest, ties to even) and stand for q * scale.  |x| * inv
// passes 448 by at most two f32 roundings, which e4m3 rounds back.  NaN is not
// seen by the maximum; NaN * inv stays NaN, inf * 0 becomes it, and so a row
// with either gives NaN.
struct F8Factors {
    float scale, inv;
};
__device__ __forceinline__ F8Factors f8_factors(float a) {
    if (a < kF8Tiny) return F8Factors{0.0f, 0.0f};
    return F8Factors{a / kF8Max, kF8Max / a};
}
__device__ __forceinline__ uint32_t f8_pack4(float a, float b, float c, float d) {
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
}
// Eight e4m3 values as bf16 (exact).
__device__ __forceinline__ bf16x8 f8_widen(uint32_t lo, uint32_t hi) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// ---- elements of the callers' types ------------------------------------------
// N consecutive elements at p as f32, the first `valid` of them (0 past that).
// The wide loads need no alignment but the elements'.
template <int N>
__device__ __forceinline__ void load_row(const float *p, int valid, float (&v)[N]) {
    if (valid >= N) {
#pragma unroll
        for (int i = 0; i < N; i += 4) __builtin_memcpy(&v[i], p + i, 16);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = i < valid ? p[i] : 0.0f;
    }
}
template <int N>
__device__ __forceinline__ void load_row(const uint16_t *p, int valid, float (&v)[N]) {
    if (valid >= N) {
#pragma unroll
        for (int i = 0; i < N; i += 8) {
            u32x4 f;
            __builtin_memcpy(&f, p + i, 16);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[i + 2 * j] = __uint_as_float(f[j] << 16);
                v[i + 2 * j + 1] = __uint_as_float(f[j] & 0xFFFF0000u);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = i < valid ? __uint_as_float((uint32_t)p[i] << 16) : 0.0f;
    }
}

// Four consecutive outputs at p, the first `valid` of them, at any alignment.
// bf16 is rounded to nearest, ties to even.
__device__ __forceinline__ uint32_t bf16_bits2(float a, float b) {
    return (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)a) | ((uint32_t)__builtin_bit_cast(uint16_t, (__bf16)b) << 16);
}
__device__ __forceinline__ void store4(float *p, int valid, f32x4 v) {
    if (valid >= 4) {
        __builtin_memcpy(p, &v, 16);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < valid) p[i] = v[i];
    }
}
__device__ __forceinline__ void store4(uint16_t *p, int valid, f32x4 v) {
    if (valid >= 4) {
        const uint2 b = make_uint2(bf16_bits2(v[0], v[1]), bf16_bits2(v[2], v[3]));
        __builtin_memcpy(p, &b, 8);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < valid) p[i] = __builtin_bit_cast(uint16_t, (__bf16)v[i]);
    }
}

}  // namespace tqf
