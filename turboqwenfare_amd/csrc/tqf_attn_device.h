// tqf_attn_device.h -- what the attention kernels share.
#pragma once

#include "tqf_attn.h"
#include "tqf_f8.h"

namespace tqf {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kInf = __builtin_inff();

// Four rows of 16 elements of 16 bits, transposed: lane i of 16 points at four
// elements, 4 (i % 4) on, of row i / 4, and gets element i of the four rows.
__device__ __forceinline__ uint2 read_transposed(const uint8_t *lds) {
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)lds));
}

__device__ __forceinline__ float sigmoid(float x) { return 1.0f / (1.0f + __builtin_amdgcn_exp2f(-kLog2e * x)); }

// Weights of 0 do not keep infinities and NaN out of a matrix product.  A tile of
// values with any that not every row sees is multiplied four times: its finite
// values by the weights, then, as ones, its infinities of either sign and its NaN
// by whether a row sees their key; a row with any gets their sum.
enum Odd { kFinite, kPlusInf, kMinusInf, kNan };
__device__ __forceinline__ float odd_value(int what) { return what == kPlusInf ? kInf : what == kMinusInf ? -kInf : __builtin_nanf(""); }
__device__ __forceinline__ bf16x8 pick(u32x4 v, int what) {
    u32x4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        uint32_t both = 0;
#pragma unroll
        for (int b = 0; b < 32; b += 16) {
            const uint32_t bits = v[e] >> b & 0xFFFFu, mag = bits & 0x7FFFu;
            const bool hit = what == kNan ? mag > 0x7F80u : bits == (what == kPlusInf ? 0x7F80u : 0xFF80u);
            both |= (what == kFinite ? (mag >= 0x7F80u ? 0u : bits) : hit ? 0x3F80u : 0u) << b;
        }
        x[e] = both;
    }
    return __builtin_bit_cast(bf16x8, x);
}

}  // namespace tqf
