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

}  // namespace tqf
