// tqf_attn_device.h -- what the attention kernels share.
#pragma once

#include <atomic>

#include "tqf_attn.h"
#include "tqf_f8.h"

namespace tqf {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kInf = __builtin_inff();

// A row's reference m follows its maximum only when that is 2^8 above it: the
// weights are then at most 2^8, their sums in f32 as exact as ever, and the sums
// of values are hardly ever multiplied again.
constexpr float kSlack = 8.0f;

// Compute units of the current device.
inline int cu_count() {
    static std::atomic<int> known[64];
    int dev = 0, n = 0;
    if (hipGetDevice(&dev) != hipSuccess) return 256;
    if (dev >= 0 && dev < 64 && (n = known[dev].load(std::memory_order_relaxed)) > 0) return n;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) return 256;
    if (dev >= 0 && dev < 64) known[dev].store(n, std::memory_order_relaxed);
    return n;
}

// Copies to LDS: lane l's 16 bytes go to lds + 16 l.
typedef __amdgpu_buffer_rsrc_t Desc;  // loads past its bytes give zero
typedef __attribute__((address_space(3))) void lds_void;
// p and bytes are the same in every lane: said to the compiler, which would else make
// a loop over their values of each copy.
__device__ __forceinline__ Desc make_desc(const void *p, uint32_t bytes) {
    const uint64_t at = reinterpret_cast<uint64_t>(p);
    const uint64_t low = __builtin_amdgcn_readfirstlane((uint32_t)at), high = __builtin_amdgcn_readfirstlane((uint32_t)(at >> 32));
    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void *>(high << 32 | (uint32_t)low), (short)0, __builtin_amdgcn_readfirstlane((int)bytes),
                                             0x00020000);
}
__device__ __forceinline__ void copy16(Desc d, uint32_t voff, void *lds) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(d, (lds_void *)lds, 16, voff, 0, 0, 0);
}
// soff: the same in every lane, and not held against the descriptor's end.
__device__ __forceinline__ void copy16(Desc d, uint32_t voff, uint32_t soff, void *lds) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(d, (lds_void *)lds, 16, voff, soff, 0, 0);
}

// 16 bytes at an offset; past the descriptor's end nothing is read (zeros) or written.
__device__ __forceinline__ u32x4 read16(Desc d, uint32_t voff) { return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(d, voff, 0, 0)); }
__device__ __forceinline__ void write16(Desc d, uint32_t voff, u32x4 x) { __builtin_amdgcn_raw_buffer_store_b128(x, d, voff, 0, 0); }

// Four rows of 16 elements of 16 bits, transposed: lane i of 16 points at four
// elements, 4 (i % 4) on, of row i / 4, and gets element i of the four rows.
__device__ __forceinline__ uint2 read_transposed(const uint8_t *lds) {
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)lds));
}

// The larger of lanes l and l ^ 32.
__device__ __forceinline__ float other_half_max(float x) {
    const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
}
// Of lanes l and l ^ 16.
__device__ __forceinline__ float other_row_max(float x) {
    const auto both = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
}

// x, as a value that is made here: what is computed from it is computed where it is
// used, and takes no register all along.
__device__ __forceinline__ uint32_t here(uint32_t x) {
    asm volatile("" : "+v"(x));
    return x;
}

// The reciprocal instruction is off by a last bit at most; a division would be ten instructions for each element.
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * x)); }

}  // namespace tqf
