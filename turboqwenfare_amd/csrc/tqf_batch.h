// tqf_batch.h -- what the API needs of the kernels that take a batch's rows: the
// F8 products and the router.
#pragma once

#include "tqf_internal.h"

// The routed experts of a layer in the e4m3 format, prepared for
// tqf_hip_f8_experts_device.
struct tqf_hip_f8_experts {
    const uint8_t **d_mats;  // device [n_experts x 3], owned
    uint32_t n_experts, hidden, width;
};

namespace tqf {

// ---- e4m3 with a scale for each block of 128 (tqf_f8.hip) ------------------
struct F8Shape {
    uint32_t rows, cols;
    uint32_t kb;     // K blocks of 128
    uint32_t tiles;  // tiles of 32 rows: a multiple of 4
};
// Largest rows and columns of an F8 matrix: offsets inside a tile's K blocks
// stay in 32 bits.
constexpr uint32_t kF8MaxRows = 1u << 24, kF8MaxCols = 1u << 16;
__host__ __device__ inline F8Shape f8_shape(uint32_t rows, uint32_t cols) {
    return F8Shape{rows, cols, (cols + 127) / 128, (rows + 127) / 128 * 4};
}
__host__ __device__ inline size_t f8_tile_bytes(const F8Shape &s) { return (size_t)s.tiles * s.kb * 4096; }
inline size_t f8_scale_count(const F8Shape &s) { return (size_t)(s.tiles / 4) * s.kb; }
inline size_t f8_layout_bytes(const F8Shape &s) { return f8_tile_bytes(s) + f8_scale_count(s) * 4; }
// Byte of element (row, col) in the tiles.
__host__ __device__ inline size_t f8_offset(const F8Shape &s, size_t row, size_t col) {
    return ((row >> 5) * s.kb + (col >> 7)) * 4096 + ((col >> 4) & 7) * 512 + (row & 31) * 16 + (col & 15);
}
hipError_t launch_f8_repack(hipStream_t s, const uint8_t *q, const float *scales, const F8Shape &d, uint8_t *out);

// y [t x rows] = Q(x [t x cols]) W^T; types TQF_HIP_TYPE_*.  scratch holds
// f8_matmul_scratch_bytes.
size_t f8_matmul_scratch_bytes(const F8Shape &d, uint32_t t);
hipError_t launch_f8_matmul(hipStream_t s, const uint8_t *mat, const F8Shape &d, const void *x, int32_t x_type, uint32_t t,
                            void *y, int32_t y_type, void *scratch);

// The routed experts of a layer: mats [n_experts x 3] (gate, up, down).
struct F8ExpertsDev {
    const uint8_t *const *mats;
    uint32_t n_experts, hidden, width;
};
size_t f8_experts_scratch_bytes(const F8ExpertsDev &ex, uint32_t t, uint32_t top_k, int32_t y_type);
hipError_t launch_f8_experts(hipStream_t s, const F8ExpertsDev &ex, const void *x, int32_t x_type, uint32_t t,
                             const uint16_t *ids, const float *w, uint32_t top_k, void *y, int32_t y_type, int32_t *status,
                             void *scratch);

// ---- the batched router (tqf_router.hip) ------------------------------------
hipError_t launch_router_logits(hipStream_t s, const float *router, const void *x, int32_t x_type, uint32_t t,
                                uint32_t n_experts, uint32_t hidden, float *logits);
hipError_t launch_route_tokens(hipStream_t s, const void *logits, int32_t logits_type, uint32_t t, uint32_t n_experts,
                               const float *bias, const tqf_hip_route_options &o, uint16_t *ids, float *w, int32_t *status);

}  // namespace tqf
