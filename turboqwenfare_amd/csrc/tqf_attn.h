// tqf_attn.h -- what the API needs of the attention kernels: heads with their
// rotation and cache, prompts, and rows over a paged cache.
#pragma once

#include "tqf_batch.h"

// The turns (revolutions) that each pair of a head makes from one position to
// the next, in 64 bits: at position 2^20 an f32 would be off by 2^-5 of one.
struct tqf_hip_rope {
    double *d_turns;  // device [pairs], owned
    uint32_t pairs;
};

namespace tqf {

// Element (t, h, i) at d[t * row + h * head + i].
struct HeadRows {
    const void *d;
    uint64_t row, head;
};

// A layer's cache: [n_pages][kv_heads][page][dim], f32 scales [n_pages][kv_heads][page] with e4m3.
struct KvCache {
    void *k, *v;
    float *k_scales, *v_scales;
    bool f8;
    uint32_t n_pages, page;  // page: a power of two, 16..256
    uint32_t kv_heads, dim;
};

struct RopeArgs {
    HeadRows q, k, v;
    uint32_t t, q_heads, kv_heads, dim;
    const float *q_norm, *k_norm;  // null: no norm
    float eps;
    const double *turns;  // [pairs]
    uint32_t pairs;       // 0: no rotation
    bool neighbours;      // pairs (2 i, 2 i + 1), else (i, i + pairs)
    const int32_t *positions;
    uint16_t *q_out, *k_out, *v_out;  // k_out, v_out: may be null
    KvCache cache;                    // k null: none
    const int32_t *slots;
    int32_t *status;
};
hipError_t launch_qk_rope(hipStream_t s, const RopeArgs &a, int32_t x_type);

struct PromptArgs {
    HeadRows q, k, v, gate;  // bf16; gate.d may be null
    const int32_t *cu_q, *cu_k;
    uint32_t n_seqs, total_q, total_k, q_heads, kv_heads, dim;
    float scale;
    uint16_t *y;
    int32_t *status;
};
size_t attn_prompt_scratch_bytes(const PromptArgs &a);
hipError_t launch_attn_prompt(hipStream_t s, const PromptArgs &a, void *scratch);

struct PagedArgs {
    HeadRows q, gate;
    uint32_t n_seqs, rows, q_heads;
    float scale;
    KvCache cache;
    const int32_t *pages;  // [n_seqs][max_pages]
    uint32_t max_pages;
    const int32_t *lens;
    uint16_t *y;
    int32_t *status;
};
size_t attn_paged_scratch_bytes(const PagedArgs &a);
hipError_t launch_attn_paged(hipStream_t s, const PagedArgs &a, void *scratch);

// d_out = d_a + d_b, element by element (tqf_loop.hip's kind of row kernel).
hipError_t launch_add_rows(hipStream_t s, const float *a, const float *b, size_t n, float *out);

}  // namespace tqf
