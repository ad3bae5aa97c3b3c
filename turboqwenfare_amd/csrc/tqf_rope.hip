// tqf_rope.hip -- the heads of an attention layer between its projection and the
// attention (gfx950):
//
//   q' = turn(q / sqrt(mean(q^2) + eps) * w_q)   for every query head,
//   k' = turn(k / sqrt(mean(k^2) + eps) * w_k)   for every key head,
//   turn: the pair (a, b) becomes (a cos - b sin, b cos + a sin), the angle
//         position * frequency of the pair,
//   q' and, if asked, k' and v as packed bf16 rows; k' and v into the cache slots,
//   as bf16 or as e4m3 with a scale for each token and head.
// And the residual add of the decode loop's attention block.
//
// Bound by the bytes, each read and written once: 4096 rows of 16 + 2 + 2 heads of
// 256 in bf16 (88 MB) take 21 us, 4.2 TB/s, where a copy reaches 5.1; into an e4m3
// cache they take as long (80 MB).  The add: 65536 rows of 2048 312 us, 5.2 TB/s.
#include <hip/hip_runtime.h>

#include "tqf_attn_device.h"
#include "tqf_f8.h"

namespace tqf {

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ void store8(uint16_t *p, const float (&v)[8]) {
    const u32x4 b = {bf16_bits2(v[0], v[1]), bf16_bits2(v[2], v[3]), bf16_bits2(v[4], v[5]), bf16_bits2(v[6], v[7])};
    *reinterpret_cast<u32x4 *>(p) = b;
}

// Workgroups (.x) take a token, alone or with others (.y) that have some of its
// heads; dim / 8 lanes take a head, eight values each.
template <typename XT, int D>
__global__ __launch_bounds__(kThreads) void qk_rope_kernel(RopeArgs a) {
    constexpr int kLanes = D / 8, kGroups = kThreads / kLanes;
    __shared__ float s_cos[D / 2], s_sin[D / 2];
    const uint32_t t = blockIdx.x, tid = threadIdx.x, lane = tid % kLanes, e0 = lane * 8;
    if (tid < a.pairs) {
        // the angle in turns, its whole turns taken off in 64 bits; what is left is at most half a turn
        const double turns = (double)a.positions[t] * a.turns[tid];
        const float part = (float)(turns - __builtin_rint(turns));
        sincospif(2.0f * part, &s_sin[tid], &s_cos[tid]);
    }
    __syncthreads();
    const uint32_t heads = a.q_heads + 2 * a.kv_heads;
    const int32_t slot = a.slots ? a.slots[t] : -1;
    const bool cached = slot >= 0 && (uint32_t)slot < a.cache.n_pages * a.cache.page;
    if (a.slots && slot != -1 && !cached && tid == 0 && a.status) *a.status = TQF_HIP_ERR_INVALID;
    const uint32_t page = cached ? (uint32_t)slot / a.cache.page : 0, at = cached ? (uint32_t)slot % a.cache.page : 0;
    for (uint32_t h = blockIdx.y * kGroups + tid / kLanes; h < heads; h += gridDim.y * kGroups) {
        const int kind = h < a.q_heads ? 0 : h < a.q_heads + a.kv_heads ? 1 : 2;
        const HeadRows &from = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
        const uint32_t hh = h - (kind == 0 ? 0 : kind == 1 ? a.q_heads : a.q_heads + a.kv_heads);
        float v[8];
        load_row<8>(static_cast<const XT *>(from.d) + t * from.row + hh * from.head + e0, 8, v);
        const float *w = kind == 0 ? a.q_norm : kind == 1 ? a.k_norm : nullptr;
        if (w) {
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(v[i], v[i], ss);
#pragma unroll
            for (int o = kLanes / 2; o >= 1; o /= 2) ss += __shfl_xor(ss, o);
            const float inv = 1.0f / sqrtf(ss * (1.0f / D) + a.eps);
            float g[8];
            load_row<8>(w + e0, 8, g);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = v[i] * inv * g[i];
        }
        if (kind < 2 && a.pairs) {
            if (a.neighbours) {
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const uint32_t p = (e0 + i) / 2;
                    if (p < a.pairs) {
                        const float c = s_cos[p], s = s_sin[p], x = v[i], y = v[i + 1];
                        v[i] = x * c - y * s;
                        v[i + 1] = y * c + x * s;
                    }
                }
            } else {
                // pairs is a multiple of 8: the partners of a lane's values are another lane's, in order
                const bool first = e0 < a.pairs, in = e0 < 2 * a.pairs;
                const int step = (int)(a.pairs / 8), other = (int)(tid & 63) + (first ? step : in ? -step : 0);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float y = __shfl(v[i], other);
                    if (in) {
                        const uint32_t p = first ? e0 + i : e0 + i - a.pairs;
                        v[i] = v[i] * s_cos[p] + (first ? -y : y) * s_sin[p];
                    }
                }
            }
        }
        if (kind == 0) store8(a.q_out + ((size_t)t * a.q_heads + hh) * D + e0, v);
        if (kind == 1 && a.k_out) store8(a.k_out + ((size_t)t * a.kv_heads + hh) * D + e0, v);
        if (kind == 2 && a.v_out) store8(a.v_out + ((size_t)t * a.kv_heads + hh) * D + e0, v);
        if (kind == 0 || !a.cache.k) continue;
        const size_t row = ((size_t)page * a.kv_heads + hh) * a.cache.page + at;
        if (!a.cache.f8) {
            if (cached) store8(static_cast<uint16_t *>(kind == 1 ? a.cache.k : a.cache.v) + row * D + e0, v);
        } else {
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(v[i]));
#pragma unroll
            for (int o = kLanes / 2; o >= 1; o /= 2) m = fmaxf(m, __shfl_xor(m, o));
            const F8Factors f = f8_factors(m);
            if (cached) {
                const uint2 b = make_uint2(f8_pack4(v[0] * f.inv, v[1] * f.inv, v[2] * f.inv, v[3] * f.inv),
                                           f8_pack4(v[4] * f.inv, v[5] * f.inv, v[6] * f.inv, v[7] * f.inv));
                *reinterpret_cast<uint2 *>(static_cast<uint8_t *>(kind == 1 ? a.cache.k : a.cache.v) + row * D + e0) = b;
                if (lane == 0) (kind == 1 ? a.cache.k_scales : a.cache.v_scales)[row] = f.scale;
            }
        }
    }
}

__global__ __launch_bounds__(kThreads) void add_rows_kernel(const float *a, const float *b, size_t n, float *out) {
    const size_t i = (size_t)blockIdx.x * kThreads + threadIdx.x;
    if (i < n) out[i] = a[i] + b[i];
}

template <typename XT>
void launch_for(hipStream_t s, const RopeArgs &a) {
    const uint32_t groups = kThreads / (a.dim / 8), heads = a.q_heads + 2 * a.kv_heads, want = (heads + groups - 1) / groups;
    // A workgroup that has all heads of a token reads them in turn (16 of 256 and 4 for k and v: three trips to memory).
    // While all of the workgroups run at once each takes those of one trip: 1 row 8.1 -> 6.4 us, 515 rows 9.7 -> 8.5 (with
    // events' time), 1024 rows 11.8 either way; with more than run at once the angles are made too often, 4096 rows 25.3
    // whole and 27.7.
    const dim3 grid(a.t, (uint64_t)a.t * want <= 8 * (uint64_t)cu_count() ? want : 1), block(kThreads);
    if (a.dim == 64) qk_rope_kernel<XT, 64><<<grid, block, 0, s>>>(a);
    if (a.dim == 128) qk_rope_kernel<XT, 128><<<grid, block, 0, s>>>(a);
    if (a.dim == 256) qk_rope_kernel<XT, 256><<<grid, block, 0, s>>>(a);
}

}  // namespace

hipError_t launch_qk_rope(hipStream_t s, const RopeArgs &a, int32_t x_type) {
    if (x_type == TQF_HIP_TYPE_F32) launch_for<float>(s, a);
    else launch_for<uint16_t>(s, a);
    return hipGetLastError();
}

hipError_t launch_add_rows(hipStream_t s, const float *a, const float *b, size_t n, float *out) {
    add_rows_kernel<<<dim3((uint32_t)((n + kThreads - 1) / kThreads)), dim3(kThreads), 0, s>>>(a, b, n, out);
    return hipGetLastError();
}

}  // namespace tqf
